// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + gain scale[s] B_s (A_s x[t]) for the rows t of adapter s.
//
// A tile is up to 16 or 128 rows of one adapter, gathered by number, so decoded tokens of requests that share an adapter and the rows of a prompt are one thing.  A
// cluster of CTAs takes a tile in one launch: each CTA multiplies a share of K (v = A x, rank columns), the shares are added in a fixed order, and each CTA then makes a share of the
// columns (B v) and adds it to y.  v stays in shared memory.  The shares of 16 rows meet through distributed shared memory; those of 128 through L2, see there.
//
// Matrix instructions take 16-bit operands; v is fp32 and is handed on as two bf16 terms where the output is bf16 (error 2^-17 of v, the output's rounding is
// 2^-9) and as three where it is fp32.  fp32 operands are three terms each, six products.  The instruction cuts off what it adds to a long sum: in tiles of 16 rows sums of 32
// products are added up in fp32; in tiles of 128 K / 16 additions are cut off (numbers of one sign, K of 2048 in one share: 5e-6 of the sum; 2e-7 the other way).
// Fragments are 16-byte pieces of the operands' rows: the k index is permuted alike in both factors, and four column tiles are interleaved so that a thread
// holds eight neighbouring outputs.
//
// What bounds it: for decoded tokens a chain of trips to memory (one row beside 2048 x 2560 columns 8 us, 64 requests of 20 adapters 10); for prompts how long a CTA takes from one block
// of columns to the next (6516 rows of 7 adapters beside 2048 x 2560 columns, rank 3 x 64: 44 us, 42 in a row of launches, 27 of them in ten blocks, 7 in the share of K, 6 in the join; 35 without y and out, 93 MB
// in all: 2.1 TB/s).
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 256, kWarps = 8, kMostRanks = 8, kMostShared = 220 * 1024, kTwoShared = 110 * 1024;  // (a CTA's; of two on an SM)

PG_DEVINL uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// eight elements as one to three bf16 terms (the sum of the terms has 8 bits a term)
template <int TERMS>
PG_DEVINL void split8(const float (&f)[8], uint4 (&t)[TERMS]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = f[i];
#pragma unroll
  for (int k = 0; k < TERMS; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pg::pack_bf16(rest[2 * i], rest[2 * i + 1]);
      rest[2 * i] -= __uint_as_float(w[i] << 16);
      rest[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
    }
    t[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// 16 bytes where `there`, zeros else, without a branch: what is merged behind a branch is waited for there, and the loads come one after another
PG_DEVINL uint4 ld16(const void* p, bool there) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.u32 q, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@q ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(there)));
  return v;
}

// Eight elements k .. k + 7 of a row as they are; zeros from `end` on.  vec: rows start on 16-byte boundaries.
template <bool F32>
struct Raw8 {
  uint4 v[F32 ? 2 : 1];
  PG_DEVINL void load(const void* row, int k, int end, bool vec) {
    constexpr int kSize = F32 ? 4 : 2;
    const char* p = static_cast<const char*>(row) + static_cast<long long>(k) * kSize;
    const bool whole = vec && k + 8 <= end;
    v[0] = ld16(p, whole);
    if constexpr (F32) v[1] = ld16(p + 16, whole);
    if (!whole && k < end) {
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = k + i >= end ? 0u : F32 ? reinterpret_cast<const uint32_t*>(p)[i] : reinterpret_cast<const uint16_t*>(p)[i];
      if constexpr (F32) v[0] = make_uint4(h[0], h[1], h[2], h[3]), v[1] = make_uint4(h[4], h[5], h[6], h[7]);
      else v[0] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
  PG_DEVINL void terms(uint4 (&t)[F32 ? 3 : 1]) const {
    if constexpr (F32) {
      const float f[8] = {__uint_as_float(v[0].x), __uint_as_float(v[0].y), __uint_as_float(v[0].z), __uint_as_float(v[0].w),
                          __uint_as_float(v[1].x), __uint_as_float(v[1].y), __uint_as_float(v[1].z), __uint_as_float(v[1].w)};
      split8<3>(f, t);
    } else {
      t[0] = v[0];
    }
  }
};

// Where elements k .. k + 7 of row n of an adapter's a lie: bf16 in blocks of 64 k's, 128-byte rows whose 16-byte pieces are exchanged by the row's last bits (the matrix unit's operand
// layout: a block is copied as it is); fp32 row by row.
template <bool F32>
PG_DEVINL const char* down_at(const char* a, int rows16, int K8, int n, int k) {
  if constexpr (F32) return a + (static_cast<long long>(n) * K8 + k) * 4;
  else return a + (static_cast<long long>(k / 64) * rows16 + n) * 128 + ((k / 8 % 8 ^ (n & 7)) * 16);
}
template <bool F32>
PG_DEVINL long long down_bytes(int R, int K) {
  return F32 ? static_cast<long long>(R) * ((K + 7) / 8 * 8) * 4 : static_cast<long long>((R + 15) / 16 * 16) * ((K + 63) / 64) * 128;
}

// d += (rows g and g + 8: 32 k's) x (column g: 32 k's)
PG_DEVINL void mma32(float (&d)[4], const uint4& lo, const uint4& hi, const uint4& b) {
  const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
  pg::mma_bf16_16816(d, a0, b.x, b.y);
  pg::mma_bf16_16816(d, a1, b.z, b.w);
}

PG_DEVINL int cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return static_cast<int>(n);
}
PG_DEVINL float4 get_f4(const float* p, int rank, int own) {  // (its own memory a CTA reads by the address that it has there)
  uint32_t there;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(p)), "r"(rank));
  there = rank == own ? pg::smem_u32(p) : there;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there));
  return v;
}

struct Layout {  // of v in shared memory
  int R, partial_ld, rank32, v_ld;
};

// The tile of a cluster: its adapter and the numbers of its rows
struct Tile {
  int who, count;
  bool none;
};
template <int M>
PG_DEVINL Tile tile_of(const PgAdapter& a, int item, int subs, int (&row_of)[M]) {
  const int* tile = a.tiles + 3 * (item / subs);
  const int skip = item % subs * M, first = tile[1] + skip;
  Tile t;
  t.who = tile[0];
  t.count = min(tile[2] - skip, M);
  t.none = t.who < 0 || t.who >= a.slots;
  if (threadIdx.x < M) {
    const int r = static_cast<int>(threadIdx.x) < t.count ? a.rows[first + threadIdx.x] : -1;
    row_of[threadIdx.x] = r < a.T ? r : -1;
  }
  __syncthreads();
  return t;
}

// Rows without an adapter: pieces of 16 bytes (or one element), four under way
template <typename U>
PG_DEVINL void copy_pieces(const PgAdapter& a, const int* row_of, int count, int rank, int ranks, int bytes, int element) {
  const int per_row = bytes / static_cast<int>(sizeof(U)), all = count * per_row;
  const int step = ranks * blockDim.x;
  for (int i0 = rank * blockDim.x + threadIdx.x; i0 < all; i0 += 4 * step) {
    U v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * step, t = i < all ? row_of[i / per_row] : -1;
      if (t >= 0) v[k] = reinterpret_cast<const U*>(static_cast<const char*>(a.y) + t * a.ldy * element)[i % per_row];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * step, t = i < all ? row_of[i / per_row] : -1;
      if (t >= 0) reinterpret_cast<U*>(static_cast<char*>(a.out) + t * a.ldo * element)[i % per_row] = v[k];
    }
  }
}
template <bool OUT32>
PG_DEVINL void copy_rows(const PgAdapter& a, const int* row_of, int count, int rank, int ranks, bool vec) {
  constexpr int kOut = OUT32 ? 4 : 2;
  if (vec && a.F * kOut % 16 == 0) copy_pieces<uint4>(a, row_of, count, rank, ranks, a.F * kOut, kOut);
  else copy_pieces<uint16_t>(a, row_of, count, rank, ranks, a.F * kOut, kOut);
}

// Eight numbers of v, the CTAs' shares added in their order, four asked for at once
PG_DEVINL void joined8(const float* from, int ranks, float (&f)[8]) {
  const int own = pg::cluster_ctarank();
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.0f;
  for (int p = 0; p < ranks; p += 4) {
    float4 v[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[k][h] = get_f4(from + 4 * h, min(p + k, ranks - 1), own);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (p + k < ranks)
#pragma unroll
        for (int h = 0; h < 2; ++h) f[4 * h] += v[k][h].x, f[4 * h + 1] += v[k][h].y, f[4 * h + 2] += v[k][h].z, f[4 * h + 3] += v[k][h].w;
  }
}

// v as bf16 terms, every part's ranks rounded up to 32
template <int M, int VT>
PG_DEVINL void join_shares(const PgAdapter& a, const Layout& lay, const float* partial, uint16_t* vt, int count, int ranks) {
  const int per_row = a.parts * lay.rank32 / 8;
  for (int i = threadIdx.x; i < M * per_row; i += kThreads) {
    const int m = i / per_row, c = i % per_row * 8, part = c / lay.rank32, r = c % lay.rank32;
    uint4 t[VT];
#pragma unroll
    for (int k = 0; k < VT; ++k) t[k] = zero4();
    if (m < count && r < a.rank) {
      float f[8];
      joined8(partial + m * lay.partial_ld + part * a.rank + r, ranks, f);
      split8<VT>(f, t);
    }
#pragma unroll
    for (int k = 0; k < VT; ++k) *reinterpret_cast<uint4*>(vt + (k * M + m) * lay.v_ld + c) = t[k];
  }
}

// Eight neighbouring outputs: y, then y + factor v.  What is not 16-byte pieces is read when it is needed: registers that a load and a branch both write are waited for where they merge.
template <bool OUT32>
struct Eight {
  uint4 y[OUT32 ? 2 : 1];
  PG_DEVINL void load(const void* base, long long at, int n, bool vec, bool there) {
    const char* p = static_cast<const char*>(base) + at * (OUT32 ? 4 : 2);
    const bool whole = there && vec && n >= 8;
    y[0] = ld16(p, whole);
    if constexpr (OUT32) y[1] = ld16(p + 16, whole);
  }
  PG_DEVINL void store(const void* from, long long from_at, void* to, long long to_at, int n, bool vec, float factor, const float (&v)[8]) const {
    if constexpr (OUT32) {
      float* p = static_cast<float*>(to) + to_at;
      if (vec && n >= 8) {
        const uint32_t w[8] = {y[0].x, y[0].y, y[0].z, y[0].w, y[1].x, y[1].y, y[1].z, y[1].w};
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = fmaf(factor, v[k], __uint_as_float(w[k]));
        reinterpret_cast<float4*>(p)[0] = make_float4(o[0], o[1], o[2], o[3]), reinterpret_cast<float4*>(p)[1] = make_float4(o[4], o[5], o[6], o[7]);
      } else {
        const float* q = static_cast<const float*>(from) + from_at;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) p[k] = fmaf(factor, v[k], q[k]);
      }
    } else {
      uint16_t* p = static_cast<uint16_t*>(to) + to_at;
      if (vec && n >= 8) {
        const uint32_t w[4] = {y[0].x, y[0].y, y[0].z, y[0].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          o[k] = pg::pack_bf16(fmaf(factor, v[2 * k], __uint_as_float(w[k] << 16)), fmaf(factor, v[2 * k + 1], __uint_as_float(w[k] & 0xffff0000u)));
        *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
        const uint16_t* q = static_cast<const uint16_t*>(from) + from_at;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) p[k] = static_cast<uint16_t>(pg::pack_bf16(fmaf(factor, v[k], __uint_as_float(static_cast<uint32_t>(q[k]) << 16)), 0.0f));
      }
    }
  }
};

// out = y + B v of 16 rows: units of 32 columns, a warp each.  A unit's part of B (two runs of 32 ranks at once) and of y are asked for before they are needed, the first unit's while v
// is still made (`start`).
template <bool IN32, bool OUT32>
struct Columns {
  static constexpr int M = 16, XT = IN32 ? 3 : 1, VT = IN32 || OUT32 ? 3 : 2, KC = IN32 ? 1 : 2;
  const PgAdapter& a;
  const Layout& lay;
  const int* row_of;
  int who, stride, u, part = 0, col = 0, unit0 = 0, f0 = 0, wide = 0, g, q;
  bool vec;
  Raw8<IN32> bf[KC][4];
  Eight<OUT32> y[2];

  PG_DEVINL Columns(const PgAdapter& a_, const Layout& lay_, const int* row_of_, int who_, int rank, int ranks, bool vec_)
      : a(a_), lay(lay_), row_of(row_of_), who(who_), stride(ranks * kWarps), u(rank * kWarps + threadIdx.x / 32), g(threadIdx.x % 32 / 4), q(threadIdx.x % 4), vec(vec_) {}
  PG_DEVINL bool find() {  // the part that holds the unit, its first column
    while (part < a.parts && u - unit0 >= (a.part_cols[part] + 31) / 32) {
      unit0 += (a.part_cols[part] + 31) / 32;
      col += a.part_cols[part];
      ++part;
    }
    if (part >= a.parts) return false;
    f0 = col + 32 * (u - unit0), wide = min(32, col + a.part_cols[part] - f0);
    return true;
  }
  PG_DEVINL void ask_b(int r0) {
    constexpr int kIn = IN32 ? 4 : 2;
    const char* B = static_cast<const char*>(a.b) + static_cast<long long>(who) * a.F * a.rank * kIn;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int f = g / 2 * 8 + 2 * j + g % 2, r = r0 + 32 * c + 8 * q;
        bf[c][j].load(B + static_cast<long long>(f0 + f) * a.rank * kIn, r, f < wide ? a.rank : 0, true);
      }
  }
  PG_DEVINL void ask_y() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = row_of[8 * h + g];
      y[h].load(a.y, t * a.ldy + f0 + 8 * q, wide - 8 * q, vec, t >= 0 && 8 * q < wide);
    }
  }
  PG_DEVINL void start() {
    if (find()) ask_b(0), ask_y();
  }
  PG_DEVINL void run(const uint16_t* vt) {
    const float factor = a.gain * a.scale[who];
    for (bool first = true; find(); u += stride, first = false) {
      if (!first) ask_b(0), ask_y();
      float acc[4][4] = {};
      for (int r0 = 0; r0 < lay.rank32; r0 += 32 * KC) {
        if (r0 > 0) ask_b(r0);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if (r0 + 32 * c >= lay.rank32) break;
          const uint16_t* from = vt + g * lay.v_ld + part * lay.rank32 + r0 + 32 * c + 8 * q;
          uint4 lo[VT], hi[VT];
#pragma unroll
          for (int k = 0; k < VT; ++k) {
            lo[k] = *reinterpret_cast<const uint4*>(from + k * M * lay.v_ld);
            hi[k] = *reinterpret_cast<const uint4*>(from + (k * M + 8) * lay.v_ld);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 b[XT];
            bf[c][j].terms(b);
#pragma unroll
            for (int k = VT - 1; k >= 0; --k)
#pragma unroll
              for (int i = (IN32 ? VT - 1 - k : 0); i >= 0; --i) mma32(acc[j], lo[k], hi[k], b[i]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = row_of[8 * h + g];
        if (t < 0 || 8 * q >= wide) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = acc[j][2 * h], v[2 * j + 1] = acc[j][2 * h + 1];
        y[h].store(a.y, t * a.ldy + f0 + 8 * q, a.out, t * a.ldo + f0 + 8 * q, wide - 8 * q, vec, factor, v);
      }
    }
  }
};

// Tiles of 16 rows, any type and alignment: operands come straight from global memory as fragments.  NW: column tiles of 8 that a warp holds in the first product.
template <int NW, bool IN32, bool OUT32>
__global__ void __launch_bounds__(kThreads, 2) adapter_rows_kernel(const PgAdapter a, const Layout lay, int subs, int x_vec, int y_vec) {
  constexpr int M = 16, XT = IN32 ? 3 : 1, VT = IN32 || OUT32 ? 3 : 2, kIn = IN32 ? 4 : 2;
  extern __shared__ __align__(16) char raw[];
  __shared__ int row_of[M];
  const int ranks = cluster_size(), rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, q = lane % 4;
  const Tile tile = tile_of<M>(a, item, subs, row_of);
  pg::griddep_wait();  // (CTAs without work as well: the kernel behind counts on this one's end; the plan comes from the host, ahead of the step)
  if (tile.count <= 0 || (tile.none && a.out == a.y)) return;  // (the whole cluster)
  if (tile.none) return copy_rows<OUT32>(a, row_of, tile.count, rank, ranks, y_vec);
  const int R = lay.R, K8 = (a.K + 7) / 8 * 8, tiles8 = R / 8;
  int wn = 1;  // warps share out columns first, then K
  while (wn < kWarps && wn * NW < tiles8) wn *= 2;
  const int wk = kWarps / wn, kg = warp / wn;
  float* partial = reinterpret_cast<float*>(raw);                                                // [wk][M][partial_ld]
  uint16_t* vt = reinterpret_cast<uint16_t*>(raw + sizeof(float) * wk * M * lay.partial_ld);     // [VT][M][v_ld]
  Columns<IN32, OUT32> columns(a, lay, row_of, tile.who, rank, ranks, y_vec);
  columns.start();
  {
    const int steps = (a.K + 31) / 32, per = (steps + ranks - 1) / ranks, s0 = min(rank * per, steps), s1 = min(s0 + per, steps);
    const char* A = static_cast<const char*>(a.a) + tile.who * down_bytes<IN32>(R, a.K);
    const int rows16 = (R + 15) / 16 * 16;
    const char* xrow[2];
    int x_end[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = row_of[8 * h + g];
      xrow[h] = static_cast<const char*>(a.x) + max(t, 0) * a.ldx * kIn;
      x_end[h] = t >= 0 ? a.K : 0;
    }
    for (int base = 0; base < tiles8; base += wn * NW) {
      const int n0 = base + warp % wn * NW;
      float sum[NW][4] = {};
      for (int s = s0 + kg; s < s1; s += wk) {
        const int k = 32 * s + 8 * q;
        Raw8<IN32> xr[2], ar[NW];
#pragma unroll
        for (int h = 0; h < 2; ++h) xr[h].load(xrow[h], k, x_end[h], x_vec);
#pragma unroll
        for (int j = 0; j < NW; ++j) ar[j].load(down_at<IN32>(A, rows16, K8, (n0 + j) * 8 + g, k), 0, n0 + j < tiles8 && k < K8 ? 8 : 0, true);
        uint4 xf[2][XT];
        xr[0].terms(xf[0]), xr[1].terms(xf[1]);
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          uint4 af[XT];
          ar[j].terms(af);
          float d[4] = {};
#pragma unroll
          for (int o = XT - 1; o >= 0; --o)  // the smallest products first
#pragma unroll
            for (int i = 0; i <= o; ++i) mma32(d, xf[0][i], xf[1][i], af[o - i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[j][i] += d[i];
        }
      }
#pragma unroll
      for (int j = 0; j < NW; ++j)
        if (n0 + j < tiles8)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(partial + (kg * M + 8 * h + g) * lay.partial_ld + (n0 + j) * 8 + 2 * q) = make_float2(sum[j][2 * h], sum[j][2 * h + 1]);
    }
  }
  if (wk > 1) {  // the warps that share K, in their order
    __syncthreads();
    for (int i = tid; i < tile.count * (R / 4); i += kThreads) {
      float4* p = reinterpret_cast<float4*>(partial + i / (R / 4) * lay.partial_ld) + i % (R / 4);
      float4 v = *p;
      for (int w = 1; w < wk; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + w * M * lay.partial_ld);
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      *p = v;
    }
  }
  pg::cluster_sync_all();
  join_shares<M, VT>(a, lay, partial, vt, tile.count, ranks);
  pg::cluster_arrive();
  __syncthreads();
  columns.run(vt);
  pg::cluster_wait();  // nobody leaves while its share is read
}

// Tiles of 128 bf16 rows, both products on the tensor cores with their sums in tensor memory.
//   v = x A^T        x and A come in stages of 64 k's by asynchronous copies, 128-byte rows whose 16-byte pieces are exchanged by the row's last bits; N = ranks of all parts, up to 256
//   shares of K      added over the cluster by way of L2 (through distributed shared memory a CTA read 6 bytes a clock: 18,000 clocks for 192 columns of v, 11,000 this way, half of
//                    them until all shares are written), as bf16 terms into shared memory (operand layout, 64 ranks a block of 16 KB)
//   B v              blocks of 128 columns: every term times the same rows of B, a block ahead of the one whose sums leave; y is asked for a block ahead as well; sums leave through
//                    shared memory so that lanes read and write neighbouring pieces of y and out
// 256 columns of tensor memory for v, two times 128 for the blocks: one CTA an SM.
// A warp of its own issues the products: it waits where operands are not there yet, the others do not wait for it.  Stages are asked for three chunks ahead of five, so that the one
// that is filled was read two products ago.
constexpr int kWorkers = 512, kWorkerWarps = kWorkers / 32, kTensorThreads = kWorkers + 32, kCols = 32;  // columns of a block that a warp takes, beside three others with the same rows
constexpr int kStages = 5, kRows = 128, kBlock = 128, kStageLd = kCols + 4;                          // (+ 4: lanes' rows lie in different banks)
constexpr int kFull = 0, kEmpty = kStages, kShare = 2 * kStages, kThere = kShare + 1, kDone = kThere + 2, kLeft = kDone + 2, kBars = kLeft + 2;  // barriers: stages, v, blocks
struct Plan {                                                       // of shared memory
  int R16, stages, stage_bytes, v_at, blocks64, smem;               // v: [parts][blocks of 64 ranks][terms] operands of 16 KB
};

struct Blocks {  // of 128 columns, of all parts
  const PgAdapter& a;
  struct Block {
    int part, f0, wide, left;  // left: of the part, this block among them
  };
  PG_DEVINL Block at(int u) const { return next(Block{0, 0, 1, a.part_cols[0]}, u); }
  PG_DEVINL Block next(Block b, int u) const {  // u blocks on; wide 0: there is none
    if (b.wide == 0) return b;
    for (;;) {
      const int here = (b.left + kBlock - 1) / kBlock;
      if (u < here) break;
      u -= here;
      b.f0 += b.left;
      if (++b.part >= a.parts) {
        b.wide = 0;
        return b;
      }
      b.left = a.part_cols[b.part];
    }
    b.f0 += kBlock * u, b.left -= kBlock * u;
    b.wide = min(kBlock, b.left);
    return b;
  }
};

template <bool OUT32>
__global__ void __launch_bounds__(kTensorThreads, 1) adapter_tensor_kernel(const PgAdapter a, const Layout lay, const Plan plan, int y_vec) {
  constexpr int VT = OUT32 ? 3 : 2;
  extern __shared__ char raw_unaligned[];
  __shared__ int row_of[kRows];
  __shared__ __align__(8) uint64_t bars[kBars];
  __shared__ uint32_t tmem_at;
  char* raw = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  const int ranks = cluster_size(), rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const Tile tile = tile_of<kRows>(a, item, 1, row_of);
  pg::griddep_wait();
  if (tile.count <= 0 || (tile.none && a.out == a.y)) return;  // (the whole cluster)
  if (tile.none) return copy_rows<OUT32>(a, row_of, tile.count, rank, ranks, y_vec);
  const uint32_t base = pg::smem_u32(raw), bar0 = pg::smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8 * i; };
  if (warp == 0) {
    pg::tmem_alloc(pg::smem_u32(&tmem_at), 512);
    pg::tmem_relinquish();
  }
  if (tid == kWorkers) {
    for (int i = 0; i < kStages; ++i) pg::mbar_init(bar(kFull + i), kWorkerWarps + 1), pg::mbar_init(bar(kEmpty + i), 1);
    pg::mbar_init(bar(kShare), 1);
    for (int i = 0; i < 2; ++i) pg::mbar_init(bar(kThere + i), kWorkerWarps), pg::mbar_init(bar(kDone + i), 1), pg::mbar_init(bar(kLeft + i), kWorkerWarps);
    pg::mbar_fence_init();
  }
  pg::tc_fence_before();
  __syncthreads();
  pg::tc_fence_after();
  const uint32_t tmem = tmem_at;
  const int R = lay.R, k16 = (a.rank + 15) / 16, b_bytes = plan.blocks64 * kBlock * 128;
  const int all = (a.K + 63) / 64, per = (all + ranks - 1) / ranks, c0 = min(rank * per, all), chunks = min(per, all - c0);  // this CTA's share of K
  const Blocks blocks{a};

  if (warp == kWorkerWarps) {
    // ---- products: v = x A^T into columns 0 .. R of tensor memory, then B v by blocks into 256 .. 383 and 384 .. 511 ----------
    const uint32_t down = pg::make_idesc_bf16(kRows, plan.R16);
    constexpr uint32_t up = pg::make_idesc_bf16(kRows, kBlock);
    if (lane == 0) {
      // (one thread's instructions come one after another, ten clocks each: no divisions here)
      const uint64_t x0 = pg::make_sdesc_k_sw128(base);
      uint64_t x = x0;
      uint32_t phase = 0;
      for (int i = 0, stage = 0; i < chunks; ++i) {
        pg::mbar_wait(bar(kFull + stage), phase);
        pg::tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) pg::umma_f16(tmem, x + 2 * k, x + (kRows * 128 >> 4) + 2 * k, down, i > 0 || k > 0);
        pg::umma_commit(bar(kEmpty + stage));
        x += plan.stage_bytes >> 4;
        if (++stage == plan.stages) stage = 0, phase ^= 1, x = x0;
      }
      if (chunks > 0) pg::umma_commit(bar(kShare));
    }
    __syncwarp();
    if (ranks > 1) pg::cluster_sync_all();
    __syncthreads();  // (v's terms are there)
    if (lane == 0) {
      pg::tc_fence_after();
      const uint64_t v0 = pg::make_sdesc_k_sw128(base + plan.v_at), w0 = pg::make_sdesc_k_sw128(base);
      const int v_part = plan.blocks64 * VT * (kRows * 128 >> 4);
      Blocks::Block b = blocks.at(rank);
      for (int at = 0; b.wide > 0; ++at) {
        const int turn = at & 1, phase = at >> 1 & 1;
        const uint32_t to = tmem + 256 + kBlock * turn;
        uint64_t v = v0 + b.part * v_part, w = w0 + turn * (b_bytes >> 4);
        b = blocks.next(b, ranks);
        pg::mbar_wait(bar(kThere + turn), phase);
        if (at >= 2) pg::mbar_wait(bar(kLeft + turn), phase ^ 1);  // (what stood there has been read)
        pg::tc_fence_after();
        bool more = false;
        for (int left = k16; left > 0; left -= 4) {  // 64 ranks; the smallest term first within them
#pragma unroll
          for (int k = VT - 1; k >= 0; --k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < left) {
                pg::umma_f16(to, v + k * (kRows * 128 >> 4) + 2 * i, w + 2 * i, up, more);
                more = true;
              }
          v += VT * (kRows * 128 >> 4), w += kBlock * 128 >> 4;
        }
        pg::umma_commit(bar(kDone + turn));
      }
    }
    __syncwarp();
  } else {
    auto arrive = [&](int i) {  // of a warp
      __syncwarp();
      if (lane == 0) pg::mbar_arrive(bar(i));
    };
    {
      const char* A = static_cast<const char*>(a.a) + tile.who * down_bytes<false>(R, a.K);
      const int down_block = plan.R16 * 128, row0 = tid / 8, piece = tid % 8;  // a thread's piece of rows row0 and row0 + 64
      const char* from[2];
      uint32_t to[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + 64 * i, t = row_of[row];
        from[i] = t >= 0 ? static_cast<const char*>(a.x) + (t * a.ldx + 64LL * c0 + 8 * piece) * 2 : nullptr;
        to[i] = base + row * 128 + ((piece ^ (row & 7)) * 16);
      }
      int asked = 0, stage = 0;  // the next chunk and its stage
      uint32_t phase = 1;        // (of the round before: the first passes)
      auto ask = [&]() {
        if (asked < chunks) {
          const uint32_t at = stage * plan.stage_bytes;
          if (asked >= plan.stages) pg::mbar_wait(bar(kEmpty + stage), phase);
          if (tid == 0) {
            pg::mbar_expect_tx(bar(kFull + stage), down_block);
            pg::bulk_copy_g2s(base + at + kRows * 128, A + static_cast<long long>(c0 + asked) * down_block, down_block, bar(kFull + stage));
          }
          const bool in = 64 * (c0 + asked) + 8 * piece < a.K;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool there = in && from[r] != nullptr;
            pg::cp_async16(to[r] + at, there ? from[r] : static_cast<const char*>(a.x), there);
            if (from[r] != nullptr) from[r] += 128;
          }
          ++asked;
          if (++stage == plan.stages) stage = 0, phase ^= 1;
        }
        pg::cp_async_commit();
      };
      const int ahead = plan.stages - 2;
      for (int i = 0; i < ahead; ++i) ask();
      for (int i = 0, full = 0; i < chunks; ++i) {
        ask();
        if (ahead == 3) pg::cp_async_wait<3>();
        else if (ahead == 2) pg::cp_async_wait<2>();
        else pg::cp_async_wait<1>();
        pg::fence_proxy_async_smem();
        arrive(kFull + full);
        if (++full == plan.stages) full = 0;
      }
      if (chunks > 0) pg::mbar_wait(bar(kShare), 0);
      __syncwarp();
      pg::tc_fence_after();
      pg::cp_async_wait<0>();
    }
    // ---- the shares of v together ------------------------------------------------------------------------------------------
    const int quarter = warp % 4, group = warp / 4, m = 32 * quarter + lane;  // a warp reads 32 lanes of tensor memory; four warps share them
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    const long long share = static_cast<long long>(R) * kRows;
    float* shares = a.shares + item * share * ranks;  // [ranks][R / 4][rows][4]
    if (ranks > 1) {
      for (int c = 16 * group; c < R; c += 64) {
        uint32_t v[16] = {};
        if (chunks > 0) {
          pg::tmem_ld16(lanes + c, v);
          pg::tmem_ld_wait();
        }
        uint4* to = reinterpret_cast<uint4*>(shares + rank * share) + c / 4 * kRows + m;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + 4 * i < R) to[i * kRows] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      pg::cluster_sync_all();
    } else {
      asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");  // (nobody writes v's terms while a stage is still read)
    }
    const int per_row = a.parts * plan.blocks64 * 8;
    constexpr int N = 3;  // pieces at once
    for (int first = group; first < per_row; first += 4 * N) {
      float f[N][8], own[N][8];
      int at[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int q = (first + 4 * n) >> 3, part = plan.blocks64 == 1 ? q : q >> 1, r = (plan.blocks64 == 1 ? 0 : (q & 1) * 64) + ((first + 4 * n) & 7) * 8;
        at[n] = first + 4 * n < per_row && r < a.rank ? part * a.rank + r : -1;  // (the same in a whole warp)
        uint32_t v[16] = {};
        if (chunks > 0 && at[n] >= 0) {
          pg::tmem_ld8(lanes + at[n], v);
          pg::tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) f[n][i] = 0.0f, own[n][i] = __uint_as_float(v[i]);
      }
      for (int p = 0; p < ranks; ++p) {  // (the ranks' order, whoever adds)
        float4 v[N][2];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float* from = shares + p * share + (static_cast<long long>(max(at[n], 0)) / 4 * kRows + m) * 4;
          const bool there = p != rank && at[n] >= 0;
          const uint4 lo = ld16(from, there), hi = ld16(from + 4 * kRows, there);
          v[n][0] = make_float4(__uint_as_float(lo.x), __uint_as_float(lo.y), __uint_as_float(lo.z), __uint_as_float(lo.w));
          v[n][1] = make_float4(__uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w));
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (p == rank) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[n][i] += own[n][i];
          } else {
            f[n][0] += v[n][0].x, f[n][1] += v[n][0].y, f[n][2] += v[n][0].z, f[n][3] += v[n][0].w, f[n][4] += v[n][1].x, f[n][5] += v[n][1].y, f[n][6] += v[n][1].z, f[n][7] += v[n][1].w;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = first + 4 * n;
        if (c >= per_row) break;
        uint4 terms[VT];
        split8<VT>(f[n], terms);
        char* to = raw + plan.v_at + (c >> 3) * VT * (kRows * 128) + m * 128 + (((c & 7) ^ (m & 7)) * 16);
#pragma unroll
        for (int k = 0; k < VT; ++k) *reinterpret_cast<uint4*>(to + k * (kRows * 128)) = m < tile.count && at[n] >= 0 ? terms[k] : zero4();
      }
    }
    pg::fence_proxy_async_smem();
    pg::tc_fence_before();
    __syncthreads();
    pg::tc_fence_after();

    // ---- out = y + B v: blocks of 128 columns ------------------------------------------------------------------------------
    const char* B = static_cast<const char*>(a.b) + static_cast<long long>(tile.who) * a.F * a.rank * 2;
    const float factor = a.gain * a.scale[tile.who];
    float* stage = reinterpret_cast<float*>(raw + 2 * b_bytes) + warp * 32 * kStageLd;
    const int c = kCols * group + lane % 4 * 8;  // the first of a lane's columns of a block; four lanes a row
    int row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = row_of[32 * quarter + 8 * i + lane / 4];
    auto ask_b = [&](const Blocks::Block& b, int turn) {
      if (b.wide > 0)
        for (int q = 0; q < plan.blocks64; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = tid / 8 + 64 * i, piece = tid % 8, r = 64 * q + 8 * piece;
            const bool there = n < b.wide && r < a.rank;
            if (piece < 2 * k16 - 8 * q)  // (what the product reads)
              pg::cp_async16(base + turn * b_bytes + q * (kBlock * 128) + n * 128 + ((piece ^ (n & 7)) * 16), B + (there ? static_cast<long long>(b.f0 + n) * a.rank + r : 0) * 2, there);
          }
      pg::cp_async_commit();
    };
    auto ask_y = [&](const Blocks::Block& b, Eight<OUT32> (&y)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i].load(a.y, row[i] * a.ldy + b.f0 + c, b.wide - c, y_vec, row[i] >= 0 && c < b.wide);
    };
    Eight<OUT32> y[2][4];
    Blocks::Block b[2];
    b[0] = blocks.at(rank), b[1] = blocks.next(b[0], ranks);
    ask_b(b[0], 0);
    ask_b(b[1], 1);
    ask_y(b[0], y[0]);
    pg::cp_async_wait<1>();
    pg::fence_proxy_async_smem();
    arrive(kThere);
    pg::cp_async_wait<0>();
    pg::fence_proxy_async_smem();
    arrive(kThere + 1);
    for (int at = 0; b[0].wide > 0; at += 2) {
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        if (b[turn].wide <= 0) break;
        const Blocks::Block now = b[turn];
        ask_y(b[turn ^ 1], y[turn ^ 1]);
        b[turn] = blocks.next(b[turn ^ 1], ranks);
        pg::mbar_wait(bar(kDone + turn), at / 2 % 2);
        __syncwarp();
        pg::tc_fence_after();
        ask_b(b[turn], turn);
        {
          uint32_t v[kCols / 16][16];
#pragma unroll
          for (int i = 0; i < kCols / 16; ++i) pg::tmem_ld16(lanes + 256 + kBlock * turn + kCols * group + 16 * i, v[i]);
          pg::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < kCols / 4; ++j)
            *reinterpret_cast<uint4*>(stage + lane * kStageLd + 4 * j) = make_uint4(v[j / 4][4 * (j % 4)], v[j / 4][4 * (j % 4) + 1], v[j / 4][4 * (j % 4) + 2], v[j / 4][4 * (j % 4) + 3]);
        }
        pg::tc_fence_before();
        arrive(kLeft + turn);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* from = stage + (8 * i + lane / 4) * kStageLd + lane % 4 * 8;
          const float4 lo = *reinterpret_cast<const float4*>(from), hi = *reinterpret_cast<const float4*>(from + 4);
          const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          if (row[i] >= 0 && c < now.wide) y[turn][i].store(a.y, row[i] * a.ldy + now.f0 + c, a.out, row[i] * a.ldo + now.f0 + c, now.wide - c, y_vec, factor, v);
        }
        pg::cp_async_wait<0>();
        pg::fence_proxy_async_smem();
        arrive(kThere + turn);
      }
    }
  }
  pg::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    pg::tc_fence_after();
    pg::tmem_dealloc(tmem, 512);
  }
}

template <typename Kern>
bool allow_shared(Kern kern, bool (&configured)[pg::kMaxDevices]) {
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    done = true;
  }
  return true;
}
struct Config {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  Config(long long ctas, int ranks, int threads, size_t smem, cudaStream_t st) {
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pg_pdl_enabled() ? 2 : 1;
  }
};
template <typename Kern, typename... Args>
int launch(Kern kern, long long items, int ranks, int threads, size_t smem, cudaStream_t st, Args... args) {
  if (smem > kMostShared || items * ranks > 0x7fffffff) return PG_ERR_ARG;
  const Config c(items * ranks, ranks, threads, smem, st);
  pg_count_launch(1);
  return cudaLaunchKernelEx(&c.cfg, kern, args...) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
// How many clusters of `ranks` CTAs run at once: fewer than SMs / ranks, since a cluster lies in one part of the device (asked once; `known` is the kernel's)
template <typename Kern>
int at_once(Kern kern, int (&known)[pg::kMaxDevices][kMostRanks + 1], int ranks, int threads, size_t smem) {
  int& n = known[pg::current_device()][ranks];
  if (n == 0) {
    Config c(ranks, ranks, threads, smem, nullptr);
    c.cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &c.cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
  }
  return n;
}

Layout layout_of(const PgAdapter& a) {
  Layout lay;
  lay.R = a.parts * a.rank;
  lay.partial_ld = lay.R + 4;
  lay.rank32 = (a.rank + 31) / 32 * 32;
  lay.v_ld = a.parts * lay.rank32;
  lay.v_ld += (lay.v_ld % 64 == 32) ? 0 : 32;  // eight lanes' 16-byte pieces of two rows lie in different banks
  return lay;
}
// Shared memory of a tile of 128 rows; no stages: it does not go over the tensor memory (few rows of an adapter, more than 256 columns of v, no room for its terms: every run takes blocks of 64
// ranks, so that four runs do not fit at any rank.  6432 rows of 7 adapters, K 2048, rank 64: three runs of 2560 columns 44 us, four of 4608 in tiles of 16 180)
template <int VT>
void plan_of(const PgAdapter& a, const Layout& lay, Plan& plan) {
  plan.R16 = (lay.R + 15) / 16 * 16;
  plan.stage_bytes = (kRows + plan.R16) * 128;
  plan.blocks64 = (a.rank + 63) / 64;
  const int v_bytes = a.parts * plan.blocks64 * VT * kRows * 128;
  const int leave = 2 * plan.blocks64 * kBlock * 128 + static_cast<int>(sizeof(float)) * kWorkerWarps * 32 * kStageLd;  // B's blocks and the sums that leave, in front of v's terms
  plan.v_at = (leave + 1023) / 1024 * 1024;
  plan.stages = kStages;
  while (plan.stages * plan.stage_bytes + 1024 > kMostShared) --plan.stages;
  const int behind = plan.v_at + v_bytes, stages = plan.stages * plan.stage_bytes;
  plan.smem = (stages > behind ? stages : behind) + 1024;
  if (a.tile_rows != kRows || a.in_f32 || plan.R16 > 256 || plan.smem > kMostShared) plan.stages = 0;
}
// Shares of K and of the columns, a CTA each: as many as leave all clusters of the launch room at once.  (16 tiles of 2048 x 2560 with as many as fit and with 8: 24 and 43 us.)
template <bool OUT32>
int shares_of(const PgAdapter& a) {
  static bool configured[pg::kMaxDevices] = {};
  static int known[pg::kMaxDevices][kMostRanks + 1] = {};
  if (!allow_shared(adapter_tensor_kernel<OUT32>, configured)) return 0;
  int ranks = kMostRanks;
  while (ranks > 1 && (a.K / ranks < 128 || at_once(adapter_tensor_kernel<OUT32>, known, ranks, kTensorThreads, kMostShared) < a.tile_count)) --ranks;
  return ranks;
}

template <bool IN32, bool OUT32>
int pick(const PgAdapter& a, cudaStream_t st, int x_vec, int y_vec) {
  constexpr int VT = IN32 || OUT32 ? 3 : 2, NW = IN32 ? 2 : 6;  // (fp32: three terms of every fragment)
  const Layout lay = layout_of(a);
  if constexpr (!IN32) {
    Plan plan;
    plan_of<VT>(a, lay, plan);
    if (plan.stages > 0 && x_vec && a.K % 8 == 0) {
      const int ranks = shares_of<OUT32>(a);
      if (ranks < 1) return PG_ERR_CUDA;
      if (ranks > 1 && a.shares == nullptr) return PG_ERR_ARG;
      return launch(adapter_tensor_kernel<OUT32>, a.tile_count, ranks, kTensorThreads, plan.smem, st, a, lay, plan, y_vec);
    }
  }
  auto kern = adapter_rows_kernel<NW, IN32, OUT32>;
  static bool configured[pg::kMaxDevices] = {};
  static int known[2][pg::kMaxDevices][kMostRanks + 1] = {};  // two CTAs an SM, one
  if (!allow_shared(kern, configured)) return PG_ERR_CUDA;
  const int subs = a.tile_rows / 16;
  const long long items = static_cast<long long>(a.tile_count) * subs;
  int ranks = 1, wn = 1;
  while (wn < kWarps && wn * NW < lay.R / 8) wn *= 2;
  const size_t smem = sizeof(float) * (kWarps / wn) * 16 * lay.partial_ld + sizeof(uint16_t) * VT * 16 * lay.v_ld;
  const bool two = smem <= kTwoShared;
  // A share is read by all CTAs of its cluster: eight for few tiles alone.  (2048 x 2560, us with 2, 4, 8: rank 3 x 64, 8 tiles 21, 14, 13, 16 tiles 22, 16, 26; rank 3 x 16, 8 tiles 12,
  // 8.8, 7.9, 32 tiles 13, 10, 13.)
  const int most = items <= pg::num_sms() / 16 ? kMostRanks : kMostRanks / 2;
  while (ranks < most && a.K / (ranks * 2) >= 128 && at_once(kern, known[!two], ranks * 2, kThreads, two ? kTwoShared : kMostShared) >= items) ranks *= 2;
  return launch(kern, items, ranks, kThreads, smem, st, a, lay, subs, x_vec, y_vec);
}

}  // namespace

extern "C" long long pg_adapter_scratch(const PgAdapter* args) {
  if (args == nullptr || args->parts < 1 || args->parts > 8 || args->rank < 8 || args->rank > 128 || args->tile_count < 1 || args->K < 1) return 0;
  Plan plan;
  if (args->out_f32) plan_of<3>(*args, layout_of(*args), plan);
  else plan_of<2>(*args, layout_of(*args), plan);
  const int ranks = plan.stages == 0 ? 1 : args->out_f32 ? shares_of<true>(*args) : shares_of<false>(*args);
  return ranks > 1 ? static_cast<long long>(sizeof(float)) * args->tile_count * ranks * kRows * args->parts * args->rank : 0;
}

extern "C" int pg_adapter_add(const PgAdapter* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgAdapter& a = *args;
  if (a.x == nullptr || a.y == nullptr || a.out == nullptr || a.a == nullptr || a.b == nullptr || a.scale == nullptr || a.rows == nullptr || a.tiles == nullptr || a.parts < 1 ||
      a.parts > 8 || a.K < 1 || a.rank < 8 || a.rank > 128 || a.rank % 8 || a.slots < 1 || a.tile_count < 1 || (a.tile_rows != 16 && a.tile_rows != 128) || a.T < 1 || a.ldx < a.K ||
      a.ldy < a.F || a.ldo < a.F || (a.in_f32 && !a.out_f32) || ((reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b)) & 15))
    return PG_ERR_ARG;
  long long cols = 0;
  for (int i = 0; i < a.parts; ++i) {
    if (a.part_cols[i] < 1) return PG_ERR_ARG;
    cols += a.part_cols[i];
  }
  if (cols != a.F) return PG_ERR_ARG;
  const int in = a.in_f32 ? 4 : 2, out = a.out_f32 ? 4 : 2;
  const int x_vec = ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx) * in) & 15) == 0;
  int y_vec = ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldy) * out | static_cast<uintptr_t>(a.ldo) * out) & 15) == 0;
  for (int i = 0; i < a.parts - 1; ++i) y_vec = y_vec && a.part_cols[i] * out % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.in_f32) return pick<true, true>(a, st, x_vec, y_vec);
  return a.out_f32 ? pick<false, true>(a, st, x_vec, y_vec) : pick<false, false>(a, st, x_vec, y_vec);
}
