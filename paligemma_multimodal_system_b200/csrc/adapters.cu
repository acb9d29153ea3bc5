// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + gain scale[s] B_s (A_s x[t]) for the rows t of adapter s.
//
// A tile is up to 16 or 64 rows of one adapter, gathered by number, so decoded tokens of requests that share an adapter and the rows of a prompt are one thing.  A
// cluster of CTAs takes a tile in one launch: each CTA multiplies a share of K (v = A x, rank columns), the shares are added through distributed shared memory in
// a fixed order, and each CTA then makes a share of the columns (B v) and adds it to y.  v stays in shared memory.
//
// Matrix instructions take 16-bit operands; v is fp32 and is handed on as two bf16 terms where the output is bf16 (error 2^-17 of v, the output's rounding is
// 2^-9) and as three where it is fp32.  fp32 operands are three terms each, six products.  The instruction cuts off what it adds to a long sum: sums of 64
// products are added up in fp32.
// Fragments are 16-byte pieces of the operands' rows: the k index is permuted alike in both factors, and four column tiles are interleaved so that a thread
// holds eight neighbouring outputs.
//
// What bounds it: the bytes of y in and out and of x for prompts; the adapters' bytes and a chain of trips to memory for decoded tokens.
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 256, kWarps = 8, kMostRanks = 8, kMostShared = 220 * 1024;

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

// Eight elements k .. k + 7 of a row as bf16 terms; zeros from `end` on.  vec: 16-byte pieces start on 16-byte boundaries and `end` is a multiple of 8.
template <bool F32>
PG_DEVINL void load8(const void* row, int k, int end, bool vec, uint4 (&t)[F32 ? 3 : 1]) {
  if constexpr (F32) {
    const float* p = static_cast<const float*>(row) + k;
    float f[8];
    if (vec && k + 8 <= end) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = k + i < end ? p[i] : 0.f;
    }
    split8<3>(f, t);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(row) + k;
    if (vec && k + 8 <= end) {
      t[0] = *reinterpret_cast<const uint4*>(p);
    } else {
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = k + i < end ? p[i] : 0u;
      t[0] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
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
PG_DEVINL float4 get_f4(const float* p, int rank) {
  uint32_t there;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
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

// Rows without an adapter
template <bool OUT32>
PG_DEVINL void copy_rows(const PgAdapter& a, const int* row_of, int count, int rank, int ranks, bool vec) {
  constexpr int kOut = OUT32 ? 4 : 2;
  const int tid = threadIdx.x, bytes = a.F * kOut;
  for (int i = 0; i < count; ++i) {
    const int t = row_of[i];
    if (t < 0) continue;
    const char* from = static_cast<const char*>(a.y) + t * a.ldy * kOut;
    char* to = static_cast<char*>(a.out) + t * a.ldo * kOut;
    const int step = vec ? 16 : 2, whole = bytes / step * step;
    for (int c = (rank * kThreads + tid) * step; c < whole; c += ranks * kThreads * step) {
      if (vec) *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(from + c);
      else *reinterpret_cast<uint16_t*>(to + c) = *reinterpret_cast<const uint16_t*>(from + c);
    }
    for (int c = whole + 2 * tid; rank == 0 && c < bytes; c += 2 * kThreads) *reinterpret_cast<uint16_t*>(to + c) = *reinterpret_cast<const uint16_t*>(from + c);
  }
}

// The CTAs' shares of v (partial, [SHARES] one behind another in each) together, in a fixed order; v as bf16 terms, every part's ranks rounded up to 32
template <int M, int VT>
PG_DEVINL void join_shares(const PgAdapter& a, const Layout& lay, const float* partial, int shares, uint16_t* vt, int count, int ranks) {
  const int per_row = a.parts * lay.rank32 / 8;
  for (int i = threadIdx.x; i < M * per_row; i += kThreads) {
    const int m = i / per_row, c = i % per_row * 8, part = c / lay.rank32, r = c % lay.rank32;
    uint4 t[VT];
#pragma unroll
    for (int k = 0; k < VT; ++k) t[k] = zero4();
    if (m < count && r < a.rank) {
      float f[8] = {};
      for (int w = 0; w < shares; ++w) {
        const float* from = partial + (w * M + m) * lay.partial_ld + part * a.rank + r;
#pragma unroll 4
        for (int p = 0; p < ranks; ++p) {
          const float4 lo = get_f4(from, p), hi = get_f4(from + 4, p);
          f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w, f[4] += hi.x, f[5] += hi.y, f[6] += hi.z, f[7] += hi.w;
        }
      }
      split8<VT>(f, t);
    }
#pragma unroll
    for (int k = 0; k < VT; ++k) *reinterpret_cast<uint4*>(vt + (k * M + m) * lay.v_ld + c) = t[k];
  }
}

// Eight neighbouring outputs: y, then y + factor v
template <bool OUT32>
struct Eight {
  uint4 y[OUT32 ? 2 : 1];
  PG_DEVINL void load(const void* base, long long at, int n, bool vec) {
    if constexpr (OUT32) {
      const float* p = static_cast<const float*>(base) + at;
      if (vec && n >= 8) {
        y[0] = reinterpret_cast<const uint4*>(p)[0], y[1] = reinterpret_cast<const uint4*>(p)[1];
      } else {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = k < n ? __float_as_uint(p[k]) : 0u;
        y[0] = make_uint4(w[0], w[1], w[2], w[3]), y[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(base) + at;
      if (vec && n >= 8) {
        y[0] = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = k < n ? p[k] : 0u;
        y[0] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
    }
  }
  PG_DEVINL void store(void* base, long long at, int n, bool vec, float factor, const float (&v)[8]) const {
    if constexpr (OUT32) {
      float* p = static_cast<float*>(base) + at;
      float o[8];
      const uint32_t w[8] = {y[0].x, y[0].y, y[0].z, y[0].w, y[1].x, y[1].y, y[1].z, y[1].w};
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = fmaf(factor, v[k], __uint_as_float(w[k]));
      if (vec && n >= 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(o[0], o[1], o[2], o[3]), reinterpret_cast<float4*>(p)[1] = make_float4(o[4], o[5], o[6], o[7]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) p[k] = o[k];
      }
    } else {
      uint16_t* p = static_cast<uint16_t*>(base) + at;
      const uint32_t w[4] = {y[0].x, y[0].y, y[0].z, y[0].w};
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[k] = pg::pack_bf16(fmaf(factor, v[2 * k], __uint_as_float(w[k] << 16)), fmaf(factor, v[2 * k + 1], __uint_as_float(w[k] & 0xffff0000u)));
      if (vec && n >= 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) p[k] = static_cast<uint16_t>(o[k / 2] >> 16 * (k % 2));
      }
    }
  }
};

// out = y + B v: units of 32 columns, a warp each.  A unit's part of B and of y are asked for before they are needed: the first unit's while v is still made (`start`), and two runs of
// 32 ranks at once.
template <int MT, bool IN32, bool OUT32>
struct Columns {
  static constexpr int M = 16 * MT, XT = IN32 ? 3 : 1, VT = IN32 || OUT32 ? 3 : 2, H = MT < 2 ? MT : 2, KC = IN32 ? 1 : 2;  // H: row tiles at once
  const PgAdapter& a;
  const Layout& lay;
  const int* row_of;
  int who, stride, u, part = 0, col = 0, unit0 = 0, f0 = 0, wide = 0, g, q;
  bool vec;
  uint4 bf[KC][4][XT];
  Eight<OUT32> y[H][2];

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
#pragma unroll
        for (int i = 0; i < XT; ++i) bf[c][j][i] = zero4();
        if (f < wide && r < a.rank) load8<IN32>(B + static_cast<long long>(f0 + f) * a.rank * kIn, r, a.rank, true, bf[c][j]);
      }
  }
  PG_DEVINL void ask_y(int m0) {
#pragma unroll
    for (int m = 0; m < H; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = row_of[16 * (m0 + m) + 8 * h + g];
        if (t >= 0 && 8 * q < wide) y[m][h].load(a.y, t * a.ldy + f0 + 8 * q, wide - 8 * q, vec);
      }
  }
  PG_DEVINL void start() {
    if (find()) ask_b(0), ask_y(0);
  }
  PG_DEVINL void run(const uint16_t* vt) {
    const float factor = a.gain * a.scale[who];
    for (bool first = true; find(); u += stride, first = false) {
      if (!first) ask_b(0);
      for (int m0 = 0; m0 < MT; m0 += H) {
        if (!first || m0 > 0) ask_y(m0);
        float acc[H][4][4] = {};
        for (int r0 = 0; r0 < lay.rank32; r0 += 32 * KC) {
          if (r0 > 0 || (m0 > 0 && lay.rank32 > 32 * KC)) ask_b(r0);
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            if (r0 + 32 * c >= lay.rank32) break;
#pragma unroll
            for (int m = 0; m < H; ++m) {
              const uint16_t* from = vt + (16 * (m0 + m) + g) * lay.v_ld + part * lay.rank32 + r0 + 32 * c + 8 * q;
              uint4 lo[VT], hi[VT];
#pragma unroll
              for (int k = 0; k < VT; ++k) {
                lo[k] = *reinterpret_cast<const uint4*>(from + k * M * lay.v_ld);
                hi[k] = *reinterpret_cast<const uint4*>(from + (k * M + 8) * lay.v_ld);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = VT - 1; k >= 0; --k)
#pragma unroll
                  for (int i = (IN32 ? VT - 1 - k : 0); i >= 0; --i) mma32(acc[m][j], lo[k], hi[k], bf[c][j][i]);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < H; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = row_of[16 * (m0 + m) + 8 * h + g];
            if (t < 0 || 8 * q >= wide) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[2 * j] = acc[m][j][2 * h], v[2 * j + 1] = acc[m][j][2 * h + 1];
            y[m][h].store(a.out, t * a.ldo + f0 + 8 * q, wide - 8 * q, vec, factor, v);
          }
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
  Columns<1, IN32, OUT32> columns(a, lay, row_of, tile.who, rank, ranks, y_vec);
  columns.start();
  {
    const int steps = (a.K + 31) / 32, per = (steps + ranks - 1) / ranks, s0 = min(rank * per, steps), s1 = min(s0 + per, steps);
    const char* A = static_cast<const char*>(a.a) + static_cast<long long>(tile.who) * R * K8 * kIn;
    const char* xrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) xrow[h] = row_of[8 * h + g] >= 0 ? static_cast<const char*>(a.x) + row_of[8 * h + g] * a.ldx * kIn : nullptr;
    for (int base = 0; base < tiles8; base += wn * NW) {
      const int n0 = base + warp % wn * NW;
      float sum[NW][4] = {};
      for (int s = s0 + kg; s < s1; s += wk) {
        const int k = 32 * s + 8 * q;
        uint4 xf[2][XT], af[NW][XT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < XT; ++i) xf[h][i] = zero4();
          if (xrow[h] != nullptr && k < a.K) load8<IN32>(xrow[h], k, a.K, x_vec, xf[h]);
        }
#pragma unroll
        for (int j = 0; j < NW; ++j) {
#pragma unroll
          for (int i = 0; i < XT; ++i) af[j][i] = zero4();
          if (n0 + j < tiles8 && k < K8) load8<IN32>(A + static_cast<long long>((n0 + j) * 8 + g) * K8 * kIn, k, K8, true, af[j]);
        }
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          float d[4] = {};
#pragma unroll
          for (int o = XT - 1; o >= 0; --o)  // the smallest products first
#pragma unroll
            for (int i = 0; i <= o; ++i) mma32(d, xf[0][i], xf[1][i], af[j][o - i]);
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
  join_shares<M, VT>(a, lay, partial, 1, vt, tile.count, ranks);
  __syncthreads();
  columns.run(vt);
  pg::cluster_sync_all();  // nobody leaves while its share is read
}

// Tiles of 64 bf16 rows: x and A go through shared memory, three stages of 64 k's, 128-byte rows whose 16-byte pieces are exchanged by the row's last bits; warps two by four.
constexpr int kStages = 3;
template <bool OUT32>
__global__ void __launch_bounds__(kThreads, OUT32 ? 1 : 2) adapter_tiles_kernel(const PgAdapter a, const Layout lay, int y_vec) {
  constexpr int M = 64, VT = OUT32 ? 3 : 2;
  extern __shared__ __align__(16) char raw[];
  __shared__ int row_of[M];
  const int ranks = cluster_size(), rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const Tile tile = tile_of<M>(a, item, 1, row_of);
  pg::griddep_wait();
  if (tile.count <= 0 || (tile.none && a.out == a.y)) return;  // (the whole cluster)
  if (tile.none) return copy_rows<OUT32>(a, row_of, tile.count, rank, ranks, y_vec);
  const int R = lay.R, K8 = (a.K + 7) / 8 * 8, blocks = (R + 15) / 16, per_warp = (blocks + 3) / 4, wm = warp % 2, n0 = warp / 2 * per_warp;
  const int stage_bytes = (M + blocks * 16) * 128;
  float* partial = reinterpret_cast<float*>(raw);  // (in the stages' place behind the product)
  uint16_t* vt = reinterpret_cast<uint16_t*>(raw + sizeof(float) * M * lay.partial_ld);
  {
    const int chunks = (a.K + 63) / 64, per = (chunks + ranks - 1) / ranks, c0 = min(rank * per, chunks), c1 = min(c0 + per, chunks);
    const char* A = static_cast<const char*>(a.a) + static_cast<long long>(tile.who) * R * K8 * 2;
    const uint32_t base = pg::smem_u32(raw);
    auto ask = [&](int c) {
      if (c < c1) {
        const uint32_t to = base + (c - c0) % kStages * stage_bytes;
        for (int i = tid; i < (M + blocks * 16) * 8; i += kThreads) {
          const int row = i / 8, piece = i % 8, k = 64 * c + 8 * piece;
          const char* from;
          bool there;
          if (row < M) {
            there = row_of[row] >= 0 && k < a.K;
            from = static_cast<const char*>(a.x) + ((there ? row_of[row] : 0) * a.ldx + (there ? k : 0)) * 2;
          } else {
            there = row - M < R && k < K8;
            from = A + (there ? static_cast<long long>(row - M) * K8 + k : 0) * 2;
          }
          pg::cp_async16(to + row * 128 + ((piece ^ (row & 7)) * 16), from, there);
        }
      }
      pg::cp_async_commit();
    };
    for (int i = 0; i < kStages - 1; ++i) ask(c0 + i);
    float sum[2][4][2][4] = {};
    for (int c = c0; c < c1; ++c) {
      pg::cp_async_wait<kStages - 2>();
      __syncthreads();
      ask(c + kStages - 1);
      const uint32_t at = base + (c - c0) % kStages * stage_bytes;
      float d[OUT32 ? 2 : 1][OUT32 ? 4 : 1][2][4] = {};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t xf[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int row = 32 * wm + 16 * m + lane % 16, piece = 2 * kk + lane / 16;
          pg::ldmatrix_x4(at + row * 128 + ((piece ^ (row & 7)) * 16), xf[m][0], xf[m][1], xf[m][2], xf[m][3]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b >= per_warp || n0 + b >= blocks) continue;
          const int row = M + 16 * (n0 + b) + lane % 8 + lane / 16 * 8, piece = 2 * kk + lane / 8 % 2;
          uint32_t w0, w1, w2, w3;
          pg::ldmatrix_x4(at + row * 128 + ((piece ^ (row & 7)) * 16), w0, w1, w2, w3);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            if constexpr (OUT32) {
              pg::mma_bf16_16816(d[m][b][0], xf[m], w0, w1);
              pg::mma_bf16_16816(d[m][b][1], xf[m], w2, w3);
            } else {
              pg::mma_bf16_16816(sum[m][b][0], xf[m], w0, w1);
              pg::mma_bf16_16816(sum[m][b][1], xf[m], w2, w3);
            }
          }
        }
      }
      if constexpr (OUT32) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[m][b][i / 4][i % 4] += d[m][b][i / 4][i % 4];
      }
    }
    pg::cp_async_wait<0>();
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (b < per_warp && n0 + b < blocks)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int row = 32 * wm + 16 * m + 8 * h + lane / 4, n = 16 * (n0 + b) + 8 * i + lane % 4 * 2;
              if (n < R) *reinterpret_cast<float2*>(partial + row * lay.partial_ld + n) = make_float2(sum[m][b][i][2 * h], sum[m][b][i][2 * h + 1]);
            }
  }
  Columns<4, false, OUT32> columns(a, lay, row_of, tile.who, rank, ranks, y_vec);
  columns.start();
  pg::cluster_sync_all();
  join_shares<M, VT>(a, lay, partial, 1, vt, tile.count, ranks);
  __syncthreads();
  columns.run(vt);
  pg::cluster_sync_all();  // nobody leaves while its share is read
}

template <typename Kern, typename... Args>
int launch(Kern kern, bool (&configured)[pg::kMaxDevices], long long items, int ranks, size_t smem, cudaStream_t st, Args... args) {
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  if (smem > kMostShared || items * ranks > 0x7fffffff) return PG_ERR_ARG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pg_pdl_enabled() ? 2 : 1;
  pg_count_launch(1);
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}

template <bool IN32, bool OUT32>
int pick(const PgAdapter& a, cudaStream_t st, int x_vec, int y_vec) {
  constexpr int VT = IN32 || OUT32 ? 3 : 2, NW = IN32 ? 2 : 6;  // (fp32: three terms of every fragment)
  Layout lay;
  lay.R = a.parts * a.rank;
  lay.partial_ld = lay.R + 4;
  lay.rank32 = (a.rank + 31) / 32 * 32;
  lay.v_ld = a.parts * lay.rank32;
  lay.v_ld += (lay.v_ld % 64 == 32) ? 0 : 32;  // eight lanes' 16-byte pieces of two rows lie in different banks
  if constexpr (!IN32) {
    // many rows of an adapter (up to 256 columns of v in a warp's registers)
    if (a.tile_rows == 64 && lay.R <= 256 && x_vec && a.K % 8 == 0) {
      const size_t stages = static_cast<size_t>(kStages) * (64 + (lay.R + 15) / 16 * 16) * 128, behind = sizeof(float) * 64 * lay.partial_ld + sizeof(uint16_t) * VT * 64 * lay.v_ld;
      const int room = (OUT32 ? 1 : 2) * pg::num_sms();
      int ranks = room / a.tile_count;  // shares of K: all CTAs at once
      ranks = ranks < 1 ? 1 : ranks > kMostRanks ? kMostRanks : ranks;
      while (ranks > 1 && a.K / ranks < 128) --ranks;
      static bool configured[pg::kMaxDevices] = {};
      return launch(adapter_tiles_kernel<OUT32>, configured, a.tile_count, ranks, stages > behind ? stages : behind, st, a, lay, y_vec);
    }
  }
  const int subs = a.tile_rows / 16;
  const long long items = static_cast<long long>(a.tile_count) * subs;
  int ranks = 1, wn = 1;
  while (ranks < kMostRanks && items * ranks * 2 <= 2 * pg::num_sms() && a.K / (ranks * 2) >= 128) ranks *= 2;
  while (wn < kWarps && wn * NW < lay.R / 8) wn *= 2;
  const size_t smem = sizeof(float) * (kWarps / wn) * 16 * lay.partial_ld + sizeof(uint16_t) * VT * 16 * lay.v_ld;
  static bool configured[pg::kMaxDevices] = {};
  return launch(adapter_rows_kernel<NW, IN32, OUT32>, configured, items, ranks, smem, st, a, lay, subs, x_vec, y_vec);
}

}  // namespace

extern "C" int pg_adapter_add(const PgAdapter* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgAdapter& a = *args;
  if (a.x == nullptr || a.y == nullptr || a.out == nullptr || a.a == nullptr || a.b == nullptr || a.scale == nullptr || a.rows == nullptr || a.tiles == nullptr || a.parts < 1 ||
      a.parts > 8 || a.K < 1 || a.rank < 8 || a.rank > 128 || a.rank % 8 || a.slots < 1 || a.tile_count < 1 || (a.tile_rows != 16 && a.tile_rows != 64) || a.T < 1 || a.ldx < a.K ||
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
