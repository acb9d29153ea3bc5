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

constexpr int kThreads = 256, kWarps = 8, kMostRanks = 8;

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

// MT: row tiles of 16; NW: column tiles of 8 that a warp holds in the first product
template <int MT, int NW, bool IN32, bool OUT32>
__global__ void __launch_bounds__(kThreads) adapter_kernel(const PgAdapter a, const Layout lay, int subs, int x_vec, int y_vec) {
  constexpr int M = 16 * MT, XT = IN32 ? 3 : 1, VT = IN32 || OUT32 ? 3 : 2;
  extern __shared__ __align__(16) char raw[];
  float* partial = reinterpret_cast<float*>(raw);                                                   // [M][partial_ld]
  uint16_t* vt = reinterpret_cast<uint16_t*>(raw + sizeof(float) * M * lay.partial_ld);             // [VT][M][v_ld]
  __shared__ int row_of[M];
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, q = lane % 4;
  const int* tile = a.tiles + 3 * (item / subs);
  const int who = tile[0], skip = item % subs * M, first = tile[1] + skip, count = min(tile[2] - skip, M);
  const bool none = who < 0 || who >= a.slots;
  pg::griddep_wait();  // (CTAs without work as well: the kernel behind counts on this one's end; the plan comes from the host, ahead of the step)
  if (count <= 0 || (none && a.out == a.y)) return;  // (the whole cluster)
  if (tid < M) {
    const int t = tid < count ? a.rows[first + tid] : -1;
    row_of[tid] = t < a.T ? t : -1;
  }
  __syncthreads();
  constexpr int kOut = OUT32 ? 4 : 2;
  if (none) {
    for (int i = 0; i < count; ++i) {
      const int t = row_of[i];
      if (t < 0) continue;
      const char* from = static_cast<const char*>(a.y) + t * a.ldy * kOut;
      char* to = static_cast<char*>(a.out) + t * a.ldo * kOut;
      if (y_vec)
        for (int c = (rank * kThreads + tid) * 16; c < a.F * kOut; c += ranks * kThreads * 16) {
          if (c + 16 <= a.F * kOut) *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(from + c);
          else
            for (int k = c; k < a.F * kOut; k += 2) *reinterpret_cast<uint16_t*>(to + k) = *reinterpret_cast<const uint16_t*>(from + k);
        }
      else
        for (int c = (rank * kThreads + tid) * 2; c < a.F * kOut; c += ranks * kThreads * 2) *reinterpret_cast<uint16_t*>(to + c) = *reinterpret_cast<const uint16_t*>(from + c);
    }
    return;
  }
  constexpr int kIn = IN32 ? 4 : 2;
  const int R = lay.R, K8 = (a.K + 7) / 8 * 8, tiles8 = R / 8;

  // ---- v = A x: this CTA's share of K, warps share out columns first, then K -------------------------------------------
  {
    const int steps = (a.K + 31) / 32, per = (steps + ranks - 1) / ranks, s0 = min(rank * per, steps), s1 = min(s0 + per, steps);
    int wn = 1;
    while (wn < kWarps && wn * NW < tiles8) wn *= 2;
    const int wk = kWarps / wn, kg = warp / wn;
    const char* A = static_cast<const char*>(a.a) + static_cast<long long>(who) * R * K8 * kIn;
    const char* xrow[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = row_of[16 * m + 8 * h + g];
        xrow[m][h] = t >= 0 ? static_cast<const char*>(a.x) + t * a.ldx * kIn : nullptr;
      }
    for (int base = 0; base < tiles8; base += wn * NW) {
      const int n0 = base + warp % wn * NW;
      float sum[MT][NW][4] = {};
      for (int s = s0 + kg; s < s1; s += wk) {
        const int k = 32 * s + 8 * q;
        uint4 xf[MT][2][XT], af[NW][XT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < XT; ++i) xf[m][h][i] = zero4();
            if (xrow[m][h] != nullptr && k < a.K) load8<IN32>(xrow[m][h], k, a.K, x_vec, xf[m][h]);
          }
#pragma unroll
        for (int j = 0; j < NW; ++j) {
#pragma unroll
          for (int i = 0; i < XT; ++i) af[j][i] = zero4();
          if (n0 + j < tiles8 && k < K8) load8<IN32>(A + static_cast<long long>((n0 + j) * 8 + g) * K8 * kIn, k, K8, true, af[j]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < NW; ++j) {
            float d[4] = {};
#pragma unroll
            for (int o = XT - 1; o >= 0; --o)  // the smallest products first
#pragma unroll
              for (int i = 0; i <= o; ++i) mma32(d, xf[m][0][i], xf[m][1][i], af[j][o - i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[m][j][i] += d[i];
          }
      }
      for (int turn = 0; turn < wk; ++turn) {  // the warps that share K, one after another
        if (kg == turn)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NW; ++j)
              if (n0 + j < tiles8)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float2* p = reinterpret_cast<float2*>(partial + (16 * m + 8 * h + g) * lay.partial_ld + (n0 + j) * 8 + 2 * q);
                  float2 v = make_float2(sum[m][j][2 * h], sum[m][j][2 * h + 1]);
                  if (turn > 0) v.x += p->x, v.y += p->y;
                  *p = v;
                }
        __syncthreads();
      }
    }
  }
  // ---- the shares of K together; v as bf16 terms, every part's ranks rounded up to 32 ------------------------------------
  pg::cluster_sync_all();
  {
    const int per_row = a.parts * lay.rank32 / 8;
    for (int i = tid; i < M * per_row; i += kThreads) {
      const int m = i / per_row, c = i % per_row * 8, part = c / lay.rank32, r = c % lay.rank32;
      uint4 t[VT];
#pragma unroll
      for (int k = 0; k < VT; ++k) t[k] = zero4();
      if (m < count && r < a.rank) {
        const float* from = partial + m * lay.partial_ld + part * a.rank + r;
        float f[8] = {};
        for (int p = 0; p < static_cast<int>(ranks); ++p) {
          const float4 lo = get_f4(from, p), hi = get_f4(from + 4, p);
          f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w, f[4] += hi.x, f[5] += hi.y, f[6] += hi.z, f[7] += hi.w;
        }
        split8<VT>(f, t);
      }
#pragma unroll
      for (int k = 0; k < VT; ++k) *reinterpret_cast<uint4*>(vt + (k * M + m) * lay.v_ld + c) = t[k];
    }
  }
  __syncthreads();
  // ---- out = y + B v: units of 32 columns, a warp each ------------------------------------------------------------------
  {
    const char* B = static_cast<const char*>(a.b) + static_cast<long long>(who) * a.F * a.rank * kIn;
    const float factor = a.gain * a.scale[who];
    int part = 0, col = 0, unit0 = 0;  // the part that holds the unit, its first column and unit
    for (int u = rank * kWarps + warp;; u += ranks * kWarps) {
      while (part < a.parts && u - unit0 >= (a.part_cols[part] + 31) / 32) {
        unit0 += (a.part_cols[part] + 31) / 32;
        col += a.part_cols[part];
        ++part;
      }
      if (part >= a.parts) break;
      const int f0 = col + 32 * (u - unit0), wide = min(32, col + a.part_cols[part] - f0);
      float acc[MT][4][4] = {};
      for (int r0 = 0; r0 < lay.rank32; r0 += 32) {
        uint4 bf[4][XT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = g / 2 * 8 + 2 * j + g % 2;
#pragma unroll
          for (int i = 0; i < XT; ++i) bf[j][i] = zero4();
          if (c < wide && r0 + 8 * q < a.rank) load8<IN32>(B + static_cast<long long>(f0 + c) * a.rank * kIn, r0 + 8 * q, a.rank, true, bf[j]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint16_t* from = vt + (16 * m + g) * lay.v_ld + part * lay.rank32 + r0 + 8 * q;
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
              for (int i = (IN32 ? VT - 1 - k : 0); i >= 0; --i) mma32(acc[m][j], lo[k], hi[k], bf[j][i]);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = row_of[16 * m + 8 * h + g], c = 8 * q;
          if (t < 0 || c >= wide) continue;
          float v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[2 * j] = acc[m][j][2 * h], v[2 * j + 1] = acc[m][j][2 * h + 1];
          if constexpr (OUT32) {
            const float* from = static_cast<const float*>(a.y) + t * a.ldy + f0 + c;
            float* to = static_cast<float*>(a.out) + t * a.ldo + f0 + c;
            if (y_vec && c + 8 <= wide) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float4 y = reinterpret_cast<const float4*>(from)[k];
                reinterpret_cast<float4*>(to)[k] = make_float4(fmaf(factor, v[4 * k], y.x), fmaf(factor, v[4 * k + 1], y.y), fmaf(factor, v[4 * k + 2], y.z), fmaf(factor, v[4 * k + 3], y.w));
              }
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (c + k < wide) to[k] = fmaf(factor, v[k], from[k]);
            }
          } else {
            const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(a.y) + t * a.ldy + f0 + c;
            __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.out) + t * a.ldo + f0 + c;
            if (y_vec && c + 8 <= wide) {
              const uint4 y = *reinterpret_cast<const uint4*>(from);
              const uint32_t w[4] = {y.x, y.y, y.z, y.w};
              uint32_t o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                o[k] = pg::pack_bf16(fmaf(factor, v[2 * k], __uint_as_float(w[k] << 16)), fmaf(factor, v[2 * k + 1], __uint_as_float(w[k] & 0xffff0000u)));
              *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (c + k < wide) to[k] = __float2bfloat16(fmaf(factor, v[k], __bfloat162float(from[k])));
            }
          }
        }
    }
  }
  pg::cluster_sync_all();  // nobody leaves while its share is read
}

template <int MT, int NW, bool IN32, bool OUT32>
int launch(const PgAdapter& a, cudaStream_t st, int x_vec, int y_vec) {
  constexpr int M = 16 * MT, VT = IN32 || OUT32 ? 3 : 2;
  Layout lay;
  lay.R = a.parts * a.rank;
  lay.partial_ld = lay.R + 4;
  lay.rank32 = (a.rank + 31) / 32 * 32;
  lay.v_ld = a.parts * lay.rank32;
  lay.v_ld += (lay.v_ld % 64 == 32) ? 0 : 32;  // eight lanes' 16-byte pieces of two rows lie in different banks
  const size_t smem = sizeof(float) * M * lay.partial_ld + sizeof(uint16_t) * VT * M * lay.v_ld;
  auto kern = adapter_kernel<MT, NW, IN32, OUT32>;
  static bool configured[pg::kMaxDevices] = {};
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  if (smem > 220 * 1024) return PG_ERR_ARG;
  const int subs = a.tile_rows / M;
  const long long items = static_cast<long long>(a.tile_count) * subs;
  int ranks = 1;
  while (ranks < kMostRanks && items * ranks * 2 <= 2 * pg::num_sms() && a.K / (ranks * 2) >= 128) ranks *= 2;
  if (items * ranks > 0x7fffffff) return PG_ERR_ARG;
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
  return cudaLaunchKernelEx(&cfg, kern, a, lay, subs, x_vec, y_vec) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}

template <bool IN32, bool OUT32>
int pick(const PgAdapter& a, cudaStream_t st, int x_vec, int y_vec) {
  // (64 rows of more than 256 columns of v do not fit beside their terms)
  return a.tile_rows == 64 && a.parts * a.rank <= 256 ? launch<4, 3, IN32, OUT32>(a, st, x_vec, y_vec) : launch<1, 6, IN32, OUT32>(a, st, x_vec, y_vec);
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
