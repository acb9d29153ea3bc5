// Log probability, rank and entropy of given tokens, and the top alternatives, from fp32 logits rows: one pass over the row.
//
// With z = x / T, m = max x, d = (x - m) / T, S = sum e^d, U = sum d e^d:
//   log p(t) = d_t - ln S        entropy = ln S - U / S        rank(t) = #{x > x_t} + #{x = x_t in front of t}
// S and U are kept by every thread against its own maximum and joined once (S' = S f, U' = (U + (m - m') S / T) f, f = e^((m - m') / T)).
//
// The largest `top` values without a second pass and without sorting: the order is by value, then by the lower index, as one 64-bit key.  Every
// half of a warp knows the largest key that it has met; the smallest of those 32 is below at least 32 keys, so only keys that reach it can be among
// the first 32: they go to a list in shared memory (some hundreds of a row), whose order is counted at the end.  A list that fills up is cut to its
// first `top` and the tile is offered again against the last of those.
//
// What bounds it: the bytes of the row (one read) where rows are many; for few rows the trip to memory and the joins, so up to eight CTAs of a
// cluster share a row and the first of them joins what they found through distributed shared memory: one launch, no scratch, no atomics on
// global memory (the list's order does not change results: keys are distinct and counted).
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kCap = 2048, kTop = 32;
constexpr int kVecs = 4;  // float4 a thread and tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// larger value first, then the lower index; NaN behind everything, both zeros alike
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t o = x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return o == 0u ? __uint_as_float(0x7fc00000u) : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

struct Stats {
  float m, s, u;  // maximum, sum of 2^((x - m) c), sum of (x - m) c 2^((x - m) c)
};
__device__ __forceinline__ Stats join(Stats a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return Stats{m, a.s + b.s, a.u + b.u};  // nothing but -inf (or NaN) so far
  const float da = a.m == -INFINITY ? -200.f : fmaxf((a.m - m) * c, -200.f), db = b.m == -INFINITY ? -200.f : fmaxf((b.m - m) * c, -200.f);
  const float fa = ex2(da), fb = ex2(db);
  return Stats{m, a.s * fa + b.s * fb, (a.u + da * a.s) * fa + (b.u + db * b.s) * fb};
}

struct Shared {
  unsigned long long list[kCap];
  unsigned long long best[kTop];  // the list's first, in order
  unsigned long long half[32];    // largest key of every half of a warp
  Stats warp[kWarps];
  int warp_rank[kWarps];
  Stats all;
  int rank, count, over;
};

// The list's first `top` keys in order (zeros where it has fewer): every thread counts how many are in front of its own.
__device__ __forceinline__ void order(Shared& sh, int count, int top) {
  if (threadIdx.x < kTop) sh.best[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const unsigned long long mine = sh.list[i];
    int before = 0;
    for (int j = 0; j < count; ++j) before += sh.list[j] > mine;
    if (before < top) sh.best[before] = mine;
  }
  __syncthreads();
}

template <bool TOP>
__global__ void __launch_bounds__(kThreads, 2) token_logprobs_kernel(const float* __restrict__ logits, long long ld, const int* __restrict__ tokens, float* __restrict__ logprob,
                                                                     float* __restrict__ entropy, int* __restrict__ rank, int* __restrict__ top_ids, float* __restrict__ top_logprob,
                                                                     int V, int top, float inv_t, int split) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  pg::griddep_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const float* x = logits + row * ld;
  const int t = tokens[row];
  const bool known = t >= 0 && t < V;
  const float xt = known ? x[t] : INFINITY;
  // x > x_t as x >= the next number (of +inf and NaN: NaN, which nothing reaches)
  const uint32_t bt = __float_as_uint(xt + 0.0f);
  const float above = __uint_as_float(xt + 0.0f < 0.f ? bt - 1u : bt + 1u);
  const float c = inv_t * kLog2e;
  // vectors of four on 16-byte boundaries; vector v holds elements 4 v - lead ..
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const int vectors = (V + lead + 3) / 4;
  const int per = (vectors + split - 1) / split, v0 = min(part * per, vectors), v1 = min(v0 + per, vectors);
  if (tid == 0) { sh.count = 0; sh.over = 0; }

  Stats st{-INFINITY, 0.f, 0.f};
  int above_t = 0;
  unsigned long long mine = 0, floor_key = 0;  // my largest key; what a key has to reach
  const int step = kThreads * kVecs;
  for (int base = v0; base < v1; base += step) {
    float4 f[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = base + i * kThreads + tid, e = 4 * v - lead;
      if (v < v1) {
        if (e >= 0 && e + 3 < V) {
          f[i] = __ldcs(reinterpret_cast<const float4*>(x + e));
        } else {
          f[i].x = e >= 0 && e < V ? x[e] : -INFINITY;
          f[i].y = e + 1 >= 0 && e + 1 < V ? x[e + 1] : -INFINITY;
          f[i].z = e + 2 >= 0 && e + 2 < V ? x[e + 2] : -INFINITY;
          f[i].w = e + 3 >= 0 && e + 3 < V ? x[e + 3] : -INFINITY;
        }
      } else {
        f[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
    }
    float mx = st.m;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) mx = fmaxf(mx, fmaxf(fmaxf(f[i].x, f[i].y), fmaxf(f[i].z, f[i].w)));
    if (mx > st.m) {
      const float d = st.m == -INFINITY ? -200.f : fmaxf((st.m - mx) * c, -200.f), g = ex2(d);
      st.u = (st.u + d * st.s) * g;
      st.s *= g;
      st.m = mx;
    }
    const float ms = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = base + i * kThreads + tid, e = v < v1 ? 4 * v - lead : -4;  // (what is not there counts as behind t)
      const float y[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = (y[k] - ms) * c, w = ex2(d);
        st.s += w;                              // (a NaN stays one)
        st.u = fmaf(fmaxf(d, -200.f), w, st.u);
        above_t += y[k] >= (static_cast<uint32_t>(e + k) < static_cast<uint32_t>(t) ? xt : above);
      }
    }
    if (TOP) {
      // my largest key of this tile and before
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int e = 4 * (base + i * kThreads + tid) - lead;
        const float y[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
        const float top4 = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        if (mine == 0 || !(top4 <= key_value(mine))) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (e + k >= 0 && e + k < V && base + i * kThreads + tid < v1) mine = max_key(mine, key_of(y[k], e + k));
        }
      }
      unsigned long long h = mine;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) h = max_key(h, __shfl_xor_sync(0xffffffffu, h, o));
      if ((lane & 15) == 0) sh.half[tid >> 4] = h;
      __syncthreads();
      h = sh.half[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, h, o);
        h = h < other ? h : other;
      }
      floor_key = max_key(floor_key, h);
      for (bool again = false;; again = true) {
        const float floor_x = key_value(floor_key);
        const bool unordered = (floor_key >> 32) == 0;  // a NaN reaches it
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int v = base + i * kThreads + tid, e = 4 * v - lead;
          const float y[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
          if (v < v1 && (unordered || fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= floor_x)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (e + k < 0 || e + k >= V || !(unordered || y[k] >= floor_x)) continue;
              const unsigned long long key = key_of(y[k], e + k);
              if (key < floor_key) continue;
              if (again) {
                bool listed = false;
                for (int j = 0; j < top; ++j) listed |= sh.best[j] == key;
                if (listed) continue;
              }
              const int at = atomicAdd(&sh.count, 1);
              if (at < kCap) sh.list[at] = key;
              else sh.over = 1;
            }
          }
        }
        __syncthreads();
        if (!sh.over) break;
        order(sh, kCap, top);  // the list is full: its first `top`, and the tile once more against the last of them
        if (tid < top) sh.list[tid] = sh.best[tid];
        floor_key = sh.best[top - 1];
        __syncthreads();
        if (tid == 0) { sh.count = top; sh.over = 0; }
        __syncthreads();
      }
    }
  }
  // the CTA's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)}, c);
    above_t += __shfl_xor_sync(0xffffffffu, above_t, o);
  }
  if (lane == 0) { sh.warp[warp] = st; sh.warp_rank[warp] = above_t; }
  __syncthreads();
  if (tid < 32) {
    Stats a = tid < kWarps ? sh.warp[tid] : Stats{-INFINITY, 0.f, 0.f};
    int r = tid < kWarps ? sh.warp_rank[tid] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a = join(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)}, c);
      r += __shfl_xor_sync(0xffffffffu, r, o);
    }
    if (tid == 0) { sh.all = a; sh.rank = r; }
  }
  if (TOP) order(sh, sh.count, top);
  else __syncthreads();
  if (split > 1) pg::cluster_sync_all();
  if (part == 0 && tid < 32) {
    // lane p has what CTA p found
    Stats a{-INFINITY, 0.f, 0.f};
    int r = 0;
    uint32_t there = 0;
    if (lane < split) {
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(&sh)), "r"(lane));
      auto word = [&](size_t off) {
        uint32_t w;
        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(w) : "r"(there + static_cast<uint32_t>(off)) : "memory");
        return w;
      };
      a.m = __uint_as_float(word(offsetof(Shared, all)));
      a.s = __uint_as_float(word(offsetof(Shared, all) + 4));
      a.u = __uint_as_float(word(offsetof(Shared, all) + 8));
      r = static_cast<int>(word(offsetof(Shared, rank)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a = join(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)}, c);
      r += __shfl_xor_sync(0xffffffffu, r, o);
    }
    const float ln_s = logf(a.s);
    if (lane == 0) {
      logprob[row] = known ? (xt - a.m) * inv_t - ln_s : __uint_as_float(0x7fc00000u);
      entropy[row] = ln_s - kLn2 * (a.u / a.s);
      rank[row] = known ? r : -1;
    }
    if (TOP) {
      // the CTAs' lists are in order: the largest of their heads, `top` times; lane i keeps the i-th
      auto head = [&](int n) {
        unsigned long long k = 0;
        if (lane < split && n < top) asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(k) : "r"(there + static_cast<uint32_t>(offsetof(Shared, best) + 8 * n)) : "memory");
        return k;
      };
      int n = 0;
      unsigned long long k = head(0), kept = 0;
      for (int i = 0; i < top; ++i) {
        unsigned long long w = k;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) w = max_key(w, __shfl_xor_sync(0xffffffffu, w, o));
        w = __shfl_sync(0xffffffffu, w, 0);  // (at most eight CTAs: lanes 0 .. 7)
        if (lane == i) kept = w;
        if (lane < split && k == w && w != 0) k = head(++n);
      }
      if (lane < top) {
        top_ids[row * top + lane] = key_index(kept);
        top_logprob[row * top + lane] = (key_value(kept) - a.m) * inv_t - ln_s;
      }
    }
  }
  if (split > 1) pg::cluster_sync_all();  // nobody leaves while its memory is read
}

}  // namespace

extern "C" int pg_token_logprobs(const float* logits, long long ld, const int* tokens, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprob,
                                 int rows, int V, int top, float temperature, void* stream) {
  if (rows <= 0 || V <= 0 || top < 0 || top > kTop || top > V || ld < V || !(temperature > 0.f) || !(temperature < INFINITY)) return PG_ERR_ARG;
  if (logits == nullptr || tokens == nullptr || logprob == nullptr || entropy == nullptr || rank == nullptr || (top > 0 && (top_ids == nullptr || top_logprob == nullptr))) return PG_ERR_ARG;
  if (V > 0x7fffff00 / 2 || (reinterpret_cast<uintptr_t>(logits) & 3) != 0) return PG_ERR_ARG;
  // CTAs that share a row: as many as fit the GPU at two an SM, no share below a tile's half
  int split = 1;
  while (split < 8 && (long long)rows * split * 2 <= 2LL * pg::num_sms() && V / (split * 2) >= kThreads * kVecs * 4 / 2) split *= 2;
  const long long grid = (long long)rows * split;
  if (grid > 0x7fffffffLL) return PG_ERR_ARG;
  auto kern = top > 0 ? token_logprobs_kernel<true> : token_logprobs_kernel<false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pg_pdl_enabled() ? 2 : 1;
  pg_count_launch(1);
  return cudaLaunchKernelEx(&cfg, kern, logits, ld, tokens, logprob, entropy, rank, top_ids, top_logprob, V, top, 1.0f / temperature, split) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
