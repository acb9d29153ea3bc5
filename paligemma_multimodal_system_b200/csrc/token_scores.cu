// Log probability, rank and entropy of given tokens, and the top alternatives, from fp32 logits rows: one pass over the row.
//
// With z = x / T, m = max x, d = (x - m) / T, S = sum e^d, U = sum d e^d:
//   log p(t) = d_t - ln S        entropy = ln S - U / S        rank(t) = #{x > x_t} + #{x = x_t in front of t}
// S and U are kept by every thread against its own maximum and joined once (S' = S f, U' = (U + (m - m') S / T) f, f = e^((m - m') / T)).
//
// The largest `top` entries without sorting: the order is by value, then by the lower index, as one 64-bit key.  A thread leaves the largest entry of every
// tile (or of a run of tiles) in shared memory.  Behind the pass, 64 groups of threads know their largest entries; the top-th of those 64 is reached by
// `top` entries at least, so only entries that reach it can be among the first `top`.  The few tiles whose largest entry does are read once more, and
// their entries that reach it go to a list (some dozens), whose order is counted.  Masked rows (fewer than `top` entries left, or the least of them shared
// by more than the list holds) take the equal ones from the front.  Where that fails -- large entries that lie in few threads' tiles -- the part is read
// again by keys, tile by tile, and the list cut to its first `top` as often as it fills.
//
// What bounds it: the bytes of the row (one read) where rows are many; for few rows the trip to memory and the joins, so up to eight CTAs of a
// cluster share a row and the first of them joins what they found through distributed shared memory: one launch, no scratch, no atomics on
// global memory (the list's order does not change results: keys are distinct and counted).  Many rows: CTAs that stay walk them, the next row's first tile under way while one is
// joined.  64 x 257216 with 20 alternatives 26 us (2.5 TB/s; without alternatives 21), 1500 x 32000 with one 51 (3.7 TB/s; 43), one x 257216 with five 14.
// Rows of masked entries or of one number take 28 to 36 us for the first of these (read again by keys 340 to 610).
// Lists kept while the row goes by (a floor in shared memory, raised tile by tile) cost the loop its registers and took 33 to 97 us for the first of these.
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 256, kPerSm = 3, kWarps = kThreads / 32, kGroup = kThreads / 64, kCap = 2048, kTop = 32, kHits = 512;  // 64 groups of threads
constexpr int kVecs = 4, kSlots = 32;  // float4 a thread and tile; runs of tiles whose largest entries are kept
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
struct Shared {
  float slot[kSlots][kThreads];    // a thread's largest entry of a run of tiles
  unsigned long long list[kCap];
  unsigned long long best[kTop];   // the list's first, in order
  unsigned long long group_key[64];
  float group[64];                 // largest entry of every group
  Stats warp[kWarps];
  int warp_rank[kWarps];
  Stats all;
  int rank, count, over, hits, fails, any;
  uint32_t least;                  // what an entry has to reach, as an ordered number
  int hit[kHits];                  // runs of tiles that hold entries which reach it: 2^16 slot + thread
};

// The list's first `top` keys in order (zeros where it has fewer): four lanes count how many are in front of a key.
__device__ __forceinline__ void order(Shared& sh, int count, int top) {
  if (threadIdx.x < kTop) sh.best[threadIdx.x] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < count; i0 += kThreads / 4) {
    const int i = i0 + threadIdx.x / 4;
    if (i0 + (threadIdx.x & ~31u) / 4 >= count) break;  // (whole warps)
    const unsigned long long mine = i < count ? sh.list[i] : ~0ull;
    int before = 0;
#pragma unroll 4
    for (int j = threadIdx.x % 4; j < count; j += 4) before += sh.list[j] > mine;
    before += __shfl_xor_sync(0xffffffffu, before, 1);
    before += __shfl_xor_sync(0xffffffffu, before, 2);
    if (i < count && mine != 0 && before < top && threadIdx.x % 4 == 0) sh.best[before] = mine;
  }
  __syncthreads();
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float one_if_ge(float a, float b) { return a >= b ? 1.f : 0.f; }
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }

__device__ __forceinline__ void list_key(Shared& sh, unsigned long long key) {
  const int slot = atomicAdd(&sh.count, 1);
  if (slot < kCap) sh.list[slot] = key;
  else sh.over = 1;
}

// a CTA's part of a row: vectors of four on 16-byte boundaries, vector v holds entries 4 v - lead ..
struct Part {
  const float* x;
  int lead, v0, v1;
  __device__ __forceinline__ Part(const float* row, int V, int part, int split) : x(row), lead(static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 2) & 3)) {
    const int vectors = (V + lead + 3) / 4, per = (vectors + split - 1) / split;
    v0 = min(part * per, vectors);
    v1 = min(v0 + per, vectors);
  }
  __device__ __forceinline__ void load(float4 (&f)[kVecs], int base, int V) const {  // -inf for what is not there
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = base + i * kThreads + threadIdx.x, e = 4 * v - lead;
      f[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (v < v1) {
        if (e >= 0 && e + 3 < V) {
          f[i] = __ldcs(reinterpret_cast<const float4*>(x + e));
        } else {
          if (e >= 0 && e < V) f[i].x = x[e];
          if (e + 1 >= 0 && e + 1 < V) f[i].y = x[e + 1];
          if (e + 2 >= 0 && e + 2 < V) f[i].z = x[e + 2];
          if (e + 3 >= 0 && e + 3 < V) f[i].w = x[e + 3];
        }
      }
    }
  }
};

// The entries that reach `least`, from the runs of tiles whose largest one does, into the list.
__device__ __forceinline__ void list_hits(Shared& sh, const Part& p, int V, float least, int slots, int run) {
  const int tid = threadIdx.x;
  for (int k = 0; k < slots; ++k)
    if (sh.slot[k][tid] >= least) {
      const int at = atomicAdd(&sh.hits, 1);
      if (at < kHits) sh.hit[at] = k << 16 | tid;
    }
  __syncthreads();
  // four lanes a run, all of them under way together
  const int hits = min(sh.hits, kHits);
  for (int i = tid / 4; i < hits; i += kThreads / 4) {
    const int k = sh.hit[i] >> 16, who = sh.hit[i] & 0xffff;
    for (int v = p.v0 + k * run + (tid % 4) * kThreads + who; v < min(p.v0 + (k + 1) * run, p.v1); v += 4 * kThreads) {
      const int e = 4 * v - p.lead;
      float z[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) z[y] = e + y >= 0 && e + y < V ? p.x[e + y] : -INFINITY;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (z[y] >= least) list_key(sh, key_of(z[y], e + y));
    }
  }
  __syncthreads();
}

// the number behind x: what is larger than x reaches it.  Behind +inf and NaN: NaN, which nothing reaches.
__device__ __forceinline__ float number_above(float x) {
  if (x != x) return x;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return __uint_as_float(x + 0.0f < 0.f ? b - 1u : b + 1u);
}

// Masked rows: fewer than `top` entries are left (the others -inf), or more share the least value that counts (a mask of the lowest value) than the list holds.  What is larger is
// listed; of the equal ones only those in front matter, and they are met after few entries.
__device__ __noinline__ void list_ties(Shared& sh, const Part p, int V, int top, float least, int slots, int run) {
  const int tid = threadIdx.x;
  float tie = -INFINITY;
  if (sh.hits > kHits || sh.over) {
    tie = least;
    __syncthreads();
    if (tid == 0) { sh.count = 0; sh.over = 0; sh.hits = 0; }
    __syncthreads();
    list_hits(sh, p, V, number_above(least), slots, run);
    if (sh.hits > kHits || sh.over) return;  // (the careful way)
  }
  const int larger = sh.count;
  for (int v0 = p.v0; v0 < p.v1; v0 += kThreads) {
    const int v = v0 + tid, e = 4 * v - p.lead;
    __syncthreads();  // the count is read
    bool is[4];
    int front = 0;  // equal ones in front of this lane's in its warp, whose first `top` are enough
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      is[y] = v < p.v1 && e + y >= 0 && e + y < V && p.x[e + y] == tie;
      front += __popc(__ballot_sync(0xffffffffu, is[y]) & ((1u << (tid & 31)) - 1u));
    }
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (is[y] && front++ < top) list_key(sh, key_of(tie, e + y));
    __syncthreads();
    if (sh.count - larger >= top || sh.over) break;
  }
}

// The careful way: tiles by keys, with barriers.
__device__ __noinline__ void list_by_keys(Shared& sh, const Part p, int V, int top) {
  const int v0 = p.v0, v1 = p.v1, lead = p.lead;
  const int tid = threadIdx.x, lane = tid & 31, step = kThreads * kVecs;
  if (tid == 0) { sh.count = 0; sh.over = 0; }
  __syncthreads();
  unsigned long long mine = 0, floor = 0;
  for (int base = v0; base < v1; base += step) {
    float4 f[kVecs];
    p.load(f, base, V);
    auto each = [&](auto fn) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int v = base + i * kThreads + tid, e = 4 * v - lead;
        const float y[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v < v1 && e + k >= 0 && e + k < V) fn(key_of(y[k], e + k));
      }
    };
    each([&](unsigned long long key) { mine = max_key(mine, key); });
    unsigned long long h = mine;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) h = max_key(h, __shfl_xor_sync(0xffffffffu, h, o));
    if (tid % kGroup == 0) sh.group_key[tid / kGroup] = h;
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 64; part += 32) {
      h = sh.group_key[part + lane];  // (keys are distinct; 0: a group that has met nothing)
      int before = 0;
      for (int i = 0; i < 64; ++i) before += sh.group_key[i] > h;
      const uint32_t at = __ballot_sync(0xffffffffu, before == top - 1 && h != 0);
      if (at != 0) floor = max_key(floor, __shfl_sync(0xffffffffu, h, __ffs(at) - 1));
    }
    for (bool again = false;; again = true) {
      each([&](unsigned long long key) {
        if (key < floor) return;
        if (again) {
          for (int j = 0; j < top; ++j)
            if (sh.best[j] == key) return;
        }
        list_key(sh, key);
      });
      __syncthreads();
      if (!sh.over) break;
      order(sh, kCap, top);
      if (tid < top) sh.list[tid] = sh.best[tid];
      floor = max_key(floor, sh.best[top - 1]);
      __syncthreads();
      if (tid == 0) { sh.count = top; sh.over = 0; }
      __syncthreads();
    }
  }
}

// Sums of a warp against one maximum
__device__ __forceinline__ Stats join_warp(Stats a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m > -INFINITY) {
    const float d = a.m == -INFINITY ? -200.f : fmaxf((a.m - m) * c, -200.f), g = ex2(d);
    a.u = (a.u + d * a.s) * g;
    a.s *= g;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  a.m = m;
  return a;
}
__device__ __forceinline__ int sum_warp(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The list's first `top` of a row that holds (ln S, m) in the place of its alternatives (one alternative: it is m)
__device__ __forceinline__ void put_alternatives(Shared& sh, int* ids, float* logprob, long long row, int top, float inv_t) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const unsigned long long k = sh.best[lane < top ? lane : 0];
    const float ln_s = logprob[row * top], m = top > 1 ? logprob[row * top + 1] : key_value(k);
    __syncwarp();
    if (lane < top) {
      ids[row * top + lane] = key_index(k);
      logprob[row * top + lane] = (key_value(k) - m) * inv_t - ln_s;
    }
  }
}

// split 1: a CTA takes every gridDim-th row, the next row's first tile under way while the sums of one are joined; else the CTAs of a cluster share a row.
template <bool TOP>
__global__ void __launch_bounds__(kThreads, kPerSm) token_logprobs_kernel(const float* __restrict__ logits, long long ld, const int* __restrict__ tokens, float* __restrict__ logprob,
                                                                     float* __restrict__ entropy, int* __restrict__ rank, int* __restrict__ top_ids, float* __restrict__ top_logprob,
                                                                     int rows, int V, int top, float inv_t, int split) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = blockIdx.x % split;
  if (tid == 0) { sh.count = 0; sh.over = 0; sh.hits = 0; sh.least = 0xffffffffu; }
  pg::griddep_begin();
  const float c = inv_t * kLog2e;
  const uint64_t cc = pg::pair_of(c, c);
  constexpr int step = kThreads * kVecs;
  const int stride = split > 1 ? rows : gridDim.x, row0 = blockIdx.x / split;
  float4 f[kVecs];
  {
    const Part p(logits + (long long)row0 * ld, V, part, split);
    p.load(f, p.v0, V);
  }
  int t_next = tokens[row0];
  for (int row = row0; row < rows; row += stride) {
    const Part p(logits + row * ld, V, part, split);
    const int t = t_next;
    const bool more = row + stride < rows, known = t >= 0 && t < V;
    if (more) t_next = tokens[row + stride];
    const float xt = known ? p.x[t] : INFINITY;
    const float above = number_above(xt);
    const int run = ((p.v1 - p.v0 + step - 1) / step + kSlots - 1) / kSlots * step;  // vectors of a slot
    Stats st{-INFINITY, 0.f, 0.f};
    uint64_t sums = 0, weighted = 0, front = 0;  // pairs: sum of e^d, sum of d e^d, entries in front of t
    float here = -INFINITY;
    int slot = 0, slot_end = p.v0 + run;
    for (int base = p.v0; base < p.v1; base += step) {
      float4 next[kVecs];
      if (base + step < p.v1) p.load(next, base + step, V);
      else if (more) Part(logits + (row + stride) * ld, V, 0, 1).load(next, 0, V);
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) mx = fmaxf(mx, pg::max3(fmaxf(f[i].x, f[i].y), f[i].z, f[i].w));
      if (TOP) {
        here = fmaxf(here, mx);
        if (base + step >= slot_end || base + step >= p.v1) {
          sh.slot[slot][tid] = here;
          here = -INFINITY;
          ++slot;
          slot_end += run;
        }
      }
      if (mx > st.m) {
        const float d = st.m == -INFINITY ? -200.f : fmaxf((st.m - mx) * c, -200.f), g = ex2(d);
        const uint64_t gg = pg::pair_of(g, g), dd = pg::pair_of(d, d);
        weighted = mul_pair(pg::fma_pair(dd, sums, weighted), gg);
        sums = mul_pair(sums, gg);
        st.m = mx;
      }
      const float ms = st.m == -INFINITY ? 0.f : st.m;
      const uint64_t minus = pg::pair_of(-ms, -ms);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int v = base + i * kThreads + tid, e = v < p.v1 ? 4 * v - p.lead : V;  // (what is not there counts as behind t)
        const float reach = e + 3 < t && e >= 0 ? xt : above;                        // (entries of t's own vector and of a first one that is not whole: below)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = h ? f[i].z : f[i].x, b = h ? f[i].w : f[i].y;
          const uint64_t q = mul_pair(pg::add_pair(pg::pair_of(a, b), minus), cc);
          const float da = max_nan(pg::lo_f32(q), -200.f), db = max_nan(pg::hi_f32(q), -200.f);
          const uint64_t w = pg::pair_of(ex2(da), ex2(db));  // (a NaN stays one)
          sums = pg::add_pair(sums, w);
          weighted = pg::fma_pair(pg::pair_of(da, db), w, weighted);
          front = pg::add_pair(front, pg::pair_of(one_if_ge(a, reach), one_if_ge(b, reach)));
        }
      }
#pragma unroll
      for (int i = 0; i < kVecs; ++i) f[i] = next[i];
    }
    if (TOP) {
      float h = st.m;
#pragma unroll
      for (int o = kGroup / 2; o > 0; o >>= 1) h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
      if (tid % kGroup == 0) sh.group[tid / kGroup] = h;
    }
    st.s = pg::lo_f32(sums) + pg::hi_f32(sums);
    st.u = pg::lo_f32(weighted) + pg::hi_f32(weighted);
    int before = static_cast<int>(pg::lo_f32(front)) + static_cast<int>(pg::hi_f32(front));
    if (tid < 6 && known) {  // equal entries in front of t that were counted as behind it: in t's own vector, and in a first vector that is not whole
      const int own = (t + p.lead) / 4 * 4 - p.lead, i = tid < 3 ? own + tid : tid - 3;
      const bool mine = tid < 3 ? i >= 0 && i < t : i < min(t, 4 - p.lead) && p.lead > 0 && own > 0;
      const int v = (i + p.lead) / 4;
      if (mine && v >= p.v0 && v < p.v1 && p.x[i] == xt) ++before;
    }
    // the CTA's sums
    st = join_warp(st, c);
    before = sum_warp(before);
    if (lane == 0) { sh.warp[warp] = st; sh.warp_rank[warp] = before; }
    __syncthreads();
    if (TOP) {
      {  // the top-th largest of the groups' entries: a group's threads share out the others
        const float h = sh.group[tid / kGroup];
        int in_front = 0;
#pragma unroll
        for (int i = 0; i < 64 / kGroup; ++i) in_front += sh.group[tid % kGroup + i * kGroup] > h;
#pragma unroll
        for (int o = kGroup / 2; o > 0; o >>= 1) in_front += __shfl_xor_sync(0xffffffffu, in_front, o);
        if (tid % kGroup == 0 && in_front < top) atomicMin(&sh.least, ordered(h));
      }
      __syncthreads();
      const float least = fmaxf(unordered(sh.least), -3.402823466e38f);  // (masked entries are not listed)
      list_hits(sh, p, V, least, slot, run);
      if (sh.hits > kHits || sh.over || sh.count < top) list_ties(sh, p, V, top, least, slot, run);
      if (tid == 0) sh.fails = sh.hits > kHits || sh.over || (sh.count < top && p.v0 < p.v1);  // (fewer entries than `top`: the careful way lists them all)
    }
    if (warp == kWarps - 1) {
      const Stats a = join_warp(lane < kWarps ? sh.warp[lane % kWarps] : Stats{-INFINITY, 0.f, 0.f}, c);
      const int r = sum_warp(lane < kWarps ? sh.warp_rank[lane % kWarps] : 0);
      if (lane == 0) { sh.all = a; sh.rank = r; }
    }
    if (TOP) order(sh, min(sh.count, kCap), top);
    if (split > 1) {
      // the first CTA of the cluster gathers what the others found: lane p of its first warp CTA p's sums, a thread one of their keys
      pg::cluster_sync_all();
      if (part == 0) {
        auto at = [&](int cta, size_t off) {
          uint32_t there;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(&sh) + static_cast<uint32_t>(off)), "r"(cta));
          return there;
        };
        auto word = [&](uint32_t there) {
          uint32_t w;
          asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(w) : "r"(there) : "memory");
          return w;
        };
        if (TOP && tid < split * top) {
          unsigned long long k;
          asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(k) : "r"(at(tid / top, offsetof(Shared, best) + 8 * (tid % top))) : "memory");
          sh.list[tid] = k;
        }
        Stats a{-INFINITY, 0.f, 0.f};
        int r = 0, bad = 0;
        if (tid < split) {
          if (TOP) bad = static_cast<int>(word(at(tid, offsetof(Shared, fails))));
          a.m = __uint_as_float(word(at(tid, offsetof(Shared, all))));
          a.s = __uint_as_float(word(at(tid, offsetof(Shared, all) + 4)));
          a.u = __uint_as_float(word(at(tid, offsetof(Shared, all) + 8)));
          r = static_cast<int>(word(at(tid, offsetof(Shared, rank))));
        }
        __syncthreads();
        bad = __syncthreads_or(bad);
        if (TOP && tid == 0) sh.any = bad;
        if (warp == 0) {
          a = join_warp(a, c);
          r = sum_warp(r);
          if (lane == 0) { sh.all = a; sh.rank = r; }
        }
        if (TOP) order(sh, split * top, top);
      }
    }
    __syncthreads();
    if (part == 0 && warp == 0) {
      const Stats a = sh.all;
      const float ln_s = logf(a.s);
      if (lane == 0) {
        logprob[row] = known ? (xt - a.m) * inv_t - ln_s : __uint_as_float(0x7fc00000u);
        entropy[row] = ln_s - kLn2 * (a.u / a.s);
        rank[row] = known && xt == xt ? sh.rank : -1;  // (a NaN has no place among numbers)
      }
      if (TOP && lane < top) {
        const unsigned long long k = sh.best[lane];
        const bool again = split > 1 ? sh.any != 0 : sh.fails != 0;  // below; until then what it needs stands in the row
        top_ids[(long long)row * top + lane] = again ? -1 : key_index(k);
        top_logprob[(long long)row * top + lane] = again ? (lane == 0 ? ln_s : a.m) : (key_value(k) - a.m) * inv_t - ln_s;
      }
    }
    if (more) {
      if (tid == kThreads - 1) { sh.count = 0; sh.over = 0; sh.hits = 0; sh.least = 0xffffffffu; }
      __syncthreads();  // the row's results are read, the next one's may come
    }
  }
  // ---- rows whose alternatives have to be found the careful way
  if (TOP) {
    __syncthreads();
    if (split > 1) {
      pg::cluster_sync_all();
      uint32_t there;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(&sh.any)), "r"(0));
      int any;
      asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(any) : "r"(there) : "memory");
      if (any) {
        list_by_keys(sh, Part(logits + row0 * ld, V, part, split), V, top);
        order(sh, sh.count, top);
        pg::cluster_sync_all();
        if (part == 0) {
          if (tid < split * top) {
            unsigned long long k;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(&sh.best[tid % top])), "r"(tid / top));
            asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(k) : "r"(there) : "memory");
            sh.list[tid] = k;
          }
          __syncthreads();
          order(sh, split * top, top);
          put_alternatives(sh, top_ids, top_logprob, row0, top, inv_t);
        }
      }
    } else {
      for (int row = row0; row < rows; row += stride) {
        if (top_ids[(long long)row * top] != -1) continue;  // (this CTA's own, written before the barrier)
        list_by_keys(sh, Part(logits + row * ld, V, 0, 1), V, top);
        order(sh, sh.count, top);
        put_alternatives(sh, top_ids, top_logprob, row, top, inv_t);
        __syncthreads();
      }
    }
  }
  if (split > 1) pg::cluster_sync_all();  // nobody leaves while its memory is read
}

}  // namespace

extern "C" int pg_token_logprobs(const float* logits, long long ld, const int* tokens, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprob,
                                 int rows, int V, int top, float temperature, void* stream) {
  if (rows <= 0 || V <= 0 || top < 0 || top > kTop || top > V || ld < V || !(temperature > 0.f) || !(temperature < INFINITY) || !(1.0f / temperature * kLog2e < INFINITY)) return PG_ERR_ARG;
  if (logits == nullptr || tokens == nullptr || logprob == nullptr || entropy == nullptr || rank == nullptr || (top > 0 && (top_ids == nullptr || top_logprob == nullptr))) return PG_ERR_ARG;
  if (V > 0x7fffff00 / 2 || (reinterpret_cast<uintptr_t>(logits) & 3) != 0) return PG_ERR_ARG;
  // CTAs that share a row: as many as fit the GPU at three an SM, no share below a tile's half
  int split = 1;
  while (split < 8 && (long long)rows * split * 2 <= (long long)kPerSm * pg::num_sms() && V / (split * 2) >= kThreads * kVecs * 4 / 2) split *= 2;
  auto kern = top > 0 ? token_logprobs_kernel<true> : token_logprobs_kernel<false>;
  constexpr int kMost = sizeof(Shared);
  static bool configured[2][pg::kMaxDevices] = {};  // once a device
  bool& done = configured[top > 0][pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  // (clusters share rows only while all of them are there at once; else three CTAs an SM walk the rows)
  const int sms = pg::num_sms();
  const long long grid = split > 1 ? (long long)rows * split : rows < kPerSm * sms ? rows : kPerSm * sms;
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
  return cudaLaunchKernelEx(&cfg, kern, logits, ld, tokens, logprob, entropy, rank, top_ids, top_logprob, rows, V, top, 1.0f / temperature, split) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
