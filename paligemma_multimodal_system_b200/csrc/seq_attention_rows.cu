// Attention of a few rows an entry over a long paged cache: decoded tokens over the 8-bit cache, and drafted trees over a cache of any type.
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(s_ij),  s_ij = cap(scale q_i . k_j) - penalty,  j over the keys that row i sees:
//   every stored key j < ctx, and drafted key m (cache row ctx + m) where bit m of the row's mask is set (no mask: m <= i); windows go by positions.
//
// A warp owns 16 MT rows (token x query head of one k/v head) and walks key tiles of its own straight from the pages: no shared memory, no barrier in
// the loop.  Both products run on mma.sync m16n8k16 with fp32 accumulation, and the operands' k indexes are permuted so that a lane's 16-byte pieces of
// the cache ARE its fragments:
//   * keys: lane (n, c) reads piece c of key n's row; the elements of a piece are k indexes of ITS lane in consecutive 16-deep steps, and the
//     queries are stored in that order once.  Key n of fragment f is key (KT / 4)(n / 2) + 2 f + n % 2 of the tile, so lane c's scores belong to KT / 4
//     neighbouring keys, and those are the keys whose value rows it reads for the second product, columns 8 n .. 8 n + 7 of every 64.
//   * no transposition, no conversion but codes -> halves (exact) and, for fp32, the cut into three bf16 terms.
// Precision: bf16 operands as they are; codes as halves, exact, against queries scaled by a power of two per row into half range (fp32 queries: two
// halves, 22 bits); fp32 as three bf16 terms, six products.  Weights: two bf16 terms over bf16 values (16 bits); one half over codes for bf16
// rows (11 bits: an eighth of the output's own rounding), two for fp32 rows; three bf16 terms over fp32 values.  The values' powers of two
// go into the weights relative to the largest one so far.  Scores, maxima, sums and outputs are fp32.
//
// What bounds it: the bytes of keys and values while a k/v head has few rows; the tensor instructions for large trees.  Warps of a CTA share a key walk
// (few rows) or the rows (trees); CTAs split the keys further, and a merge launch joins their (maximum, sum, accumulator).
#include <cuda_fp16.h>

#include "cache8.cuh"
#include "common.cuh"
#include "paligemma_b200.h"

using bf16 = __nv_bfloat16;

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
struct e4m3 {
  uint8_t code;
};

struct Args {
  const void* q;
  const uint8_t *kp, *vp;       // pages
  const uint8_t *ke, *ve;       // powers of an 8-bit cache
  const void* gate;
  long long ldg;
  void* out;
  float* partial;
  const int *row0, *n, *ctx, *pt, *pos;
  const uint32_t* tree;
  int words, max_pages, page, singles, nsplit, blocks, H, G, dim, vdim, wr;
  float scale, softcap;
  int gate_per_head;
  PgAttnScore sx;
  int trigger;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh to fp32 accuracy: odd series near zero, else 1 - 2 / (e^(2 |x|) + 1)
__device__ __forceinline__ float tanh_f32(float x) {
  const float ax = fabsf(x), x2 = x * x;
  const float small = x * fmaf(x2, fmaf(x2, 0.13333333f, -0.33333334f), 1.0f);
  const float big = copysignf(1.0f - __fdividef(2.0f, ex2(ax * (2.f * kLog2e)) + 1.0f), x);
  return ax < 0.1f ? small : big;
}
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (lo, hi) as N terms of the operand type, each the rounding of what the ones before left
template <bool HALF, int N>
__device__ __forceinline__ void terms(float lo, float hi, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = HALF ? pack_half(lo, hi) : pg::pack_bf16(lo, hi);
    if (i + 1 < N) {
      float a, b;
      if (HALF) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&t[i]));
        a = f.x, b = f.y;
      } else {
        a = __uint_as_float(t[i] << 16), b = __uint_as_float(t[i] & 0xffff0000u);
      }
      lo -= a, hi -= b;
    }
  }
}

template <typename TQ, typename TC>
struct Kind {
  static constexpr bool C8 = sizeof(TC) == 1, F32 = sizeof(TC) == 4, HALF = C8;
  static constexpr int QT = F32 ? 3 : (C8 && sizeof(TQ) == 4) ? 2 : 1;             // terms of a query
  static constexpr int CT = F32 ? 3 : 1;                                           // terms of a cached element
  static constexpr int PT = F32 ? 3 : C8 ? (sizeof(TQ) == 4 ? 2 : 1) : 2;          // terms of a weight
  static constexpr int KL = sizeof(TC);                                            // 16-byte pieces of a lane in 64 elements of a key row
  static constexpr int VW = 2 * sizeof(TC);                                        // words of eight value columns
};

// DC, VC: 64-element pieces of a key / value row; MT: 16-row tiles of a warp; KT: keys of a tile
template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
__global__ void __launch_bounds__(32 * kWarps) attn_rows_kernel(const __grid_constant__ Args a) {
  using K = Kind<TQ, TC>;
  constexpr int NB = KT / 8, KPL = KT / 4;  // key fragments of a tile; keys of a lane
  constexpr int Q16 = 4 * DC;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ float unscale[kWarps * 16 * MT];  // what a row's scores are multiplied by (log2 units unless something comes between)
  __shared__ float2 stat[kWarps][16 * MT];
  __shared__ float top_power[kWarps];
  if (a.nsplit > 1) pg::griddep_begin<true>();  // (fp32 partials, read behind a wait)
  else pg::griddep_begin_if(a.trigger);
  const int split = blockIdx.x, g = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, e = blockIdx.z;
  const int n = a.n[e], ctx = a.ctx[e], gsz = a.H / a.G, len = ctx + n;
  const long long t0 = a.row0[e];
  const int wr = a.wr, wk = kWarps / wr, rows_cta = wr * 16 * MT, r0 = block * rows_cta, R = n * gsz;
  if ((a.singles && n != 1) || r0 >= R) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nn = lane >> 2, c = lane & 3;
  const int rg = warp % wr, kgrp = warp / wr;
  const bool special = a.softcap > 0.f || a.sx.dist_a != nullptr || a.sx.logistic;

  // ---- queries: fragments in the order of the cache's pieces
  uint4* qs = reinterpret_cast<uint4*>(raw);  // [term][row tile][step][lane]
  const int tiles_m = wr * MT;
  for (int r = warp; r < rows_cta; r += kWarps) {
    const int rr = r0 + r;
    const bool in = rr < R;
    const int i = in ? rr / gsz : 0, head = g * gsz + (in ? rr - i * gsz : 0);
    float s = a.scale * (a.sx.head_scale != nullptr ? a.sx.head_scale[head] : 1.f);
    float up = 1.f;
    const TQ* q = static_cast<const TQ*>(a.q) + (t0 + i) * (long long)a.H * a.dim + (long long)head * a.dim;
    if (K::C8) {
      float top = 0.f;
      for (int d = lane; d < a.dim; d += 32) top = fmaxf(top, in ? fabsf(ldf(q + d)) : 0.f);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // largest element to [2^14, 2^15): a half keeps eleven bits down to 2^-14, and 2^-24 below
      const int x = min(max(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100);
      up = __uint_as_float(static_cast<uint32_t>(x + 127) << 23);
      s *= __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
    }
    if (lane == 0) unscale[r] = special ? s : s * kLog2e;
    // row r of the tile: lanes 4 (r % 8) + c, first or second half of the fragment's registers
    const int m = r / 16, lo8 = (r % 16) < 8;
    for (int w = lane; w < Q16 * 4; w += 32) {
      const int st = w / 4, cc = w % 4;
      const int d0 = K::C8 ? 64 * (st / 4) + 16 * cc + 4 * (st % 4) : K::F32 ? 16 * st + 4 * cc : 32 * (st / 2) + 8 * cc + 4 * (st % 2);
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = in && d0 + k < a.dim ? ldf(q + d0 + k) * up : 0.f;
      uint32_t p[K::QT], s2[K::QT];
      terms<K::HALF>(v[0], v[1], p);
      terms<K::HALF>(v[2], v[3], s2);
#pragma unroll
      for (int t = 0; t < K::QT; ++t) {
        uint32_t* f = reinterpret_cast<uint32_t*>(qs + ((t * tiles_m + m) * Q16 + st) * 32 + 4 * (r % 8) + cc);
        f[lo8 ? 0 : 1] = p[t];
        f[lo8 ? 2 : 3] = s2[t];
      }
    }
  }
  __syncthreads();

  // ---- my rows
  int node[2 * MT];       // token of the entry
  float uns[2 * MT];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    const int r = 16 * (rg * MT + x / 2) + 8 * (x % 2) + nn;
    node[x] = min((r0 + r) / gsz, n - 1);
    uns[x] = unscale[r];
  }
  const int live = R - r0 - 16 * MT * rg;  // rows of this warp (none: nothing to walk)
  bool upper[MT];                          // the second half of a tile holds rows
#pragma unroll
  for (int m = 0; m < MT; ++m) upper[m] = live > 16 * m + 8;

  float M[2 * MT], L[2 * MT], o[MT][8 * VC][4];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) M[x] = a.sx.logistic ? 0.f : -INFINITY, L[x] = 0.f;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int b = 0; b < 8 * VC; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[m][b][k] = 0.f;
  int P = 0;  // largest power of a value row so far (byte)

  const int window = a.sx.window > 0 ? a.sx.window : 0, keep = window ? max(a.sx.keep_first, 0) : 0;
  const int ntiles = (len + KT - 1) / KT;
  const int t_lo = window ? max(0, ctx - window + 1) / KT : 0;
  const int nkeep = min(min((keep + KT - 1) / KT, ntiles), t_lo);
  const int nwalk = live > 0 ? nkeep + ntiles - t_lo : 0;
  const int* pt = a.pt + (long long)e * a.max_pages;
  const long long kpitch = (long long)a.G * a.dim * sizeof(TC), vpitch = (long long)a.G * a.vdim * sizeof(TC);
  const uint8_t* kbase = a.kp + ((long long)g * a.dim) * sizeof(TC) + 16 * c;
  const uint8_t* vbase = a.vp + ((long long)g * a.vdim + 8 * nn) * sizeof(TC);
  const int stride = a.nsplit * wk, tpp = a.page / KT;
  auto tile_of = [&](int walk) { return walk < nkeep ? walk : t_lo + (walk - nkeep); };

  uint4 kk[NB][DC * K::KL];
  uint32_t kpow[KPL / 4], vpow[KPL / 4];
  auto load_keys = [&](int it, int pid) {
    const long long first = (long long)pid * a.page + (it % tpp) * KT;
#pragma unroll
    for (int f = 0; f < NB; ++f) {
      const uint8_t* p = kbase + (first + KPL * (nn >> 1) + 2 * f + (nn & 1)) * kpitch;
#pragma unroll
      for (int x = 0; x < DC * K::KL; ++x) {
        const int d = (64 * x + 16 * c) / (int)sizeof(TC);  // my first element of the piece
        kk[f][x] = d < a.dim ? *reinterpret_cast<const uint4*>(p + 64 * x) : make_uint4(0, 0, 0, 0);
      }
    }
    if (K::C8) {
      const long long at = ((long long)pid * a.G + g) * a.page + (it % tpp) * KT + KPL * c;
#pragma unroll
      for (int x = 0; x < KPL / 4; ++x) {
        kpow[x] = *reinterpret_cast<const uint32_t*>(a.ke + at + 4 * x);
        vpow[x] = *reinterpret_cast<const uint32_t*>(a.ve + at + 4 * x);
      }
    }
  };

  int walk = split * wk + kgrp;
  int pid = 0, pid_next = 0;
  if (walk < nwalk) {
    pid = pt[tile_of(walk) / tpp];
    if (walk + stride < nwalk) pid_next = pt[tile_of(walk + stride) / tpp];
    load_keys(tile_of(walk), pid);
  }
  for (; walk < nwalk; walk += stride) {
    const int it = tile_of(walk), j0 = it * KT;
    // values of the tile: rows KPL c .. + KPL - 1
    uint32_t vv[KPL][VC][K::VW];
    {
      const uint8_t* p = vbase + ((long long)pid * a.page + (it % tpp) * KT + KPL * c) * vpitch;
      const bool whole = j0 + KT <= len;
#pragma unroll
      for (int x = 0; x < KPL; ++x) {
        const bool there = whole || j0 + KPL * c + x < len;  // rows behind the last one hold anything
#pragma unroll
        for (int b = 0; b < VC; ++b) {
          const bool in = there && 64 * b + 8 * nn < a.vdim;
          const uint8_t* s = p + x * vpitch + 64 * b * sizeof(TC);
          if (K::VW == 2) {
            const uint2 u = in ? *reinterpret_cast<const uint2*>(s) : make_uint2(0, 0);
            vv[x][b][0] = u.x, vv[x][b][1] = u.y;
          } else {
#pragma unroll
            for (int y = 0; y < K::VW / 4; ++y) {
              const uint4 u = in ? *reinterpret_cast<const uint4*>(s + 16 * y) : make_uint4(0, 0, 0, 0);
              vv[x][b][4 * y] = u.x, vv[x][b][4 * y + 1] = u.y, vv[x][b][4 * y + 2] = u.z, vv[x][b][4 * y + 3] = u.w;
            }
          }
        }
      }
    }
    // ---- S = Q K^T
    float s[MT][NB][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int f = 0; f < NB; ++f)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[m][f][k] = 0.f;
#pragma unroll
    for (int st = 0; st < Q16; ++st) {
      uint4 qa[MT][K::QT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < K::QT; ++t) qa[m][t] = qs[((t * tiles_m + rg * MT + m) * Q16 + st) * 32 + lane];
#pragma unroll
      for (int f = 0; f < NB; ++f) {
        uint32_t b0[K::CT], b1[K::CT];
        if (K::C8) {
          const uint4 u = kk[f][st / 4];
          const uint32_t w = st % 4 == 0 ? u.x : st % 4 == 1 ? u.y : st % 4 == 2 ? u.z : u.w;
          b0[0] = cache8::halves_of(w);
          b1[0] = cache8::halves_of(w >> 16);
        } else if (K::F32) {
          const uint4 u = kk[f][K::F32 ? st : 0];
          terms<false>(__uint_as_float(u.x), __uint_as_float(u.y), b0);
          terms<false>(__uint_as_float(u.z), __uint_as_float(u.w), b1);
        } else {
          const uint4 u = kk[f][K::C8 || K::F32 ? 0 : st / 2];
          b0[0] = st % 2 == 0 ? u.x : u.z;
          b1[0] = st % 2 == 0 ? u.y : u.w;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = K::QT - 1; t >= 0; --t)  // small terms first
#pragma unroll
            for (int t2 = K::CT - 1; t2 >= 0; --t2)
              if (t + t2 < 3) mma<K::HALF>(s[m][f], qa[m][t], b0[t2], b1[t2]);
      }
    }
    uint32_t kpw[KPL / 4], vpw[KPL / 4];
    if (K::C8) {
#pragma unroll
      for (int x = 0; x < KPL / 4; ++x) kpw[x] = kpow[x], vpw[x] = vpow[x];
    }
    // the next tile's keys are under way from here on
    const int pid_now = pid;
    if (walk + stride < nwalk) {
      pid = pid_next;
      load_keys(tile_of(walk + stride), pid);
      if (walk + 2 * stride < nwalk) pid_next = pt[tile_of(walk + 2 * stride) / tpp];
    }
    // ---- who sees what
    const bool plain = j0 + KT <= ctx && (window == 0 || j0 > len - 1 - window || j0 + KT <= keep);
    uint32_t vis[2 * MT];
    if (!plain) {
      const int rel = j0 - ctx;
#pragma unroll
      for (int x = 0; x < 2 * MT; ++x) {
        const uint32_t* mask = a.tree != nullptr ? a.tree + (t0 + node[x]) * a.words : nullptr;
        auto word = [&](int w) -> uint32_t {  // drafted tokens 32 w .. 32 w + 31
          if (w < 0 || 32 * w >= n) return 0u;
          const int left = n - 32 * w;
          const uint32_t have = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
          if (mask != nullptr) return w < a.words ? mask[w] & have : 0u;
          const int upto = node[x] + 1 - 32 * w;
          return upto >= 32 ? have : upto <= 0 ? 0u : have & ((1u << upto) - 1u);
        };
        uint32_t v;
        if (rel >= 0) {
          const int w = rel >> 5, sh = rel & 31;
          v = word(w) >> sh;
          if (sh) v |= word(w + 1) << (32 - sh);
        } else if (rel > -32) {
          v = word(0) << -rel | ((1u << -rel) - 1u);
        } else {
          v = 0xffffffffu;
        }
        if (window) {
          const int p = a.pos[t0 + node[x]];
          for (int k = 0; k < KT; ++k) {
            const int j = j0 + k;
            const int pj = j < ctx ? j : j < len ? a.pos[t0 + (j - ctx)] : 0;
            if (!(p - pj < window || pj < keep)) v &= ~(1u << k);
          }
        }
        vis[x] = v;
      }
    }
    // ---- weights
    float kf[KPL];
    if (K::C8) {
#pragma unroll
      for (int x = 0; x < KPL; ++x) kf[x] = cache8::value_of_power(kpw[x / 4] >> (8 * (x % 4)) & 0xffu);
    }
    float vf[KPL];
    float grow = 1.f;  // 2^(P - new P)
    if (K::C8) {
      int top = 0;
#pragma unroll
      for (int x = 0; x < KPL; ++x)
        if (j0 + KPL * c + x < len) top = max(top, static_cast<int>(vpw[x / 4] >> (8 * (x % 4)) & 0xffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (top > P) {
        grow = top - P >= 127 ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - (top - P)) << 23);
        P = top;
      }
#pragma unroll
      for (int x = 0; x < KPL; ++x) {  // 2^(15 + power - P): a weight of one is 2^15, halves reach down to 2^-24
        const int b = static_cast<int>(vpw[x / 4] >> (8 * (x % 4)) & 0xffu) - P + 15 + 127;
        vf[x] = b > 0 && b < 143 ? __uint_as_float(static_cast<uint32_t>(b) << 23) : 0.f;
      }
    }
    uint4 pa[MT][NB / 2][K::PT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float corr[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int x = 2 * m + h;
        if (h == 1 && !upper[m]) {
#pragma unroll
          for (int f = 0; f < NB; ++f) s[m][f][2] = s[m][f][3] = 0.f;
          corr[1] = 1.f;
          continue;
        }
        const int rr = min(r0 + 16 * (rg * MT + m) + 8 * h + nn, R - 1);
        const int head = g * gsz + rr % gsz;
#pragma unroll
        for (int f = 0; f < NB; ++f)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v = s[m][f][2 * h + i] * uns[x];
            if (K::C8) v *= kf[2 * f + i];
            if (special) {
              if (a.softcap > 0.f) v = a.softcap * tanh_f32(v / a.softcap);
              if (a.sx.dist_a != nullptr) {
                const int j = j0 + KPL * c + 2 * f + i, pj = j < ctx || j >= len ? j : a.pos[t0 + (j - ctx)];
                v -= a.sx.dist_a[head] * log1pf(a.sx.dist_b[head] * (float)max(a.pos[t0 + node[x]] - pj, 0));
              }
              if (a.sx.logistic) {
                v = 1.0f / (1.0f + expf(-(v + (a.sx.head_bias != nullptr ? a.sx.head_bias[head] : 0.f))));
                if (!plain && !(vis[x] >> (KPL * c + 2 * f + i) & 1u)) v = 0.f;
                s[m][f][2 * h + i] = v;
                continue;
              }
              v *= kLog2e;
            }
            if (!plain && !(vis[x] >> (KPL * c + 2 * f + i) & 1u)) v = -INFINITY;
            s[m][f][2 * h + i] = v;
          }
        if (a.sx.logistic) {
          corr[h] = 1.f;
        } else {
          float mx = s[m][0][2 * h];
#pragma unroll
          for (int f = 0; f < NB; ++f) mx = fmaxf(mx, fmaxf(s[m][f][2 * h], s[m][f][2 * h + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float now = fmaxf(M[x], mx), ref = now == -INFINITY ? 0.f : now;  // nothing seen so far: weights of zero
          corr[h] = ex2(M[x] - ref);
          M[x] = now;
          float sum = 0.f;
#pragma unroll
          for (int f = 0; f < NB; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float p = ex2(s[m][f][2 * h + i] - ref);
              sum += p;
              s[m][f][2 * h + i] = p;
            }
          L[x] = L[x] * corr[h] + sum;
        }
        if (K::C8) {
#pragma unroll
          for (int f = 0; f < NB; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) s[m][f][2 * h + i] *= vf[2 * f + i];
          corr[h] *= grow;
        }
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int b = 0; b < 8 * VC; ++b) {
          o[m][b][0] *= corr[0], o[m][b][1] *= corr[0];
          o[m][b][2] *= corr[1], o[m][b][3] *= corr[1];
        }
      }
#pragma unroll
      for (int q = 0; q < NB / 2; ++q) {
        uint32_t p0[K::PT], p1[K::PT], p2[K::PT], p3[K::PT];
        terms<K::HALF>(s[m][2 * q][0], s[m][2 * q][1], p0);
        terms<K::HALF>(s[m][2 * q][2], s[m][2 * q][3], p1);
        terms<K::HALF>(s[m][2 * q + 1][0], s[m][2 * q + 1][1], p2);
        terms<K::HALF>(s[m][2 * q + 1][2], s[m][2 * q + 1][3], p3);
#pragma unroll
        for (int t = 0; t < K::PT; ++t) pa[m][q][t] = make_uint4(p0[t], p1[t], p2[t], p3[t]);
      }
    }
    // a value that is not a number reaches only the rows that see its key: in a tile with a mask such rows are taken out and added one by one
    if (!plain) {
#pragma unroll
      for (int x = 0; x < KPL; ++x) {
        bool bad = false;
#pragma unroll
        for (int b = 0; b < VC; ++b)
#pragma unroll
          for (int y = 0; y < K::VW; ++y) {
            const uint32_t w = vv[x][b][y];
            if (K::F32) bad |= (w & 0x7f800000u) == 0x7f800000u;
            else if (K::C8) bad |= (w & 0x7fu) == 0x7fu || (w & 0x7f00u) == 0x7f00u || (w & 0x7f0000u) == 0x7f0000u || (w & 0x7f000000u) == 0x7f000000u;
            else bad |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
          }
        uint32_t lanes = __ballot_sync(0xffffffffu, bad);
        lanes |= lanes >> 16;
        lanes |= lanes >> 8;
        lanes |= lanes >> 4;
        lanes &= 15u;  // bit c: key KPL c + x
        if (lanes == 0) continue;
        if (lanes >> c & 1u) {
#pragma unroll
          for (int b = 0; b < VC; ++b)
#pragma unroll
            for (int y = 0; y < K::VW; ++y) vv[x][b][y] = 0u;
        }
        for (int cc = 0; cc < 4; ++cc) {
          if (!(lanes >> cc & 1u)) continue;
          const uint8_t* row = a.vp + ((long long)pid_now * a.page + (it % tpp) * KT + KPL * cc + x) * vpitch + (long long)g * a.vdim * sizeof(TC);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const float w0 = __shfl_sync(0xffffffffu, s[m][x / 2][x % 2], 4 * nn + cc), w1 = __shfl_sync(0xffffffffu, s[m][x / 2][2 + x % 2], 4 * nn + cc);
#pragma unroll
            for (int b = 0; b < 8 * VC; ++b)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int col = 64 * (b / 8) + 16 * c + 8 * k + b % 8;
                if (col >= a.vdim) continue;
                float v;
                if (K::C8) {
                  const uint32_t two = cache8::halves_of(row[col]);
                  v = __low2float(*reinterpret_cast<const __half2*>(&two));
                } else if (K::F32) {
                  v = reinterpret_cast<const float*>(row)[col];
                } else {
                  v = __bfloat162float(reinterpret_cast<const bf16*>(row)[col]);
                }
                if (w0 != 0.f) o[m][b][k] = fmaf(w0, v, o[m][b][k]);
                if (w1 != 0.f) o[m][b][2 + k] = fmaf(w1, v, o[m][b][2 + k]);
              }
          }
        }
      }
    }
    // ---- O += P V
#pragma unroll
    for (int q = 0; q < NB / 2; ++q) {
#pragma unroll
      for (int b = 0; b < VC; ++b) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // column 8 n + y of the piece
          uint32_t b0[K::CT], b1[K::CT];
          const int x = 4 * q;
          if (K::C8) {
            const int w = y / 4, sel = y % 4;
            const uint32_t lo = __byte_perm(vv[x][b][w], vv[x + 1][b][w], sel < 2 ? 0x5140 : 0x7362), hi = __byte_perm(vv[x + 2][b][w], vv[x + 3][b][w], sel < 2 ? 0x5140 : 0x7362);
            b0[0] = cache8::halves_of(sel % 2 ? lo >> 16 : lo);
            b1[0] = cache8::halves_of(sel % 2 ? hi >> 16 : hi);
          } else if (K::F32) {
            const int w = K::F32 ? y : 0;
            terms<false>(__uint_as_float(vv[x][b][w]), __uint_as_float(vv[x + 1][b][w]), b0);
            terms<false>(__uint_as_float(vv[x + 2][b][w]), __uint_as_float(vv[x + 3][b][w]), b1);
          } else {
            const int w = K::C8 || K::F32 ? 0 : y / 2;
            b0[0] = __byte_perm(vv[x][b][w], vv[x + 1][b][w], y % 2 ? 0x7632 : 0x5410);
            b1[0] = __byte_perm(vv[x + 2][b][w], vv[x + 3][b][w], y % 2 ? 0x7632 : 0x5410);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = K::PT - 1; t >= 0; --t)
#pragma unroll
              for (int t2 = K::CT - 1; t2 >= 0; --t2)
                if (t + t2 < 3) mma<K::HALF>(o[m][8 * b + y], pa[m][q][t], b0[t2], b1[t2]);
        }
      }
    }
  }

  // ---- the warps' results into shared memory, then row by row
  __syncthreads();  // the queries are done with
  float* os = reinterpret_cast<float*>(raw);  // [warp][16 MT][vdim]
  const int ldo_s = a.vdim + 4;
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    float l = L[x];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int r = 16 * (x / 2) + 8 * (x % 2) + nn;
    if (c == 0) stat[warp][r] = make_float2(M[x], l);
    float* dst = os + (warp * 16 * MT + r) * ldo_s;
#pragma unroll
    for (int b = 0; b < VC; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = 64 * b + 16 * c + 8 * k;
        if (col < a.vdim) {
#pragma unroll
          for (int y = 0; y < 8; y += 4)
            *reinterpret_cast<float4*>(dst + col + y) = make_float4(o[x / 2][8 * b + y][2 * (x % 2) + k], o[x / 2][8 * b + y + 1][2 * (x % 2) + k], o[x / 2][8 * b + y + 2][2 * (x % 2) + k],
                                                                    o[x / 2][8 * b + y + 3][2 * (x % 2) + k]);
        }
      }
  }
  if (K::C8 && lane == 0) top_power[warp] = static_cast<float>(P);
  __syncthreads();
  const int rows_here = min(rows_cta, R - r0);
  const long long ldo = a.sx.out_ld > 0 ? a.sx.out_ld : (long long)a.H * a.vdim;
  const float oscale = a.sx.out_scale != 0.f ? a.sx.out_scale : 1.f;
  for (int idx = tid; idx < rows_here * a.vdim; idx += 32 * kWarps) {
    const int r = idx / a.vdim, col = idx - r * a.vdim, tile = r / (16 * MT), in = r % (16 * MT);
    const int rr = r0 + r, i = rr / gsz, head = g * gsz + rr - i * gsz;
    float m = -INFINITY;
    for (int w = 0; w < wk; ++w) m = fmaxf(m, stat[w * wr + tile][in].x);
    float acc = 0.f, l = 0.f;
    const float ref = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < wk; ++w) {
      const int ww = w * wr + tile;
      const float2 st = stat[ww][in];
      float f = ex2(st.x - ref);
      l += f * st.y;  // (scores that are no numbers stay in the sum)
      if (K::C8) f *= exp2f(top_power[ww] - 142.f);  // the weights' power: 2^(P - 127 - 15)
      if (f != 0.f) acc += f * os[(ww * 16 * MT + in) * ldo_s + col];
    }
    const long long t = t0 + i;
    if (a.nsplit == 1) {
      if (!a.sx.logistic && a.sx.sink != nullptr) {
        const float sk = a.sx.sink[head] * kLog2e, mm = fmaxf(ref, sk), f = ex2(ref - mm);
        acc *= f;
        l = l * f + ex2(sk - mm);
      }
      float v = (a.sx.logistic ? acc : l == 0.f ? 0.f : acc / l) * oscale;  // a row that sees nothing: zeros
      if (a.gate != nullptr) v /= 1.0f + expf(-ldf(static_cast<const TQ*>(a.gate) + t * a.ldg + (a.gate_per_head ? head : head * a.vdim + col)));
      stf(static_cast<TQ*>(a.out) + t * ldo + (long long)head * a.vdim + col, v);
    } else {
      const long long row = (a.singles ? (long long)e : t) * a.H + head;
      float* pp = a.partial + (row * a.nsplit + split) * (a.vdim + 4);
      pp[4 + col] = acc;
      if (col == 0) pp[0] = m, pp[1] = l;
    }
  }
}

// A warp a row: the splits' factors a lane each, then the columns, two a lane.
template <typename TQ>
__global__ void __launch_bounds__(128) attn_rows_merge_kernel(const __grid_constant__ Args a, int max_n) {
  pg::griddep_begin_if(a.trigger);
  const int e = blockIdx.y, lane = threadIdx.x & 31, w = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int n = a.n[e], i = w / a.H, head = w - i * a.H;
  if (i >= n || (a.singles && n != 1)) return;
  const long long t = a.row0[e] + i;
  const float* pp = a.partial + ((a.singles ? (long long)e : t) * a.H + head) * a.nsplit * (a.vdim + 4);
  const int ld = a.vdim + 4;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < a.nsplit; s += 32) m = fmaxf(m, pp[s * ld]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = lane; s < a.nsplit; s += 32) l += ex2(pp[s * ld] - ref) * pp[s * ld + 1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const float sk = !a.sx.logistic && a.sx.sink != nullptr ? a.sx.sink[head] * kLog2e : -INFINITY;
  const float mm = fmaxf(ref, sk), fix = ex2(ref - mm);
  if (sk > -INFINITY) l = l * fix + ex2(sk - mm);
  const long long ldo = a.sx.out_ld > 0 ? a.sx.out_ld : (long long)a.H * a.vdim;
  const float oscale = a.sx.out_scale != 0.f ? a.sx.out_scale : 1.f;
  for (int col = 2 * lane; col < a.vdim; col += 64) {
    float x = 0.f, y = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.nsplit; ++s) {
      const float f = ex2(pp[s * ld] - ref);
      const float2 v = *reinterpret_cast<const float2*>(pp + s * ld + 4 + col);
      if (f != 0.f) x = fmaf(f, v.x, x), y = fmaf(f, v.y, y);
    }
    if (sk > -INFINITY) x *= fix, y *= fix;
    if (!a.sx.logistic) x = l == 0.f ? 0.f : x / l, y = l == 0.f ? 0.f : y / l;
    x *= oscale, y *= oscale;
    if (a.gate != nullptr) {
      const TQ* gt = static_cast<const TQ*>(a.gate) + t * a.ldg + (a.gate_per_head ? head : head * a.vdim + col);
      x /= 1.0f + expf(-ldf(gt));
      y /= 1.0f + expf(-ldf(gt + (a.gate_per_head ? 0 : 1)));
    }
    TQ* dst = static_cast<TQ*>(a.out) + t * ldo + (long long)head * a.vdim + col;
    stf(dst, x);
    stf(dst + 1, y);
  }
}

template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
int launch(Args a, int entries, int max_n, cudaStream_t st) {
  using K = Kind<TQ, TC>;
  const int rows = max_n * (a.H / a.G);
  int wr = 1;
  while (wr < kWarps && wr * 16 * MT < rows) wr *= 2;
  a.wr = wr;
  a.blocks = (rows + wr * 16 * MT - 1) / (wr * 16 * MT);
  const size_t qb = (size_t)K::QT * wr * MT * 4 * DC * 512, ob = (size_t)kWarps * 16 * MT * (a.vdim + 4) * 4;
  const size_t smem = qb > ob ? qb : ob;
  if ((long long)a.blocks * a.G > 65535) return PG_ERR_ARG;
  auto kern = attn_rows_kernel<TQ, TC, DC, VC, MT, KT>;
  constexpr int kMost = 128 * 1024;
  if (smem > kMost) return PG_ERR_ARG;
  static bool configured[pg::kMaxDevices] = {};  // once a device, to the most that any call asks for
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  if (pg::launch_kernel(kern, dim3(a.nsplit, a.G * a.blocks, entries), dim3(32 * kWarps), smem, st, a) != cudaSuccess) return PG_ERR_CUDA;
  if (a.nsplit > 1) {
    const int most = a.singles ? 1 : max_n;
    if (pg::launch_kernel(attn_rows_merge_kernel<TQ>, dim3((most * a.H + 3) / 4, entries), dim3(128), 0, st, a, most) != cudaSuccess) return PG_ERR_CUDA;
  }
  return PG_OK;
}

template <typename TQ, typename TC, int MT, int KT>
int by_size(const Args& a, int entries, int max_n, cudaStream_t st) {
  if (a.dim <= 64 && a.vdim <= 64) return launch<TQ, TC, 1, 1, MT, KT>(a, entries, max_n, st);
  constexpr int kWide = sizeof(TC) == 1 ? KT : 16;  // (keys and values of a tile stay in registers)
  return launch<TQ, TC, 2, 2, MT, kWide>(a, entries, max_n, st);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" long long pg_attn_rows_scratch(int rows, int H, int vdim, int nsplit) { return nsplit > 1 ? 4LL * rows * H * nsplit * (vdim + 4) : 0; }

extern "C" int pg_attn_rows(const void* q, const PgKvPages* kv, const void* gate, long long ldg, void* out, float* partial, const int* entry_row0, const int* entry_n,
                            const int* entry_ctx, const int* page_table, int max_pages, int page, const int* pos, const void* tree, int tree_words, int entries, int max_n,
                            int singles, int nsplit, int H, int G, int dim, int vdim, float scale, float softcap, int act_f32, int gate_per_head, const PgAttnScore* score,
                            void* stream) {
  if (kv == nullptr || entries <= 0 || entries > 65535 || max_n <= 0 || nsplit <= 0 || nsplit > 65535 || H <= 0 || G <= 0 || H % G != 0 || dim <= 0 || vdim <= 0 || max_pages <= 0)
    return PG_ERR_ARG;
  if (page <= 0 || page % 32 != 0 || dim > 128 || vdim > 128 || (tree != nullptr && tree_words <= 0) || (nsplit > 1 && partial == nullptr)) return PG_ERR_ARG;
  const int unit = kv->e4m3 ? 16 : act_f32 ? 4 : 8;  // elements of a 16-byte piece
  if (dim % unit != 0 || vdim % 8 != 0 || ((long long)G * dim) % unit != 0 || !aligned(kv->k, 16) || !aligned(kv->v, 16)) return PG_ERR_ARG;
  if (kv->e4m3 && (kv->k_powers == nullptr || kv->v_powers == nullptr || !aligned(kv->k_powers, 8) || !aligned(kv->v_powers, 8))) return PG_ERR_ARG;
  if (!kv->e4m3 && kv->f32 != act_f32) return PG_ERR_ARG;
  if (nsplit > 1 && !aligned(partial, 8)) return PG_ERR_ARG;
  if (score != nullptr && ((score->dist_a == nullptr) != (score->dist_b == nullptr))) return PG_ERR_ARG;
  if (pos == nullptr && score != nullptr && (score->window > 0 || score->dist_a != nullptr)) return PG_ERR_ARG;
  Args a{};
  a.q = q;
  a.kp = static_cast<const uint8_t*>(kv->k), a.vp = static_cast<const uint8_t*>(kv->v);
  a.ke = static_cast<const uint8_t*>(kv->k_powers), a.ve = static_cast<const uint8_t*>(kv->v_powers);
  a.gate = gate, a.ldg = ldg, a.out = out, a.partial = partial;
  a.row0 = entry_row0, a.n = entry_n, a.ctx = entry_ctx, a.pt = page_table, a.pos = pos, a.tree = static_cast<const uint32_t*>(tree);
  a.words = tree_words, a.max_pages = max_pages, a.page = page, a.singles = singles, a.nsplit = nsplit, a.H = H, a.G = G, a.dim = dim, a.vdim = vdim;
  a.scale = scale, a.softcap = softcap, a.gate_per_head = gate_per_head;
  a.sx = score != nullptr ? *score : PgAttnScore{};
  a.trigger = pg::weights_follow();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int most = singles ? 1 : max_n, rows = most * (H / G);
  if (kv->e4m3) {
    if (act_f32) return by_size<float, e4m3, 1, 32>(a, entries, most, st);
    return rows <= 16 ? by_size<bf16, e4m3, 1, 32>(a, entries, most, st) : by_size<bf16, e4m3, 2, 32>(a, entries, most, st);
  }
  if (act_f32) return by_size<float, float, 1, 16>(a, entries, most, st);
  return rows <= 16 ? by_size<bf16, bf16, 1, 32>(a, entries, most, st) : by_size<bf16, bf16, 2, 32>(a, entries, most, st);
}
