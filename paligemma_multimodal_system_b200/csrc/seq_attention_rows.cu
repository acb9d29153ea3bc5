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

// what comes between a score and its weight: nothing, a soft cap, or any of the options
enum { kPlain = 0, kCapped = 1, kGeneral = 2 };

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
  int words, max_pages, page, tile_shift, singles, nsplit, blocks, H, G, dim, vdim, wr, mode;  // tile_shift: log2 of a page's tiles; mode: below
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

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
struct Kind {
  static constexpr int ES = sizeof(TC);
  static constexpr bool C8 = ES == 1, F32 = ES == 4, HALF = C8;
  static constexpr int QT = F32 ? 3 : (C8 && sizeof(TQ) == 4) ? 2 : 1;     // terms of a query
  static constexpr int CT = F32 ? 3 : 1;                                   // terms of a cached element
  static constexpr int PT = F32 ? 3 : C8 ? (sizeof(TQ) == 4 ? 2 : 1) : 2;  // terms of a weight
  static constexpr int VW = 2 * ES;                                        // words of eight value columns
  static constexpr int KROW = 64 * DC * ES, VROW = 64 * VC * ES;           // bytes of a row in shared memory
  static constexpr int STAGE = KT * (KROW + VROW) + (C8 ? 2 * KT : 0);
  static constexpr int STAGES = STAGE > 8 * 1024 + 256 ? 2 : 3;
  static constexpr int Q_BYTES = QT * MT * 4 * DC * 512;  // of a warp's rows
};

// what registers and shared memory leave room for
template <typename TQ, typename TC, int DC, int VC, int MT>
constexpr int ctas_per_sm() {
#ifndef OCC
#define OCC 4
#endif
#ifndef OCCW
#define OCCW 2
#endif
#ifndef OCCM
#define OCCM 3
#endif
  return DC > 1 || VC > 1 ? OCCW : sizeof(TC) == 4 ? 2 : MT == 2 ? OCCM : sizeof(TC) == 1 ? OCC : 2;
}

// A 16-byte piece's place in a tile.  Keys: two neighbouring rows are read together, pieces 4 x .. 4 x + 3 of each: rows of 128 bytes and more turn the odd row's by four.  Values:
// four rows KPL apart are read together: each takes other banks.
template <int ROW>
__device__ __forceinline__ uint32_t key_place(int row, int piece) {
  return row * ROW + 16 * (ROW >= 128 ? piece ^ ((row & 1) << 2) : piece);
}
template <int ROW, int KPL, int ES>
__device__ __forceinline__ uint32_t value_place(int row, int piece) {
  const int c = row / KPL, turn = ES == 4 ? (c & 1) | (c >> 1) << 2 : 2 * c;
  if (ROW == 64) return (row >> 1) * 128 + 16 * (((row & 1) * 4 + piece) ^ turn);
  return row * ROW + 16 * (piece ^ turn);
}

// DC, VC: 64-element pieces of a key / value row; MT: 16-row tiles of a warp; KT: keys of a tile
template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
__global__ void __launch_bounds__(32 * kWarps, (ctas_per_sm<TQ, TC, DC, VC, MT>())) attn_rows_kernel(const __grid_constant__ Args a) {
  using K = Kind<TQ, TC, DC, VC, MT, KT>;
  constexpr int NB = KT / 8, KPL = KT / 4;  // key fragments of a tile; keys of a lane
  constexpr int Q16 = 4 * DC;
  extern __shared__ __align__(128) unsigned char raw[];
  __shared__ float unscale[kWarps * 16 * MT];  // what a row's scores are multiplied by
  __shared__ float2 stat[kWarps][16 * MT];
  __shared__ float top_power[kWarps];
  // the step's descriptors are there before its first kernel
  const int split = blockIdx.x, g = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, e = blockIdx.z;
  const int n = a.n[e], ctx = a.ctx[e], gsz = a.H / a.G, len = ctx + n;
  const long long t0 = a.row0[e];
  const int wr = a.wr, wk = kWarps / wr, rows_cta = wr * 16 * MT, r0 = block * rows_cta, R = n * gsz;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nn = lane >> 2, c = lane & 3;
  const int rg = warp % wr, kgrp = warp / wr;
  const bool mine = !(a.singles && n != 1) && r0 < R;
  const int live = mine ? R - r0 - 16 * MT * rg : 0;  // rows of this warp (none: nothing to walk)

  // ---- the key walk
  const int window = a.sx.window > 0 ? a.sx.window : 0, keep = window ? max(a.sx.keep_first, 0) : 0;
  const int ntiles = (len + KT - 1) / KT;
  const int t_lo = window ? max(0, ctx - window + 1) / KT : 0;
  const int nkeep = min(min((keep + KT - 1) / KT, ntiles), t_lo);
  const int nwalk = live > 0 ? nkeep + ntiles - t_lo : 0;
  const int* pt = a.pt + (long long)e * a.max_pages;
  const int stride = a.nsplit * wk, tpp = 1 << a.tile_shift, walk0 = split * wk + kgrp;
  auto tile_of = [&](int walk) { return walk < nkeep ? walk : t_lo + (walk - nkeep); };
  // page numbers of 32 tiles of the walk, a lane each
  auto pages_from = [&](int walk) {
    const int w = walk + lane * stride;
    return w < nwalk ? pt[tile_of(w) >> a.tile_shift] : 0;
  };
  int pids = pages_from(walk0);
  if (a.nsplit > 1) pg::griddep_begin<true>();  // (fp32 partials, read behind a wait)
  else pg::griddep_begin_if(a.trigger);
  if (!mine) return;

  // ---- copies: a ring of tiles a warp, 16 bytes a lane and request
  unsigned char* ring = raw + wr * K::Q_BYTES + warp * (K::STAGES * K::STAGE);
  const long long kpitch = (long long)a.G * a.dim * K::ES, vpitch = (long long)a.G * a.vdim * K::ES;
  const int kbytes = a.dim * K::ES, vbytes = a.vdim * K::ES;
  auto request = [&](int k, int it, int pid) {  // tile `it` into stage k % STAGES
    const uint32_t dst = pg::smem_u32(ring + (k % K::STAGES) * K::STAGE);
    const long long first = (long long)pid * a.page + (it & (tpp - 1)) * KT;
    constexpr int KP = K::KROW / 16, VP = K::VROW / 16;
    {
      const int row = lane / KP, piece = lane % KP;
      const uint8_t* p = a.kp + (first + row) * kpitch + (long long)g * kbytes + 16 * piece;
      const bool in = 16 * piece < kbytes;
#pragma unroll
      for (int i = 0; i < KT * KP / 32; ++i) {
        const int r = row + i * (32 / KP);
        pg::cp_async16(dst + key_place<K::KROW>(r, piece), p, in);
        p += (32 / KP) * kpitch;
      }
    }
    {
      const int row = lane / VP, piece = lane % VP;
      const uint8_t* p = a.vp + (first + row) * vpitch + (long long)g * vbytes + 16 * piece;
      const bool in = 16 * piece < vbytes;
      const int left = len - it * KT;  // rows behind the last one hold anything: zeros
#pragma unroll
      for (int i = 0; i < KT * VP / 32; ++i) {
        const int r = row + i * (32 / VP);
        pg::cp_async16(dst + KT * K::KROW + value_place<K::VROW, KPL, K::ES>(r, piece), p, in && r < left);
        p += (32 / VP) * vpitch;
      }
    }
    if (K::C8 && lane < KT / 8) {  // the powers: keys' in the first half of these lanes, values' in the second
      const bool is_v = lane >= KT / 16;
      const uint8_t* p = (is_v ? a.ve : a.ke) + ((long long)pid * a.G + g) * a.page + (it & (tpp - 1)) * KT + 16 * (lane % (KT / 16));
      pg::cp_async16(dst + KT * (K::KROW + K::VROW) + 16 * lane, p, true);
    }
  };
#pragma unroll
  for (int k = 0; k < K::STAGES - 1; ++k) {
    const int w = walk0 + k * stride, pid = __shfl_sync(0xffffffffu, pids, k);
    if (w < nwalk) request(k, tile_of(w), pid);
    pg::cp_async_commit();
  }

  // ---- queries: fragments in the order of the cache's pieces; four elements a lane, a warp takes every fourth row, one trip to memory
  uint4* qs = reinterpret_cast<uint4*>(raw);  // [term][row tile][step][lane]
  const int tiles_m = wr * MT;
  constexpr int QL = DC == 1 ? 16 : 32;       // lanes of a row
  constexpr int RW = 32 / QL;                 // rows a warp and pass
#pragma unroll 4
  for (int rb = 0; rb < rows_cta; rb += kWarps * RW) {
    const int r = rb + warp * RW + lane / QL, w = lane % QL;
    const int rr = r0 + r;
    const bool in = rr < R;
    const int i = in ? rr / gsz : 0, head = g * gsz + (in ? rr - i * gsz : 0);
    const int st = w / 4, cc = w % 4;
    const int d0 = K::C8 ? 64 * (st / 4) + 16 * cc + 4 * (st % 4) : K::F32 ? 16 * st + 4 * cc : 32 * (st / 2) + 8 * cc + 4 * (st % 2);
    const TQ* q = static_cast<const TQ*>(a.q) + (t0 + i) * (long long)a.H * a.dim + (long long)head * a.dim + d0;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = in && d0 + k < a.dim ? ldf(q + k) : 0.f;
    float s = a.scale * (a.sx.head_scale != nullptr ? a.sx.head_scale[head] : 1.f);
    if (K::C8) {
      float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
      for (int o = QL / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // largest element to [2^14, 2^15): a half keeps eleven bits down to 2^-14, and 2^-24 below
      const int x = min(max(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100);
      const float up = __uint_as_float(static_cast<uint32_t>(x + 127) << 23);
      s *= __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= up;
    }
    if (w == 0) unscale[r] = a.mode == kGeneral ? s : a.mode == kCapped ? s * (2.f * kLog2e / a.softcap) : s * kLog2e;
    uint32_t p[K::QT], s2[K::QT];
    terms<K::HALF>(v[0], v[1], p);
    terms<K::HALF>(v[2], v[3], s2);
#pragma unroll
    for (int t = 0; t < K::QT; ++t) {  // row r of its tile: lanes 4 (r % 8) + c, first or second half of the fragment's registers
      uint32_t* f = reinterpret_cast<uint32_t*>(qs + ((t * tiles_m + r / 16) * Q16 + st) * 32 + 4 * (r % 8) + cc) + (r % 16 < 8 ? 0 : 1);
      f[0] = p[t];
      f[2] = s2[t];
    }
  }
  __syncthreads();

  // ---- my rows
  int node[2 * MT];  // token of the entry
  float uns[2 * MT];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    const int r = 16 * (rg * MT + x / 2) + 8 * (x % 2) + nn;
    node[x] = min((r0 + r) / gsz, n - 1);
    uns[x] = unscale[r];
  }
  bool upper[MT];  // the second half of a tile holds rows
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

  // one tile; PLAIN: every row sees every key of it
  auto step = [&](auto plain_tag, int it, const unsigned char* stage) {
    constexpr bool PLAIN = decltype(plain_tag)::value;
    const int j0 = it * KT;
    // ---- S = Q K^T
    float s[MT][NB][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int f = 0; f < NB; ++f)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[m][f][k] = 0.f;
    constexpr int SPL = K::C8 ? 4 : K::F32 ? 1 : 2;  // 16-deep steps of a piece
#pragma unroll
    for (int x = 0; x < Q16 / SPL; ++x) {
      uint4 kk[NB];
#pragma unroll
      for (int f = 0; f < NB; ++f) kk[f] = *reinterpret_cast<const uint4*>(stage + key_place<K::KROW>(KPL * (nn >> 1) + 2 * f + (nn & 1), 4 * x + c));
#pragma unroll
      for (int y = 0; y < SPL; ++y) {
        const int st = SPL * x + y;
        uint4 qa[MT][K::QT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < K::QT; ++t) qa[m][t] = qs[((t * tiles_m + rg * MT + m) * Q16 + st) * 32 + lane];
#pragma unroll
        for (int f = 0; f < NB; ++f) {
          uint32_t b0[K::CT], b1[K::CT];
          const uint4 u = kk[f];
          if (K::C8) {
            const uint32_t w = y == 0 ? u.x : y == 1 ? u.y : y == 2 ? u.z : u.w;
            b0[0] = cache8::halves_of(w);
            b1[0] = cache8::halves_of(w >> 16);
          } else if (K::F32) {
            terms<false>(__uint_as_float(u.x), __uint_as_float(u.y), b0);
            terms<false>(__uint_as_float(u.z), __uint_as_float(u.w), b1);
          } else {
            b0[0] = y == 0 ? u.x : u.z;
            b1[0] = y == 0 ? u.y : u.w;
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
    }
    // ---- who sees what
    uint32_t vis[2 * MT];
    if (!PLAIN) {
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
    float kf[KPL], vf[KPL];
    float grow = 1.f;  // 2^(P - new P)
    if (K::C8) {
      uint32_t kpw[KPL / 4], vpw[KPL / 4];
#pragma unroll
      for (int x = 0; x < KPL / 4; ++x) {
        kpw[x] = *reinterpret_cast<const uint32_t*>(stage + KT * (K::KROW + K::VROW) + KPL * c + 4 * x);
        vpw[x] = *reinterpret_cast<const uint32_t*>(stage + KT * (K::KROW + K::VROW) + KT + KPL * c + 4 * x);
      }
#pragma unroll
      for (int x = 0; x < KPL; ++x) kf[x] = __uint_as_float((kpw[x / 4] >> (8 * (x % 4)) & 0xffu) << 23);  // (byte 0: what is below 2^-118 counts as zero)
      uint32_t most = 0;
#pragma unroll
      for (int x = 0; x < KPL / 4; ++x) {
        uint32_t w = vpw[x];
        if (!PLAIN) {  // rows behind the last one hold anything
          const int left = len - j0 - KPL * c - 4 * x;
          w = left >= 4 ? w : left <= 0 ? 0u : w & ((1u << (8 * left)) - 1u);
          vpw[x] = w;
        }
        most = __vmaxu4(most, w);
      }
      most = __vmaxu4(most, most >> 16);
      most = max(most & 0xffu, most >> 8 & 0xffu);
      int top = static_cast<int>(most);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (top > P) {
        grow = top - P >= 127 ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - (top - P)) << 23);
        P = top;
      }
      const int lift = 142 - P;  // 2^(15 + power - P): a weight of one is 2^15, halves reach down to 2^-24
#pragma unroll
      for (int x = 0; x < KPL; ++x) vf[x] = __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(vpw[x / 4] >> (8 * (x % 4)) & 0xffu) + lift, 0)) << 23);
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
#pragma unroll
        for (int f = 0; f < NB; ++f)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v = s[m][f][2 * h + i] * uns[x];
            if (K::C8) v *= kf[2 * f + i];
            s[m][f][2 * h + i] = v;
          }
        if (a.mode == kCapped) {  // cap tanh(v / cap) in log2 units; v comes as 2 log2(e) v / cap
          const float cap = a.softcap * kLog2e;
#pragma unroll
          for (int f = 0; f < NB; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float v = s[m][f][2 * h + i];
              if (sizeof(TQ) == 2) s[m][f][2 * h + i] = fmaf(-2.f * cap, rcp(ex2(v) + 1.f), cap);  // off by 2^-22 cap: the output's rounding is 2^-9
              else s[m][f][2 * h + i] = cap * tanh_f32(v * (0.5f / kLog2e));
            }
        } else if (a.mode == kGeneral) {
          const int head = g * gsz + min(r0 + 16 * (rg * MT + m) + 8 * h + nn, R - 1) % gsz;
#pragma unroll 1
          for (int f = 0; f < NB; ++f) {
            float two[2];
#pragma unroll
            for (int y = 0; y < NB; ++y)
              if (y == f) two[0] = s[m][y][2 * h], two[1] = s[m][y][2 * h + 1];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float v = two[i];
              if (a.softcap > 0.f) v = a.softcap * tanh_f32(v / a.softcap);
              if (a.sx.dist_a != nullptr) {
                const int j = j0 + KPL * c + 2 * f + i, pj = j < ctx || j >= len ? j : a.pos[t0 + (j - ctx)];
                v -= a.sx.dist_a[head] * log1pf(a.sx.dist_b[head] * (float)max(a.pos[t0 + node[x]] - pj, 0));
              }
              if (a.sx.logistic) v = 1.0f / (1.0f + expf(-(v + (a.sx.head_bias != nullptr ? a.sx.head_bias[head] : 0.f))));
              else v *= kLog2e;
              two[i] = v;
            }
#pragma unroll
            for (int y = 0; y < NB; ++y)
              if (y == f) s[m][y][2 * h] = two[0], s[m][y][2 * h + 1] = two[1];
          }
        }
        if (!PLAIN) {
          const float nothing = a.sx.logistic ? 0.f : -INFINITY;
#pragma unroll
          for (int f = 0; f < NB; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (!(vis[x] >> (KPL * c + 2 * f + i) & 1u)) s[m][f][2 * h + i] = nothing;
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
    // ---- O += P V: rows KPL c + 4 q .. + 3 of the tile, columns 8 n .. 8 n + 7 of every 64
    const unsigned char* vt = stage + KT * K::KROW;
#pragma unroll
    for (int q = 0; q < NB / 2; ++q) {
      uint32_t vv[4][VC][K::VW];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int b = 0; b < VC; ++b) {
          const int row = KPL * c + 4 * q + x;
          if (K::C8) {
            const uint2 u = *reinterpret_cast<const uint2*>(vt + value_place<K::VROW, KPL, K::ES>(row, 4 * b + (nn >> 1)) + 8 * (nn & 1));
            vv[x][b][0] = u.x, vv[x][b][1] = u.y;
          } else {
#pragma unroll
            for (int y = 0; y < K::VW / 4; ++y) {
              const uint4 u = *reinterpret_cast<const uint4*>(vt + value_place<K::VROW, KPL, K::ES>(row, (K::F32 ? 16 * b + 2 * nn : 8 * b + nn) + y));
              vv[x][b][4 * y] = u.x, vv[x][b][4 * y + 1] = u.y, vv[x][b][4 * y + 2] = u.z, vv[x][b][4 * y + 3] = u.w;
            }
          }
        }
      // a value that is not a number reaches only the rows that see its key: in a tile with a mask such rows are taken out and added one by one
      if (!PLAIN) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
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
          lanes &= 15u;  // bit c: key KPL c + 4 q + x
          if (lanes == 0) continue;
          if (lanes >> c & 1u) {
#pragma unroll
            for (int b = 0; b < VC; ++b)
#pragma unroll
              for (int y = 0; y < K::VW; ++y) vv[x][b][y] = 0u;
          }
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            if (!(lanes >> cc & 1u)) continue;
            const int row = KPL * cc + 4 * q + x;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const float w0 = __shfl_sync(0xffffffffu, s[m][2 * q + x / 2][x % 2], 4 * nn + cc), w1 = __shfl_sync(0xffffffffu, s[m][2 * q + x / 2][2 + x % 2], 4 * nn + cc);
#pragma unroll
              for (int b = 0; b < 8 * VC; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int byte = (64 * (b / 8) + 16 * c + 8 * k + b % 8) * K::ES;  // my column's
                  const unsigned char* at = vt + value_place<K::VROW, KPL, K::ES>(row, byte / 16) + byte % 16;
                  float v;
                  if (K::C8) {
                    const uint32_t two = cache8::halves_of(*at);
                    v = __low2float(*reinterpret_cast<const __half2*>(&two));
                  } else if (K::F32) {
                    v = *reinterpret_cast<const float*>(at);
                  } else {
                    v = __bfloat162float(*reinterpret_cast<const bf16*>(at));
                  }
                  if (w0 != 0.f) o[m][b][k] = fmaf(w0, v, o[m][b][k]);
                  if (w1 != 0.f) o[m][b][2 + k] = fmaf(w1, v, o[m][b][2 + k]);
                }
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < VC; ++b) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // column 8 n + y of the piece
          uint32_t b0[K::CT], b1[K::CT];
          if (K::C8) {
            const int w = y / 4, sel = y % 4;
            const uint32_t lo = __byte_perm(vv[0][b][w], vv[1][b][w], sel < 2 ? 0x5140 : 0x7362), hi = __byte_perm(vv[2][b][w], vv[3][b][w], sel < 2 ? 0x5140 : 0x7362);
            b0[0] = cache8::halves_of(sel % 2 ? lo >> 16 : lo);
            b1[0] = cache8::halves_of(sel % 2 ? hi >> 16 : hi);
          } else if (K::F32) {
            const int w = K::F32 ? y : 0;
            terms<false>(__uint_as_float(vv[0][b][w]), __uint_as_float(vv[1][b][w]), b0);
            terms<false>(__uint_as_float(vv[2][b][w]), __uint_as_float(vv[3][b][w]), b1);
          } else {
            const int w = K::C8 || K::F32 ? 0 : y / 2;
            b0[0] = __byte_perm(vv[0][b][w], vv[1][b][w], y % 2 ? 0x7632 : 0x5410);
            b1[0] = __byte_perm(vv[2][b][w], vv[3][b][w], y % 2 ? 0x7632 : 0x5410);
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
  };
#pragma unroll 1
  for (int k = 0, walk = walk0; walk < nwalk; ++k, walk += stride) {
    pg::cp_async_wait<K::STAGES - 2>();
    __syncwarp();  // tile k is here for all lanes, and all are done with the tile before
    const int ahead = k + K::STAGES - 1;
    if ((ahead & 31) == 0) pids = pages_from(walk0 + ahead * stride);
    const int wa = walk0 + ahead * stride, pid = __shfl_sync(0xffffffffu, pids, ahead & 31);
    if (wa < nwalk) request(ahead, tile_of(wa), pid);
    pg::cp_async_commit();
    const int it = tile_of(walk), j0 = it * KT;
    const unsigned char* stage = ring + (k % K::STAGES) * K::STAGE;
    if (j0 + KT <= ctx && (window == 0 || j0 > len - 1 - window || j0 + KT <= keep)) step(Yes{}, it, stage);
    else step(No{}, it, stage);
  }

  // ---- the warps' results into shared memory, then row by row
  pg::cp_async_wait<0>();
  __syncthreads();  // queries and tiles are done with
  float* os = reinterpret_cast<float*>(raw);  // [warp][16 MT][vdim + 4]
  const int ldo_s = a.vdim + 4;
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    float l = L[x];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int r = 16 * (x / 2) + 8 * (x % 2) + nn;
    if (c == 0) stat[warp][r] = make_float2(M[x], l);
    if (x % 2 == 1 && !upper[x / 2]) continue;
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
  const int quads = a.vdim / 4;  // four columns a thread
  for (int idx = tid; idx < rows_here * quads; idx += 32 * kWarps) {
    const int r = idx / quads, col = 4 * (idx - r * quads), tile = r / (16 * MT), in = r % (16 * MT);
    const int rr = r0 + r, i = rr / gsz, head = g * gsz + rr - i * gsz;
    const long long t = t0 + i;
    const TQ* gt = static_cast<const TQ*>(a.gate) + t * a.ldg + (a.gate_per_head ? head : head * a.vdim + col);
    float gv[4];
    if (a.nsplit == 1 && a.gate != nullptr) {
#pragma unroll
      for (int y = 0; y < 4; ++y) gv[y] = ldf(gt + (a.gate_per_head ? 0 : y));
    }
    float m = -INFINITY;
    for (int w = 0; w < wk; ++w) m = fmaxf(m, stat[w * wr + tile][in].x);
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
    const float ref = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < wk; ++w) {
      const int ww = w * wr + tile;
      const float2 st = stat[ww][in];
      float f = ex2(st.x - ref);
      l += f * st.y;  // (scores that are no numbers stay in the sum)
      if (K::C8) f *= exp2f(top_power[ww] - 142.f);  // the weights' power: 2^(P - 127 - 15)
      if (f != 0.f) {
        const float4 v = *reinterpret_cast<const float4*>(os + (ww * 16 * MT + in) * ldo_s + col);
        acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
      }
    }
    if (a.nsplit == 1) {
      if (!a.sx.logistic && a.sx.sink != nullptr) {
        const float sk = a.sx.sink[head] * kLog2e, mm = fmaxf(ref, sk), f = ex2(ref - mm);
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[y] *= f;
        l = l * f + ex2(sk - mm);
      }
      TQ* dst = static_cast<TQ*>(a.out) + t * ldo + (long long)head * a.vdim + col;
      const float inv = a.sx.logistic ? 1.f : l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        float v = acc[y] * inv * oscale;
        if (a.gate != nullptr) v /= 1.0f + expf(-gv[y]);
        stf(dst + y, v);
      }
    } else {
      const long long row = (a.singles ? (long long)e : t) * a.H + head;
      float* pp = a.partial + (row * a.nsplit + split) * (a.vdim + 4);
      *reinterpret_cast<float4*>(pp + 4 + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (col == 0) *reinterpret_cast<float2*>(pp) = make_float2(m, l);
    }
  }
}

// A CTA a row: its warps take every fourth split, four columns a lane (vdim <= 128), the first splits' values requested before their factors are known.
template <typename TQ>
__global__ void __launch_bounds__(128) attn_rows_merge_kernel(const __grid_constant__ Args a) {
  constexpr int AHEAD = 8;
  __shared__ float4 sums[4][32];
  __shared__ float fs[64];
  __shared__ float whole[2];
  const int e = blockIdx.z, head = blockIdx.x, i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = a.n[e];
  const long long t = a.row0[e] + i;
  pg::griddep_begin_if(a.trigger);
  if (i >= n || (a.singles && n != 1)) return;
  const int ld = a.vdim + 4, col = 4 * lane;
  const float* pp = a.partial + ((a.singles ? (long long)e : t) * a.H + head) * a.nsplit * ld;
  float4 ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (warp + 4 * k < a.nsplit && col < a.vdim) ahead[k] = *reinterpret_cast<const float4*>(pp + (warp + 4 * k) * ld + 4 + col);
  if (warp == 0) {  // (at most 64 splits: two a lane)
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 x = lane < a.nsplit ? *reinterpret_cast<const float2*>(pp + lane * ld) : none, y = lane + 32 < a.nsplit ? *reinterpret_cast<const float2*>(pp + (lane + 32) * ld) : none;
    float m = fmaxf(x.x, y.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.f : m, fx = ex2(x.x - ref), fy = ex2(y.x - ref);
    float l = fx * x.y + fy * y.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float fix = 1.f;
    if (!a.sx.logistic && a.sx.sink != nullptr) {
      const float sk = a.sx.sink[head] * kLog2e, mm = fmaxf(ref, sk);
      fix = ex2(ref - mm);
      l = l * fix + ex2(sk - mm);
    }
    const float oscale = a.sx.out_scale != 0.f ? a.sx.out_scale : 1.f;
    fs[lane] = fx;
    fs[lane + 32] = fy;
    if (lane == 0) whole[0] = (a.sx.logistic ? 1.f : l == 0.f ? 0.f : fix / l) * oscale;
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < a.vdim) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int s = warp + 4 * k;
      if (s >= a.nsplit) break;
      const float f = fs[s];
      if (f == 0.f) continue;  // (a split without keys left zeros)
      const float4 v = k < AHEAD ? ahead[k % AHEAD] : *reinterpret_cast<const float4*>(pp + s * ld + 4 + col);
      acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    }
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && col < a.vdim) {
    float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 x = sums[w][lane];
      v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
    }
    const long long ldo = a.sx.out_ld > 0 ? a.sx.out_ld : (long long)a.H * a.vdim;
    TQ* dst = static_cast<TQ*>(a.out) + t * ldo + (long long)head * a.vdim + col;
    const TQ* gt = static_cast<const TQ*>(a.gate) + t * a.ldg + (a.gate_per_head ? head : head * a.vdim + col);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      float z = v[y] * whole[0];
      if (a.gate != nullptr) z /= 1.0f + expf(-ldf(gt + (a.gate_per_head ? 0 : y)));
      stf(dst + y, z);
    }
  }
}

template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
int launch(Args a, int entries, int max_n, cudaStream_t st) {
  using K = Kind<TQ, TC, DC, VC, MT, KT>;
  const int rows = max_n * (a.H / a.G);
  int wr = 1;
  while (wr < kWarps && wr * 16 * MT < rows) wr *= 2;
  a.wr = wr;
  a.blocks = (rows + wr * 16 * MT - 1) / (wr * 16 * MT);
  a.tile_shift = 0;
  while ((KT << a.tile_shift) < a.page) ++a.tile_shift;
  constexpr size_t kRing = (size_t)kWarps * K::STAGES * K::STAGE;
  const size_t in = (size_t)wr * K::Q_BYTES + kRing, out = (size_t)kWarps * 16 * MT * (a.vdim + 4) * 4;
  const size_t smem = in > out ? in : out;
  if ((long long)a.blocks * a.G > 65535) return PG_ERR_ARG;
  auto kern = attn_rows_kernel<TQ, TC, DC, VC, MT, KT>;
  constexpr size_t kOut = (size_t)kWarps * 16 * MT * (64 * VC + 4) * 4, kIn = (size_t)kWarps * K::Q_BYTES + kRing, kMost = kIn > kOut ? kIn : kOut;
  static_assert(kMost <= 220 * 1024, "shared memory of a block");
  static bool configured[pg::kMaxDevices] = {};  // once a device, to the most that any call asks for
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  if (pg::launch_kernel(kern, dim3(a.nsplit, a.G * a.blocks, entries), dim3(32 * kWarps), smem, st, a) != cudaSuccess) return PG_ERR_CUDA;
  if (a.nsplit > 1 && pg::launch_kernel(attn_rows_merge_kernel<TQ>, dim3(a.H, a.singles ? 1 : max_n, entries), dim3(128), 0, st, a) != cudaSuccess) return PG_ERR_CUDA;
  return PG_OK;
}

template <typename TQ, typename TC, int MT, int KT>
int by_size(const Args& a, int entries, int max_n, cudaStream_t st) {
  if (a.dim <= 64 && a.vdim <= 64) return launch<TQ, TC, 1, 1, MT, KT>(a, entries, max_n, st);
  constexpr int kWide = sizeof(TC) == 1 && MT == 1 ? KT : 16;
  return launch<TQ, TC, 2, 2, MT, kWide>(a, entries, max_n, st);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" long long pg_attn_rows_scratch(int rows, int H, int vdim, int nsplit) { return nsplit > 1 ? 4LL * rows * H * nsplit * (vdim + 4) : 0; }

extern "C" int pg_attn_rows(const void* q, const PgKvPages* kv, const void* gate, long long ldg, void* out, float* partial, const int* entry_row0, const int* entry_n,
                            const int* entry_ctx, const int* page_table, int max_pages, int page, const int* pos, const void* tree, int tree_words, int entries, int max_n,
                            int singles, int nsplit, int H, int G, int dim, int vdim, float scale, float softcap, int act_f32, int gate_per_head, const PgAttnScore* score,
                            void* stream) {
  if (kv == nullptr || entries <= 0 || entries > 65535 || max_n <= 0 || nsplit <= 0 || nsplit > 64 || max_n > 65535 || H <= 0 || G <= 0 || H % G != 0 || dim <= 0 || vdim <= 0 || max_pages <= 0)
    return PG_ERR_ARG;
  if (page < 32 || (page & (page - 1)) != 0 || dim > 128 || vdim > 128 || (tree != nullptr && tree_words <= 0) || (nsplit > 1 && partial == nullptr)) return PG_ERR_ARG;
  const int unit = kv->e4m3 ? 16 : act_f32 ? 4 : 8;  // elements of a 16-byte piece
  if (dim % unit != 0 || vdim % 8 != 0 || ((long long)G * dim) % unit != 0 || !aligned(kv->k, 16) || !aligned(kv->v, 16)) return PG_ERR_ARG;
  if (kv->e4m3 && (kv->k_powers == nullptr || kv->v_powers == nullptr || !aligned(kv->k_powers, 16) || !aligned(kv->v_powers, 16))) return PG_ERR_ARG;
  if (!kv->e4m3 && kv->f32 != act_f32) return PG_ERR_ARG;
  if (nsplit > 1 && !aligned(partial, 16)) return PG_ERR_ARG;
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
  a.mode = a.sx.dist_a != nullptr || a.sx.logistic ? kGeneral : softcap > 0.f ? kCapped : kPlain;
  a.trigger = pg::weights_follow();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int most = singles ? 1 : max_n, rows = most * (H / G);
#ifndef KTE
#define KTE 32
#endif
#ifdef ONLY8
  if (kv->e4m3) {
    return rows <= 16 ? by_size<bf16, e4m3, 1, KTE>(a, entries, most, st) : by_size<bf16, e4m3, 2, KTE>(a, entries, most, st);
  }
  return -1;
#endif
  if (kv->e4m3) {
    if (act_f32) return by_size<float, e4m3, 1, 32>(a, entries, most, st);
    return rows <= 16 ? by_size<bf16, e4m3, 1, 32>(a, entries, most, st) : by_size<bf16, e4m3, 2, 32>(a, entries, most, st);
  }
  if (act_f32) return by_size<float, float, 1, 16>(a, entries, most, st);
  return rows <= 16 ? by_size<bf16, bf16, 1, 32>(a, entries, most, st) : by_size<bf16, bf16, 2, 32>(a, entries, most, st);
}
