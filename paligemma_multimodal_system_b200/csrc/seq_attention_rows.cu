// Attention of a few rows an entry over a long paged cache: decoded tokens over the 8-bit cache, and drafted trees over a cache of any type.
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(s_ij),  s_ij = cap(scale q_i . k_j) - penalty,  j over the keys that row i sees:
//   every stored key j < ctx, and drafted key m (cache row ctx + m) where bit m of the row's mask is set (no mask: m <= i); windows go by positions.
//
// A warp owns 16 MT rows (token x query head of one k/v head) and walks key tiles through a ring in shared memory that asynchronous copies fill two tiles ahead (one where a tile
// is 16 KB).  Both products run on mma.sync m16n8k16 with fp32 accumulation, and the operands' k indexes are permuted so that a lane's 16-byte pieces of the cache ARE its
// fragments:
//   * keys: lane (n, c) reads piece c of key n's row; the elements of a piece are k indexes of ITS lane in consecutive 16-deep steps, and the
//     queries are stored in that order once.  Key n of fragment f is key (KT / 4)(n / 2) + 2 f + n % 2 of the tile, so lane c's scores belong to KT / 4
//     neighbouring keys, and those are the keys whose value rows it reads for the second product, columns 8 n .. 8 n + 7 of every 64.
//   * no transposition, no conversion but codes -> halves (exact) and, for fp32, the cut into three bf16 terms.
//   * at most eight rows a k/v head (decoded tokens): the second product is transposed, O^T = V^T P^T, sixteen columns x eight rows an instruction; the weights are its second
//     operand as they stand, and no half of the instruction is empty.
// Few rows: the CTA's four warps walk tiles of their own and join in shared memory.  More: warps that hold rows of one head share a ring (a barrier a tile), since four private
// copies of every tile cost shared memory and L2 (24 trees of 31 x 4 rows over 1500 keys, bf16 pages: 154 -> 90 us).  CTAs split the keys further; up to eight join in a
// cluster, more through scratch and a second launch.
//
// Precision: bf16 operands as they are; codes as halves, exact, against queries scaled by a power of two per row into half range (fp32 queries: two
// halves, 22 bits); fp32 as three bf16 terms, six products.  Weights: two halves over codes (22 bits; one half, 11 bits, left
// one output of bf16 rows in forty beside the one that fp32 weights give, two one in 1,700: 24 trees of 31 x 4 rows 80 -> 90 us, decoded tokens 6 %); two bf16 terms over bf16 values
// (16 bits: one output in 1,000 beside it, three terms one in 1,400 at 12 % of the time); three over fp32 values.  The values' powers of two
// go into the weights, which are taken relative to the row's largest product of weight and power so far: what falls 2^-38 below it counts as zero (the head with that product keeps its
// own elements no finer than 2^-10 of its power).  Relative to the largest power met, a row that a query does not see or one of no weight took the others' values away.  24 trees of
// 31 x 4 rows over codes 76 -> 80 us, decoded tokens as before.  Weights below 2^-126 of a row's largest are zero.  Scores, maxima, sums and outputs are fp32.
// The matrix instruction cuts off what it adds to a larger sum; over many it adds up (fp32, 4700 keys: 1.0e-5 off).  For fp32 queries the small terms' products and every tile's
// outputs have sums of their own, added with a rounding (1.2e-6, as fp32 operators have); for bf16 ones it is a hundredth of the output's rounding.
//
// What bounds it: while a k/v head has few rows, the bytes of keys and values where walks are long (6 x 32000 keys of 4 x 128 over codes 45 us, 4.4 TB/s), the unequal lengths of a
// batch (64 x 1125 .. 2250 of 8 x 64 with soft cap and gate 39 us: the loop runs at the memory's rate, then short entries leave SMs empty), else a chain of trips
// (descriptors, pages, tiles, join: one x 3000 10 us).  Large trees: instructions -- conversions, exponentials and a tensor rate of 550 TFLOP/s (one m16n8k16 in 2.1 clocks an SM) --
// at ten warps an SM (24 trees of 31 x 4 rows over codes 90 us).
// The loop body is one straight line but for masks, options and new maxima: branches between the row halves cost a quarter (98 -> 84 us); a second body for masked tiles cost
// as much in instruction fetch as it saved.
#include <cuda_fp16.h>

#include "cache8.cuh"
#include "common.cuh"
#include "paligemma_b200.h"

using bf16 = __nv_bfloat16;

namespace {

static_assert(sizeof(PgAttnRows) == 192, "callers pack this struct by its size");

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
  int words, max_pages, page, max_n, tile_shift, singles, nsplit, cluster, blocks, H, G, dim, vdim, wr, mode;  // tile_shift: log2 of a page's tiles
  float scale, softcap;
  int gate_per_head, vec_q, vec_gate, vec_out;  // vec_*: four elements in one piece
  PgAttnScore sx;
  int trigger;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh to fp32 accuracy: an odd polynomial below 0.625 (least squares on tanh(x) / x, 6e-9 off) -- scores are small against their cap --, else 1 - 2 / (e^(2 |x|) + 1)
constexpr float kSmall = 0.625f;
constexpr float kTanh0 = -0.33333281f, kTanh1 = 0.13331431f, kTanh2 = -0.053739157f, kTanh3 = 0.020637862f, kTanh4 = -0.0057040425f;
__device__ __forceinline__ float tanh_f32(float x) {
  const float ax = fabsf(x), z = x * x;
  const float p = fmaf(z, fmaf(z, fmaf(z, fmaf(z, kTanh4, kTanh3), kTanh2), kTanh1), kTanh0);
  const float big = copysignf(1.0f - __fdividef(2.0f, ex2(ax * (2.f * kLog2e)) + 1.0f), x);
  return ax < kSmall ? fmaf(x * z, p, x) : big;
}
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const bf16* p) { return __bfloat162float(*p); }

// four neighbouring elements; VEC: they lie on a boundary of their own size
template <bool VEC>
__device__ __forceinline__ void ld4(float (&v)[4], const float* p) {
  if (VEC) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void ld4(float (&v)[4], const bf16* p) {
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  const uint2 u = VEC ? *reinterpret_cast<const uint2*>(p) : make_uint2(e[0] | static_cast<uint32_t>(e[1]) << 16, e[2] | static_cast<uint32_t>(e[3]) << 16);
  v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u), v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void st4(float* p, const float (&v)[4], bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = v[i];
  }
}
__device__ __forceinline__ void st4(bf16* p, const float (&v)[4], bool vec) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pg::pack_bf16(v[0], v[1]), pg::pack_bf16(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(v[i]);
  }
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
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

// the elements of a word that are infinite or NaN, as a mask
template <int ES>
__device__ __forceinline__ uint32_t no_numbers(uint32_t w) {
  if (ES == 1) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
  if (ES == 2) return __vcmpeq2(w & 0x7f807f80u, 0x7f807f80u);
  return (w & 0x7f800000u) == 0x7f800000u ? 0xffffffffu : 0u;
}

// The power (as an exponent's byte) that takes a row's largest product of weight and power to [2^14, 2^15): halves reach 38 bits below.
__device__ __forceinline__ int lift_of(float largest) { return min(14 + 2 * 127 - static_cast<int>(__float_as_uint(largest) >> 23), 254); }

template <typename TQ, typename TC, int DC, int VC, int MT, int KT>
struct Kind {
  static constexpr int ES = sizeof(TC);
  static constexpr bool C8 = ES == 1, F32 = ES == 4, HALF = C8;
  static constexpr bool APART = sizeof(TQ) == 4;
  static constexpr int QT = F32 ? 3 : (C8 && sizeof(TQ) == 4) ? 2 : 1;     // terms of a query
  static constexpr int STEPS = 4 * DC;                                     // 16-deep steps of the first product
  static constexpr int CT = F32 ? 3 : 1;                                   // terms of a cached element
  static constexpr int PT = F32 ? 3 : 2;  // terms of a weight
  static constexpr int VW = 2 * ES;                                        // words of eight value columns
  static constexpr int KROW = 64 * DC * ES, VROW = 64 * VC * ES;           // bytes of a row in shared memory
  static constexpr int STAGE = KT * (KROW + VROW) + (C8 ? 2 * KT : 0);
  static constexpr int STAGES = STAGE > 8 * 1024 + 256 ? 2 : 3;
  static constexpr int Q_BYTES = QT * MT * STEPS * 512;  // of a warp's rows
};

// what registers and shared memory leave room for
template <typename TQ, typename TC, int DC, int VC, int MT>
constexpr int ctas_per_sm() {
  return DC > 1 || VC > 1 || sizeof(TC) == 4 ? 2 : MT == 2 ? 3 : sizeof(TC) == 1 ? 4 : 2;
}

// where a row of a k/v head's block goes
struct Row {
  long long t;
  int head;
};
__device__ __forceinline__ void add(float4& acc, float f, float4 v) {
  acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
}
// a row's four columns of the gate as factors
template <typename TQ>
__device__ __forceinline__ void gates(const Args& a, const Row& r, int col, float (&gv)[4]) {
  gv[0] = gv[1] = gv[2] = gv[3] = 1.f;
  if (a.gate == nullptr) return;
  const TQ* g = static_cast<const TQ*>(a.gate) + r.t * a.ldg + (a.gate_per_head ? r.head : r.head * a.vdim + col);
  if (a.gate_per_head) gv[0] = gv[1] = gv[2] = gv[3] = ldf(g);
  else if (a.vec_gate) ld4<true>(gv, g);
  else ld4<false>(gv, g);
#pragma unroll
  for (int y = 0; y < 4; ++y)  // (a NaN stays one; bf16 rows: off by 2^-20 at most, the output's rounding is 2^-9; a division there costs 24 trees of 31 x 4 rows 3 of 80 us)
    gv[y] = sizeof(TQ) == 4 ? 1.0f / (1.0f + expf(-gv[y])) : rcp(1.0f + ex2(-kLog2e * gv[y]));
}
// what a row's sum against the maximum `ref` is multiplied by: sink, division, scale.  A row that sees nothing: zeros.
__device__ __forceinline__ float last_factor(const Args& a, int head, float ref, float l) {
  float by = a.sx.out_scale != 0.f ? a.sx.out_scale : 1.f;
  if (a.sx.logistic) return by;
  if (a.sx.sink != nullptr) {
    const float sk = a.sx.sink[head] * kLog2e, mm = fmaxf(ref, sk), f = ex2(ref - mm);
    by *= f;
    l = l * f + ex2(sk - mm);
  }
  return l == 0.f ? 0.f : by / l;
}
template <typename TQ>
__device__ __forceinline__ void put(const Args& a, const Row& r, int col, float4 acc, const float (&gv)[4]) {
  TQ* dst = static_cast<TQ*>(a.out) + r.t * (a.sx.out_ld > 0 ? a.sx.out_ld : (long long)a.H * a.vdim) + (long long)r.head * a.vdim + col;
  const float v[4] = {acc.x * gv[0], acc.y * gv[1], acc.z * gv[2], acc.w * gv[3]};
  st4(dst, v, a.vec_out);
}

// The sum of the values that are no numbers, among the keys with a mask that this CTA walks and the row sees.
template <typename TC>
__device__ __noinline__ float4 no_number_values(const Args& a, int e, int g, const Row r, int col, int split, int wk, int keys, int newest) {
  const int n = a.n[e], ctx = a.ctx[e], len = ctx + n, window = a.sx.window > 0 ? a.sx.window : 0, keep = window ? max(a.sx.keep_first, 0) : 0;
  const long long t0 = a.row0[e];
  const int i = static_cast<int>(r.t - t0), mine = a.pos != nullptr ? a.pos[r.t] : ctx + i;
  const int ntiles = (len + keys - 1) / keys, t_lo = window ? max(0, ctx - window + 1) / keys : 0, nkeep = min(min((keep + keys - 1) / keys, ntiles), t_lo);
  float out[4] = {0.f, 0.f, 0.f, 0.f};
  for (int walk = 0; walk < nkeep + ntiles - t_lo; ++walk) {
    if (walk / wk % a.nsplit != split) continue;
    const int j0 = (walk < nkeep ? walk : t_lo + walk - nkeep) * keys;
    if (j0 + keys <= ctx && (window == 0 || j0 > newest - window || j0 + keys <= keep)) continue;  // without a mask: in the sums
    for (int j = j0; j < min(j0 + keys, len); ++j) {
      const int m = j - ctx, pj = m < 0 ? j : a.pos != nullptr ? a.pos[t0 + m] : j;
      const bool seen = m < 0 || (a.tree == nullptr ? m <= i : m / 32 < a.words && (a.tree[r.t * a.words + m / 32] >> (m % 32) & 1u));
      if (!seen || (window && mine - pj >= window && pj >= keep)) continue;
      const long long row = ((long long)a.pt[(long long)e * a.max_pages + j / a.page] * a.page + j % a.page) * a.G + g;
      for (int y = 0; y < 4; ++y) {
        const long long at = row * a.vdim + col + y;
        float v;
        if (sizeof(TC) == 1) v = (a.vp[at] & 0x7f) == 0x7f ? __uint_as_float(0x7fffffffu) : 0.f;
        else if (sizeof(TC) == 2) v = __bfloat162float(reinterpret_cast<const bf16*>(a.vp)[at]);
        else v = reinterpret_cast<const float*>(a.vp)[at];
        if (!(fabsf(v) < INFINITY)) out[y] += v;
      }
    }
  }
  return make_float4(out[0], out[1], out[2], out[3]);
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

// DC, VC: 64-element pieces of a key / value row; MT: 16-row tiles of a warp; KT: keys of a tile; R8: a k/v head has at most eight rows, the tile's upper half is empty
template <typename TQ, typename TC, int DC, int VC, int MT, int KT, bool R8>
__global__ void __launch_bounds__(32 * kWarps, (ctas_per_sm<TQ, TC, DC, VC, MT>())) attn_rows_kernel(const __grid_constant__ Args a) {
  using K = Kind<TQ, TC, DC, VC, MT, KT>;
  constexpr int NB = KT / 8, KPL = KT / 4;  // key fragments of a tile; keys of a lane
  extern __shared__ __align__(128) unsigned char raw[];
  __shared__ float unscale[kWarps * 16 * MT];  // what a row's scores are multiplied by
  __shared__ float2 stat[kWarps][16 * MT];
  __shared__ float power[kWarps][16 * MT];  // what a warp's sums of a row are multiplied by (8-bit cache)
  __shared__ float2 joined[kWarps * 16 * MT];
  __shared__ int2 where_to[kWarps * 16 * MT];  // a row's token of the entry and its head; past the last row: the last one's
  __shared__ float share[8][kWarps * 16 * MT];
  __shared__ int any_bad;
  __shared__ int last_pos;  // windows: the farthest position of the CTA's rows
  if (threadIdx.x == 0) any_bad = 0, last_pos = 0;
  // (the step's descriptors, too, may come from the kernel in front)
  if (a.nsplit > 1 && !a.cluster) pg::griddep_begin<true>();  // (fp32 partials, read behind a wait)
  else pg::griddep_begin_if(a.trigger);
  const int split = blockIdx.x, g = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, e = blockIdx.z;
  const int n = a.n[e], ctx = a.ctx[e], gsz = a.H / a.G, len = ctx + n;
  const long long t0 = a.row0[e];
  const int wr = R8 ? 1 : a.wr, wk = kWarps / wr, rows_cta = wr * 16 * MT, r0 = block * rows_cta, R = min(n, a.max_n) * gsz;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nn = lane >> 2, c = lane & 3;
  const int rg = warp % wr, kgrp = warp / wr;
  const bool mine = !(a.singles && n != 1) && r0 < R;
  const int live = mine ? R - r0 - 16 * MT * rg : 0;  // rows of this warp (none: nothing to walk)

  // ---- the key walk
  const int window = a.sx.window > 0 ? a.sx.window : 0, keep = window ? max(a.sx.keep_first, 0) : 0;
  const int ntiles = (len + KT - 1) / KT;
  const int t_lo = window ? max(0, ctx - window + 1) / KT : 0;
  const int nkeep = min(min((keep + KT - 1) / KT, ntiles), t_lo);
  const int nwalk = mine ? nkeep + ntiles - t_lo : 0;
  const int* pt = a.pt + (long long)e * a.max_pages;
  const int stride = a.nsplit * wk, tpp = 1 << a.tile_shift, walk0 = split * wk + kgrp;
  auto tile_of = [&](int walk) { return walk < nkeep ? walk : t_lo + (walk - nkeep); };
  // page numbers of 32 tiles of the walk, a lane each
  auto pages_from = [&](int walk) {
    const int w = walk + lane * stride;
    return w < nwalk ? pt[tile_of(w) >> a.tile_shift] : 0;
  };
  int pids = pages_from(walk0);
  if (!mine) return;

  // ---- copies: a ring of tiles for the warps that walk together, 16 bytes a thread and request
  unsigned char* ring = raw + wr * K::Q_BYTES + kgrp * (K::STAGES * K::STAGE);
  const int tg = rg * 32 + lane, group = 32 * wr;
  auto meet = [&] {
    if (wr == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + kgrp), "r"(group) : "memory");
  };
  const long long kpitch = (long long)a.G * a.dim * K::ES, vpitch = (long long)a.G * a.vdim * K::ES;
  const int kbytes = a.dim * K::ES, vbytes = a.vdim * K::ES;
  auto request = [&](int k, int it, int pid) {  // tile `it` into stage k % STAGES
    const uint32_t dst = pg::smem_u32(ring + (k % K::STAGES) * K::STAGE);
    const long long first = (long long)pid * a.page + (it & (tpp - 1)) * KT;
    constexpr int KP = K::KROW / 16, VP = K::VROW / 16;
    {
      const int piece = tg % KP;  // (a group is a multiple of a row's pieces)
      const uint8_t* p = a.kp + first * kpitch + (long long)g * kbytes + 16 * piece;
      const bool in = 16 * piece < kbytes;
#pragma unroll (R8 ? KT * KP / 32 : 4)
      for (int r = tg / KP; r < KT; r += group / KP) pg::cp_async16(dst + key_place<K::KROW>(r, piece), p + r * kpitch, in);
    }
    {
      const int piece = tg % VP;
      const uint8_t* p = a.vp + first * vpitch + (long long)g * vbytes + 16 * piece;
      const bool in = 16 * piece < vbytes;
      const int left = len - it * KT;  // rows behind the last one hold anything: zeros
#pragma unroll (R8 ? KT * VP / 32 : 4)
      for (int r = tg / VP; r < KT; r += group / VP) pg::cp_async16(dst + KT * K::KROW + value_place<K::VROW, KPL, K::ES>(r, piece), p + r * vpitch, in && r < left);
    }
    if (K::C8 && tg < KT / 8) {  // the powers: keys' in the first half of these threads, values' in the second
      const bool is_v = tg >= KT / 16;
      const uint8_t* p = (is_v ? a.ve : a.ke) + ((long long)pid * a.G + g) * a.page + (it & (tpp - 1)) * KT + 16 * (tg % (KT / 16));
      pg::cp_async16(dst + KT * (K::KROW + K::VROW) + 16 * tg, p, true);
    }
  };
#pragma unroll 1
  for (int k = 0; k < K::STAGES - 1; ++k) {
    const int w = walk0 + k * stride, pid = __shfl_sync(0xffffffffu, pids, k);
    if (w < nwalk) request(k, tile_of(w), pid);
    pg::cp_async_commit();
  }

  // ---- queries: fragments in the order of the cache's pieces; four elements a lane, a warp takes every fourth row, one trip to memory
  for (int r = tid; r < rows_cta; r += 32 * kWarps) {
    const int rr = min(r0 + r, R - 1), i = rr / gsz;
    where_to[r] = make_int2(i, g * gsz + rr - i * gsz);
  }
  __syncthreads();
  if (window)
    for (int r = tid; r < min(rows_cta, R - r0); r += 32 * kWarps) atomicMax(&last_pos, a.pos[t0 + where_to[r].x]);
  uint4* qs = reinterpret_cast<uint4*>(raw);  // [term][row tile][step][lane]
  const int tiles_m = wr * MT;
  constexpr int QL = DC == 1 ? 16 : 32;       // lanes of a row
  constexpr int RW = 32 / QL;                 // rows a warp and pass
  constexpr int PASS = R8 ? 1 : 4 * MT;            // passes whose loads are under way together
  const int rows_staged = R8 ? 8 : rows_cta;  // (R8: what stands in the upper half's fragments reaches no output)
  const int w = lane % QL, st = w / 4, cc = w % 4;
  const int d0 = K::C8 ? 64 * (st / 4) + 16 * cc + 4 * (st % 4) : K::F32 ? 16 * st + 4 * cc : 32 * (st / 2) + 8 * cc + 4 * (st % 2);
  const TQ* q0 = static_cast<const TQ*>(a.q) + t0 * a.H * a.dim + (d0 < a.dim ? d0 : 0);
#pragma unroll 1
  for (int rb = warp * RW + lane / QL; rb < rows_staged; rb += kWarps * RW * PASS) {  // (whole warps: rows are multiples of eight)
    float v[PASS][4], by[PASS];
    int2 to[PASS];
#pragma unroll
    for (int u = 0; u < PASS; ++u) to[u] = where_to[min(rb + u * kWarps * RW, rows_cta - 1)];
    if (a.vec_q) {
#pragma unroll
      for (int u = 0; u < PASS; ++u) ld4<true>(v[u], q0 + ((long long)to[u].x * a.H + to[u].y) * a.dim);
    } else {
#pragma unroll
      for (int u = 0; u < PASS; ++u) ld4<false>(v[u], q0 + ((long long)to[u].x * a.H + to[u].y) * a.dim);
    }
#pragma unroll
    for (int u = 0; u < PASS; ++u) by[u] = a.sx.head_scale != nullptr ? a.sx.head_scale[to[u].y] : 1.f;
#pragma unroll
    for (int u = 0; u < PASS; ++u) {
      const int r = rb + u * kWarps * RW;
      const bool in = r0 + r < R && d0 < a.dim;
      float s = a.scale * by[u];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[u][k] = in ? v[u][k] : 0.f;
      if (K::C8) {
        float top = fmaxf(fmaxf(fabsf(v[u][0]), fabsf(v[u][1])), fmaxf(fabsf(v[u][2]), fabsf(v[u][3])));
#pragma unroll
        for (int o = QL / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // largest element to [2^14, 2^15): a half keeps eleven bits down to 2^-14, and 2^-24 below
        const int x = min(max(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100);
        const float up = __uint_as_float(static_cast<uint32_t>(x + 127) << 23);
        s *= __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[u][k] *= up;
      }
      if (r >= rows_staged) break;
      if (w == 0) unscale[r] = a.mode == kGeneral ? s : a.mode == kCapped ? s / a.softcap : s * kLog2e;
      // row r of its tile: lanes 4 (r % 8) + c, first or second half of the fragment's registers
      {
        uint32_t p[K::QT], s2[K::QT];
        terms<K::HALF>(v[u][0], v[u][1], p);
        terms<K::HALF>(v[u][2], v[u][3], s2);
#pragma unroll
        for (int t = 0; t < K::QT; ++t) {
          uint32_t* f = reinterpret_cast<uint32_t*>(qs + ((t * tiles_m + r / 16) * K::STEPS + st) * 32 + 4 * (r % 8) + cc) + (r % 16 < 8 ? 0 : 1);
          f[0] = p[t];
          f[2] = s2[t];
        }
      }
    }
  }
  __syncthreads();

  // ---- my rows
  int node[2 * MT];  // token of the entry
  float uns[2 * MT];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    const int r = 16 * (rg * MT + x / 2) + 8 * (x % 2) + nn;
    node[x] = where_to[r].x;
    uns[x] = unscale[r];
  }

  constexpr int OB = R8 ? 4 * VC : 8 * VC;  // R8: transposed, 16 columns x eight rows an instruction
  float M[2 * MT], L[2 * MT], o[MT][OB][4];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) M[x] = a.sx.logistic ? 0.f : -INFINITY, L[x] = 0.f;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[m][b][k] = 0.f;
  float top[2 * MT];  // 8-bit cache: a row's largest weight times power so far, against its maximum
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) top[x] = 0.f;

  bool bad = false;  // a value that is no number in a tile with a mask
#pragma unroll 1
  for (int k = 0, walk = walk0; walk < nwalk; ++k, walk += stride) {
    pg::cp_async_wait<K::STAGES - 2>();
    meet();  // tile k is here for all, and all are done with the tile before
    const int ahead = k + K::STAGES - 1;
    if ((ahead & 31) == 0) pids = pages_from(walk0 + ahead * stride);
    const int wa = walk0 + ahead * stride, pid = __shfl_sync(0xffffffffu, pids, ahead & 31);
    if (wa < nwalk) request(ahead, tile_of(wa), pid);
    pg::cp_async_commit();
    const int it = tile_of(walk), j0 = it * KT;
    const unsigned char* stage = ring + (k % K::STAGES) * K::STAGE;
    const bool plain = j0 + KT <= ctx && (window == 0 || j0 > last_pos - window || j0 + KT <= keep);  // every row sees every key of the tile
    // ---- who sees what
    uint32_t vis[2 * MT];
    if (!plain) {
      // 32 drafted tokens a word, in front of the first one stored keys; the tile's keys start inside word w
      const int rel = j0 - ctx, w = rel >> 5;
      uint32_t lo[2 * MT], hi[2 * MT];
#pragma unroll
      for (int x = 0; x < 2 * MT; ++x) {
        if (a.tree != nullptr) {
          const uint32_t* mask = a.tree + (t0 + node[x]) * a.words;
          lo[x] = mask[min(max(w, 0), a.words - 1)];
          hi[x] = mask[min(max(w + 1, 0), a.words - 1)];
        } else {
          const int upto = node[x] + 1;  // a chain: rows up to itself
          lo[x] = upto - 32 * w >= 32 ? 0xffffffffu : upto <= 32 * w ? 0u : (1u << (upto - 32 * w)) - 1u;
          hi[x] = upto - 32 * w >= 64 ? 0xffffffffu : upto <= 32 * w + 32 ? 0u : (1u << (upto - 32 * w - 32)) - 1u;
        }
      }
      auto have = [&](int w) { return w < 0 || n - 32 * w >= 32 ? 0xffffffffu : n <= 32 * w || (a.tree != nullptr && w >= a.words) ? 0u : (1u << (n - 32 * w)) - 1u; };
      const uint32_t all_lo = a.tree != nullptr && w >= a.words ? 0u : have(w), all_hi = a.tree != nullptr && w + 1 >= a.words ? 0u : have(w + 1);
#pragma unroll
      for (int x = 0; x < 2 * MT; ++x) {
        uint32_t v = __funnelshift_r(w < 0 ? 0xffffffffu : lo[x] & all_lo, w + 1 < 0 ? 0xffffffffu : hi[x] & all_hi, rel & 31);
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
      // a value that is not a number reaches only the rows that see its key (a weight of zero times it is none): taken out here, added to their outputs below
      unsigned char* values = ring + (k % K::STAGES) * K::STAGE + KT * K::KROW;
#pragma unroll 1
      for (int at = 16 * tg; at < KT * K::VROW; at += 16 * group) {
        uint4 u = *reinterpret_cast<const uint4*>(values + at);
        const uint4 no = make_uint4(no_numbers<K::ES>(u.x), no_numbers<K::ES>(u.y), no_numbers<K::ES>(u.z), no_numbers<K::ES>(u.w));
        if (no.x | no.y | no.z | no.w) {
          bad = true;
          *reinterpret_cast<uint4*>(values + at) = make_uint4(u.x & ~no.x, u.y & ~no.y, u.z & ~no.z, u.w & ~no.w);
        }
      }
      if (K::C8 && tg < KT && j0 + tg >= len) values[KT * K::VROW + KT + tg] = 0;  // (powers of rows behind the last one)
      meet();
    }
    if (live <= 0) continue;  // no rows for this warp
    // ---- S = Q K^T
    float s[MT][NB][4], small[MT][NB][4];  // small: products of all but the first terms (fp32 queries)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int f = 0; f < NB; ++f)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[m][f][k] = small[m][f][k] = 0.f;
    constexpr int SPL = K::C8 ? 4 : K::F32 ? 1 : 2;  // steps of a piece
#pragma unroll
    for (int x = 0; x < K::STEPS / SPL; ++x) {
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
          for (int t = 0; t < K::QT; ++t) qa[m][t] = qs[((t * tiles_m + rg * MT + m) * K::STEPS + st) * 32 + lane];
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
                if (t + t2 < 3) mma<K::HALF>(K::APART && t + t2 > 0 ? small[m][f] : s[m][f], qa[m][t], b0[t2], b1[t2]);
        }
      }
    }
    if (K::APART) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int f = 0; f < NB; ++f)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[m][f][k] += small[m][f][k];
    }
    // ---- weights: one straight line but for options, masks and new maxima
    uint64_t kf[NB], vf[NB];  // pairs of powers: keys 2 f, 2 f + 1 of this lane
    if (K::C8) {
#pragma unroll
      for (int x = 0; x < KPL / 4; ++x) {
        const uint32_t kp = *reinterpret_cast<const uint32_t*>(stage + KT * (K::KROW + K::VROW) + KPL * c + 4 * x);
        const uint32_t vp = *reinterpret_cast<const uint32_t*>(stage + KT * (K::KROW + K::VROW) + KT + KPL * c + 4 * x);
#pragma unroll
        for (int y = 0; y < 2; ++y) {  // (a key's byte 0: what is below 2^-118 counts as zero)
          const int sh = 16 * y;
          kf[2 * x + y] = pg::pair_of((kp >> sh & 0xffu) << 23, (kp >> (sh + 8) & 0xffu) << 23);
          vf[2 * x + y] = pg::pair_of(cache8::value_of_power(vp >> sh & 0xffu), cache8::value_of_power(vp >> (sh + 8) & 0xffu));
        }
      }
    }
    constexpr int HS = R8 ? 1 : 2;
    uint64_t t[MT][HS][NB];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < HS; ++h) {
        const uint64_t u = pg::pair_of(uns[2 * m + h], uns[2 * m + h]);
#pragma unroll
        for (int f = 0; f < NB; ++f) t[m][h][f] = mul_pair(pg::pair_of(s[m][f][2 * h], s[m][f][2 * h + 1]), K::C8 ? mul_pair(u, kf[f]) : u);
      }
    if (a.mode == kCapped) {  // cap tanh(v / cap) in log2 units; v comes as v / cap
      const float cap = a.softcap * kLog2e;
      float far = 0.f;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < HS; ++h)
#pragma unroll
          for (int f = 0; f < NB; ++f) far = pg::max3(far, fabsf(pg::lo_f32(t[m][h][f])), fabsf(pg::hi_f32(t[m][h][f])));
      // (fp32 rows of several tokens over codes have no registers for both: 24 trees of 31 x 4 without a cap 109 -> 114 us, with one 131 -> 125)
      if ((K::C8 && K::APART && !R8) || __any_sync(0xffffffffu, far >= kSmall)) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < HS; ++h)
#pragma unroll
            for (int f = 0; f < NB; ++f) t[m][h][f] = pg::pair_of(cap * tanh_f32(pg::lo_f32(t[m][h][f])), cap * tanh_f32(pg::hi_f32(t[m][h][f])));
      } else {  // scores are small against their cap: two at a time
        auto both = [](float x) { return pg::pair_of(x, x); };
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < HS; ++h)
#pragma unroll
            for (int f = 0; f < NB; ++f) {
              const uint64_t x = t[m][h][f], z = mul_pair(x, x);
              const uint64_t p = pg::fma_pair(z, pg::fma_pair(z, pg::fma_pair(z, pg::fma_pair(z, both(kTanh4), both(kTanh3)), both(kTanh2)), both(kTanh1)), both(kTanh0));
              t[m][h][f] = mul_pair(pg::fma_pair(mul_pair(x, z), p, x), both(cap));
            }
      }
    } else if (a.mode == kGeneral) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < HS; ++h) {
          const int head = where_to[16 * (rg * MT + m) + 8 * h + nn].y, mine = a.pos != nullptr ? a.pos[t0 + node[2 * m + h]] : 0;
          auto bend = [&](float v, int j) {
            if (a.softcap > 0.f) v = a.softcap * tanh_f32(v / a.softcap);
            if (a.sx.dist_a != nullptr) v -= a.sx.dist_a[head] * log1pf(a.sx.dist_b[head] * (float)max(mine - (j < ctx || j >= len ? j : a.pos[t0 + (j - ctx)]), 0));
            // a logistic weight as a power of two against a maximum of 0
            if (a.sx.logistic) return -log2f(1.0f + expf(-(v + (a.sx.head_bias != nullptr ? a.sx.head_bias[head] : 0.f))));
            return v * kLog2e;
          };
          uint64_t* row = t[m][h];
#pragma unroll 1
          for (int f = 0; f < NB; ++f) {
            uint64_t two = 0;
#pragma unroll
            for (int y = 0; y < NB; ++y) two = y == f ? row[y] : two;
            const int j = j0 + KPL * c + 2 * f;
            two = pg::pair_of(bend(pg::lo_f32(two), j), bend(pg::hi_f32(two), j + 1));
#pragma unroll
            for (int y = 0; y < NB; ++y) row[y] = y == f ? two : row[y];
          }
        }
    }
    if (!plain) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < HS; ++h) {
          const uint32_t v = vis[2 * m + h] >> (KPL * c);
#pragma unroll
          for (int f = 0; f < NB; ++f)
            t[m][h][f] = pg::pair_of(v >> (2 * f) & 1u ? pg::lo_f32(t[m][h][f]) : -INFINITY, v >> (2 * f + 1) & 1u ? pg::hi_f32(t[m][h][f]) : -INFINITY);
        }
    }
    float corr[2 * MT];
    bool moved = false;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < HS; ++h) {
        const int x = 2 * m + h;
        float mx = fmaxf(pg::lo_f32(t[m][h][0]), pg::hi_f32(t[m][h][0]));
#pragma unroll
        for (int f = 1; f < NB; ++f) mx = pg::max3(mx, pg::lo_f32(t[m][h][f]), pg::hi_f32(t[m][h][f]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float now = a.sx.logistic ? 0.f : fmaxf(M[x], mx), ref = now == -INFINITY ? 0.f : now;  // nothing seen so far: weights of zero
        const float shrink = ex2(M[x] - ref);
        corr[x] = shrink;
        M[x] = now;
        const uint64_t minus = pg::pair_of(-ref, -ref);
        uint64_t sum = 0;
#pragma unroll
        for (int f = 0; f < NB; ++f) {
          const uint64_t d = pg::add_pair(t[m][h][f], minus);
          const uint64_t p = pg::pair_of(ex2(pg::lo_f32(d)), ex2(pg::hi_f32(d)));
          sum = f == 0 ? p : pg::add_pair(sum, p);
          t[m][h][f] = K::C8 ? mul_pair(p, vf[f]) : p;
        }
        L[x] = fmaf(L[x], shrink, pg::lo_f32(sum) + pg::hi_f32(sum));
        if (K::C8) {
          float most = fmaxf(pg::lo_f32(t[m][h][0]), pg::hi_f32(t[m][h][0]));
#pragma unroll
          for (int f = 1; f < NB; ++f) most = pg::max3(most, pg::lo_f32(t[m][h][f]), pg::hi_f32(t[m][h][f]));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          const int was = lift_of(top[x]);
          top[x] = fmaxf(top[x] * shrink, most);
          const int lift = lift_of(top[x]);
          corr[x] *= __uint_as_float(static_cast<uint32_t>(min(max(127 + lift - was, 0), 254)) << 23);
          const float by = __uint_as_float(static_cast<uint32_t>(lift) << 23);
#pragma unroll
          for (int f = 0; f < NB; ++f) t[m][h][f] = mul_pair(t[m][h][f], pg::pair_of(by, by));
        }
        moved |= corr[x] != 1.f;
      }
    if (__any_sync(0xffffffffu, moved)) {
      if (R8) {  // my accumulators are rows 2 c and 2 c + 1
        const float even = __shfl_sync(0xffffffffu, corr[0], 8 * c), odd = __shfl_sync(0xffffffffu, corr[0], 8 * c + 4);
#pragma unroll
        for (int b = 0; b < OB; ++b) o[0][b][0] *= even, o[0][b][1] *= odd, o[0][b][2] *= even, o[0][b][3] *= odd;
      } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int b = 0; b < OB; ++b) {
            o[m][b][0] *= corr[2 * m], o[m][b][1] *= corr[2 * m];
            o[m][b][2] *= corr[2 * m + HS - 1], o[m][b][3] *= corr[2 * m + HS - 1];
          }
      }
    }
    uint4 pa[MT][NB / 2][K::PT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q = 0; q < NB / 2; ++q) {
        uint32_t p0[K::PT], p1[K::PT], p2[K::PT], p3[K::PT];
        terms<K::HALF>(pg::lo_f32(t[m][0][2 * q]), pg::hi_f32(t[m][0][2 * q]), p0);
        terms<K::HALF>(pg::lo_f32(t[m][0][2 * q + 1]), pg::hi_f32(t[m][0][2 * q + 1]), p2);
        if (R8) {
#pragma unroll
          for (int i = 0; i < K::PT; ++i) p1[i] = p3[i] = 0u;
        } else {
          terms<K::HALF>(pg::lo_f32(t[m][HS - 1][2 * q]), pg::hi_f32(t[m][HS - 1][2 * q]), p1);
          terms<K::HALF>(pg::lo_f32(t[m][HS - 1][2 * q + 1]), pg::hi_f32(t[m][HS - 1][2 * q + 1]), p3);
        }
#pragma unroll
        for (int i = 0; i < K::PT; ++i) pa[m][q][i] = make_uint4(p0[i], p1[i], p2[i], p3[i]);
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
#pragma unroll
      for (int b = 0; b < VC; ++b) {
        uint32_t w0[2][K::CT], w1[2][K::CT];  // two neighbouring columns: keys 4 q, 4 q + 1 and 4 q + 2, 4 q + 3
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // column 8 n + y of the piece
          uint32_t(&b0)[K::CT] = w0[y % 2];
          uint32_t(&b1)[K::CT] = w1[y % 2];
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
          if (R8 && y % 2 == 0) continue;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float(&acc)[4] = o[m][R8 ? (4 * b + y / 2) % OB : (8 * b + y) % OB];
            float own[4] = {0.f, 0.f, 0.f, 0.f};  // fp32 queries: a tile's products apart, added with a rounding
            float(&sum)[4] = K::APART ? own : acc;
#pragma unroll
            for (int t = K::PT - 1; t >= 0; --t)
#pragma unroll
              for (int t2 = K::CT - 1; t2 >= 0; --t2)
                if (t + t2 < 3) {
                  if (R8) mma<K::HALF>(sum, make_uint4(w0[0][t2], w0[1][t2], w1[0][t2], w1[1][t2]), pa[0][q][t].x, pa[0][q][t].z);
                  else mma<K::HALF>(sum, pa[m][q][t], b0[t2], b1[t2]);
                }
            if (K::APART) {
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[x] += own[x];
            }
          }
        }
      }
    }
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
    if (K::C8 && c == 0) power[warp][r] = cache8::value_of_power(254 - lift_of(top[x]));
    if (R8) continue;
    float* dst = os + (warp * 16 * MT + r) * ldo_s;
#pragma unroll
    for (int b = 0; b < VC; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = 64 * b + 16 * c + 8 * k;
        if (col < a.vdim) {
#pragma unroll
          for (int y = 0; y < 8; y += 4)
            *reinterpret_cast<float4*>(dst + col + y) = make_float4(o[x / 2][(8 * b + y) % OB][2 * (x % 2) + k], o[x / 2][(8 * b + y + 1) % OB][2 * (x % 2) + k],
                                                                    o[x / 2][(8 * b + y + 2) % OB][2 * (x % 2) + k], o[x / 2][(8 * b + y + 3) % OB][2 * (x % 2) + k]);
        }
      }
  }
  if (R8) {
#pragma unroll
    for (int i = 0; i < 2; ++i)  // rows 2 c and 2 c + 1, columns 8 n .. 8 n + 7 of every 64
#pragma unroll
      for (int b = 0; b < VC; ++b)
        if (64 * b + 8 * nn < a.vdim) {
          float* dst = os + (warp * 16 * MT + 2 * c + i) * ldo_s + 64 * b + 8 * nn;
#pragma unroll
          for (int y = 0; y < 2; ++y)
            *reinterpret_cast<float4*>(dst + 4 * y) = make_float4(o[0][4 * b + 2 * y][i], o[0][4 * b + 2 * y][2 + i], o[0][4 * b + 2 * y + 1][i], o[0][4 * b + 2 * y + 1][2 + i]);
        }
  }
  if (bad) any_bad = 1;
  __syncthreads();
  const int rows_here = min(rows_cta, R - r0);
  for (int r = tid; r < rows_here; r += 32 * kWarps) {  // a row's factors
    const int tile = r / (16 * MT), in = r % (16 * MT);
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < wk; ++w) m = fmaxf(m, stat[w * wr + tile][in].x);
    const float ref = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < wk; ++w) l += ex2(stat[w * wr + tile][in].x - ref) * stat[w * wr + tile][in].y;  // (scores that are no numbers stay in the sum)
    const float by = a.nsplit == 1 ? last_factor(a, where_to[r].y, ref, l) : 1.f;
    for (int w = 0; w < wk; ++w) {
      float2& st = stat[w * wr + tile][in];
      st.x = ex2(st.x - ref) * by * (K::C8 ? power[w * wr + tile][in] : 1.f);
    }
    joined[r] = make_float2(m, l);
  }
  __syncthreads();
  const int quads = a.vdim / 4, per_pass = 32 * kWarps / quads, row_of = tid / quads, col = 4 * (tid - row_of * quads);  // four columns a thread
  auto row_at = [&](int r) { return Row{t0 + where_to[r].x, where_to[r].y}; };
  if (any_bad) {  // values that are no numbers, into the first warp's sums
    for (int r = row_of < per_pass ? row_of : rows_here; r < rows_here; r += per_pass) {
      const int tile = r / (16 * MT), in = r % (16 * MT);
      const float4 v = no_number_values<TC>(a, e, g, row_at(r), col, split, wk, KT, last_pos);
      add(*reinterpret_cast<float4*>(os + (tile * 16 * MT + in) * ldo_s + col), 1.f, v);
    }
    __syncthreads();
    for (int r = tid; r < rows_here; r += 32 * kWarps) {
      float2& st = stat[r / (16 * MT)][r % (16 * MT)];
      if (st.x == 0.f) st.x = __uint_as_float(1u);  // (a factor of zero would leave them out)
    }
    __syncthreads();
  }
#pragma unroll 4
  for (int r = row_of < per_pass ? row_of : rows_here; r < rows_here; r += per_pass) {
    const int tile = r / (16 * MT), in = r % (16 * MT);
    const Row where = row_at(r);
    float gv[4];
    if (a.nsplit == 1) gates<TQ>(a, where, col, gv);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < wk; ++w) {
      const int ww = w * wr + tile;
      const float f = stat[ww][in].x;
      if (f != 0.f) add(acc, f, *reinterpret_cast<const float4*>(os + (ww * 16 * MT + in) * ldo_s + col));
    }
    if (a.nsplit == 1) {
      put<TQ>(a, where, col, acc, gv);
    } else if (a.cluster) {  // over the first warp's, whose columns only this thread reads
      *reinterpret_cast<float4*>(os + (tile * 16 * MT + in) * ldo_s + col) = acc;
    } else {
      float* pp = a.partial + (((a.singles ? (long long)e : where.t) * a.H + where.head) * a.nsplit + split) * (a.vdim + 4);
      *reinterpret_cast<float4*>(pp + 4 + col) = acc;
      if (col == 0) *reinterpret_cast<float2*>(pp) = joined[r];
    }
  }
  if (!a.cluster) return;
  // ---- the CTAs of a cluster share out the rows' columns and read one another's results
  pg::cluster_sync_all();
  auto of_cta = [&](const void* p, int cta) {
    uint32_t x;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(x) : "r"(pg::smem_u32(p)), "r"(cta));
    return x;
  };
  for (int r = tid; r < rows_here; r += 32 * kWarps) {
    float2 st[8];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      st[p] = make_float2(-INFINITY, 0.f);
      if (p < a.nsplit) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(st[p].x), "=f"(st[p].y) : "r"(of_cta(&joined[r], p)) : "memory");
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) m = fmaxf(m, st[p].x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int p = 0; p < 8; ++p) l += ex2(st[p].x - ref) * st[p].y;
    const float by = last_factor(a, where_to[r].y, ref, l);
#pragma unroll
    for (int p = 0; p < 8; ++p) share[p][r] = ex2(st[p].x - ref) * by;
  }
  __syncthreads();
  for (int r = (row_of < per_pass ? row_of : rows_here) + per_pass * split; r < rows_here; r += per_pass * a.nsplit) {
    const int tile = r / (16 * MT), in = r % (16 * MT);
    const Row where = row_at(r);
    float gv[4];
    gates<TQ>(a, where, col, gv);
    const float* mine = os + (tile * 16 * MT + in) * ldo_s + col;
    float4 v[8], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (p >= a.nsplit) break;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[p].x), "=f"(v[p].y), "=f"(v[p].z), "=f"(v[p].w) : "r"(of_cta(mine, p)) : "memory");
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (p >= a.nsplit) break;
      const float f = share[p][r];
      if (f != 0.f) add(acc, f, v[p]);
    }
    put<TQ>(a, where, col, acc, gv);
  }
  pg::cluster_sync_all();  // nobody leaves while its memory is read
}

// A CTA a row: its warps take every fourth split, four columns a lane (vdim <= 128), the first splits' values requested before their factors are known.
template <typename TQ>
__global__ void __launch_bounds__(128) attn_rows_merge_kernel(const __grid_constant__ Args a) {
  constexpr int AHEAD = 8;
  __shared__ float4 sums[4][32];
  __shared__ float fs[64];
  __shared__ float whole[2];
  const int e = blockIdx.z, head = blockIdx.x, i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pg::griddep_begin_if(a.trigger);
  const int n = a.n[e];
  const long long t = a.row0[e] + i;
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
    fs[lane] = fx;
    fs[lane + 32] = fy;
    if (lane == 0) whole[0] = ref, whole[1] = l;
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < a.vdim) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int s = warp + 4 * k;
      if (s >= a.nsplit) break;
      const float f = fs[s];
      if (f != 0.f) add(acc, f, k < AHEAD ? ahead[k % AHEAD] : *reinterpret_cast<const float4*>(pp + s * ld + 4 + col));  // (a split without keys left zeros)
    }
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && col < a.vdim) {
#pragma unroll
    for (int w = 1; w < 4; ++w) add(acc, 1.f, sums[w][lane]);
    const Row where{t, head};
    float gv[4];
    gates<TQ>(a, where, col, gv);
    const float by = last_factor(a, head, whole[0], whole[1]);
    put<TQ>(a, where, col, make_float4(acc.x * by, acc.y * by, acc.z * by, acc.w * by), gv);
  }
}

// What the host decides: rows a warp, CTAs a walk.
struct Plan {
  int wr, blocks, nsplit, cluster;
};
Plan plan_of(const PgAttnRows& p, int rows, int row_tile, int keys, int per_sm) {
  Plan x;
  x.wr = 1;
  while (x.wr < kWarps && x.wr * row_tile < rows) x.wr *= 2;
  x.blocks = (rows + x.wr * row_tile - 1) / (x.wr * row_tile);
  long long reach = p.longest;
  if (p.score != nullptr && p.score->window > 0) {
    const long long w = (long long)p.score->window + (p.score->keep_first > 0 ? p.score->keep_first : 0) + p.max_n + 2 * keys;
    reach = reach < w ? reach : w;
  }
  const long long tiles = (reach + keys - 1) / keys, ctas = (long long)p.busy * p.G * x.blocks;
  // CTAs that share a walk: what the SMs hold at once, with two tiles for a warp at least, and four where there are two CTAs an SM already (24 x 1500 keys of 8 heads in three / two
  // parts 20.6 / 16.8 us; one x 3000 in eight parts of three tiles 10.3, in four 12.3)
  const long long sms = pg::num_sms(), most = tiles * x.wr / (2 * kWarps);
  long long n = per_sm * sms / (ctas > 0 ? ctas : 1);
  const long long filled = 2 * sms / (ctas > 0 ? ctas : 1), calm = most / 2 > filled ? most / 2 : filled;
  n = n < most ? n : most;
  n = n < calm ? n : calm;
  n = n > 64 ? 64 : n < 1 ? 1 : n;
  // up to eight join through distributed shared memory in one launch; more, where that leaves warps with a long walk, through global memory and a second one
  x.cluster = n <= 8 || most <= 12;
  n = x.cluster && n > 8 ? 8 : n;
  if (n == 1) x.cluster = 0;
  x.nsplit = (int)n;
  return x;
}

// need: the scratch that the call asks for, nothing is launched; NULL: launches
template <typename TQ, typename TC, int DC, int VC, int MT, int KT, bool R8>
int launch(const PgAttnRows& p, Args a, long long* need, long long scratch_bytes, cudaStream_t st) {
  using K = Kind<TQ, TC, DC, VC, MT, KT>;
  const int max_n = p.singles ? 1 : p.max_n;
  const Plan plan = plan_of(p, max_n * (a.H / a.G), 16 * MT, KT, ctas_per_sm<TQ, TC, DC, VC, MT>());
  const long long bytes = plan.nsplit > 1 && !plan.cluster ? 4LL * (p.singles ? p.entries : p.rows) * a.H * plan.nsplit * (a.vdim + 4) : 0;
  if (need != nullptr) {
    *need = bytes;
    return PG_OK;
  }
  if (bytes > 0 && (a.partial == nullptr || scratch_bytes < bytes || (reinterpret_cast<uintptr_t>(a.partial) & 15) != 0)) return PG_ERR_ARG;
  a.wr = plan.wr, a.blocks = plan.blocks, a.nsplit = plan.nsplit, a.cluster = plan.cluster;
  a.tile_shift = 0;
  while ((KT << a.tile_shift) < a.page) ++a.tile_shift;
  constexpr size_t kRing = (size_t)K::STAGES * K::STAGE;  // of the warps that walk together
  const size_t in = (size_t)a.wr * K::Q_BYTES + kWarps / a.wr * kRing, out = (size_t)kWarps * 16 * MT * (a.vdim + 4) * 4;
  const size_t smem = in > out ? in : out;
  if ((long long)a.blocks * a.G > 65535) return PG_ERR_ARG;
  auto kern = attn_rows_kernel<TQ, TC, DC, VC, MT, KT, R8>;
  constexpr size_t kOut = (size_t)kWarps * 16 * MT * (64 * VC + 4) * 4, kIn = (size_t)kWarps * (K::Q_BYTES + kRing), kMost = kIn > kOut ? kIn : kOut;
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.nsplit, a.G * a.blocks, p.entries);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (a.cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.nsplit;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pg_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  pg_count_launch(1);
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) return PG_ERR_CUDA;
  if (bytes > 0 && pg::launch_kernel(attn_rows_merge_kernel<TQ>, dim3(a.H, max_n, p.entries), dim3(128), 0, st, a) != cudaSuccess) return PG_ERR_CUDA;
  return PG_OK;
}

template <typename TQ, typename TC, int MT, int KT, bool R8>
int by_size(const PgAttnRows& p, const Args& a, long long* need, long long scratch_bytes, cudaStream_t st) {
  if (a.dim <= 64 && a.vdim <= 64) return launch<TQ, TC, 1, 1, MT, KT, R8>(p, a, need, scratch_bytes, st);
  constexpr int kWide = sizeof(TC) == 1 && MT == 1 ? KT : 16;
  return launch<TQ, TC, 2, 2, MT, kWide, R8>(p, a, need, scratch_bytes, st);
}
template <typename TQ, typename TC, int KT>
int by_rows(const PgAttnRows& p, const Args& a, long long* need, long long scratch_bytes, cudaStream_t st) {
  const int rows = (p.singles ? 1 : p.max_n) * (p.H / p.G);
  if (rows <= 8) return by_size<TQ, TC, 1, KT, true>(p, a, need, scratch_bytes, st);
  // 32 rows a warp read and convert a tile once where there are CTAs enough (24 trees of 8 x 4 rows over codes, 16 / 32 rows a warp 40 / 34 us; 16 x 4 rows 67 / 53); else, and where
  // nothing is converted, 16 for a shorter chain (one tree of 8 x 4 rows 14 / 18; 24 over bf16 pages 41 / 46)
  if (rows <= 16 || sizeof(TQ) == 4 || (sizeof(TC) == 2 && rows <= 32) || (long long)p.busy * p.G * 2 < pg::num_sms()) return by_size<TQ, TC, 1, KT, false>(p, a, need, scratch_bytes, st);
  return by_size<TQ, TC, sizeof(TQ) == 4 ? 1 : 2, KT, false>(p, a, need, scratch_bytes, st);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int attn_rows(const PgAttnRows* q, long long* need, void* scratch, long long scratch_bytes, void* stream) {
  if (q == nullptr) return PG_ERR_ARG;
  const PgAttnRows& p = *q;
  if (p.entries <= 0 || p.entries > 65535 || p.rows <= 0 || p.max_n <= 0 || p.max_n > 65535 || p.H <= 0 || p.G <= 0 || p.H % p.G != 0 || p.H > 65535 || p.dim <= 0 || p.vdim <= 0 ||
      p.max_pages <= 0 || p.longest <= 0)
    return PG_ERR_ARG;
  if (p.page < 32 || (p.page & (p.page - 1)) != 0 || p.dim > 128 || p.vdim > 128 || (p.tree != nullptr && p.tree_words <= 0)) return PG_ERR_ARG;
  const int unit = p.e4m3 ? 16 : p.act_f32 ? 4 : 8;  // elements of a 16-byte piece
  if (p.dim % unit != 0 || p.vdim % (p.e4m3 ? 16 : 8) != 0 || !aligned(p.k, 16) || !aligned(p.v, 16)) return PG_ERR_ARG;
  if (p.e4m3 && (p.k_powers == nullptr || p.v_powers == nullptr || !aligned(p.k_powers, 16) || !aligned(p.v_powers, 16))) return PG_ERR_ARG;
  const PgAttnScore* sx = p.score;
  if (sx != nullptr && ((sx->dist_a == nullptr) != (sx->dist_b == nullptr))) return PG_ERR_ARG;
  if (p.pos == nullptr && sx != nullptr && (sx->window > 0 || sx->dist_a != nullptr)) return PG_ERR_ARG;
  Args a{};
  a.q = p.q;
  a.kp = static_cast<const uint8_t*>(p.k), a.vp = static_cast<const uint8_t*>(p.v);
  a.ke = static_cast<const uint8_t*>(p.k_powers), a.ve = static_cast<const uint8_t*>(p.v_powers);
  a.gate = p.gate, a.ldg = p.ldg, a.out = p.out, a.partial = static_cast<float*>(scratch);
  a.row0 = p.entry_row0, a.n = p.entry_n, a.ctx = p.entry_ctx, a.pt = p.page_table, a.pos = p.pos, a.tree = static_cast<const uint32_t*>(p.tree);
  a.words = p.tree_words, a.max_pages = p.max_pages, a.page = p.page, a.max_n = p.max_n, a.singles = p.singles, a.H = p.H, a.G = p.G, a.dim = p.dim, a.vdim = p.vdim;
  a.scale = p.scale, a.softcap = p.softcap, a.gate_per_head = p.gate_per_head;
  a.sx = sx != nullptr ? *sx : PgAttnScore{};
  a.mode = a.sx.dist_a != nullptr || a.sx.logistic ? kGeneral : p.softcap > 0.f ? kCapped : kPlain;
  const int four = p.act_f32 ? 16 : 8;  // bytes of four elements
  a.vec_q = aligned(p.q, four), a.vec_gate = aligned(p.gate, four) && p.ldg % 4 == 0, a.vec_out = aligned(p.out, four) && a.sx.out_ld % 4 == 0;
  a.trigger = pg::weights_follow();
  if ((long long)p.max_n * (p.H / p.G) > 1 << 24) return PG_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.e4m3) return p.act_f32 ? by_rows<float, e4m3, 32>(p, a, need, scratch_bytes, st) : by_rows<bf16, e4m3, 32>(p, a, need, scratch_bytes, st);
  return p.act_f32 ? by_rows<float, float, 16>(p, a, need, scratch_bytes, st) : by_rows<bf16, bf16, 32>(p, a, need, scratch_bytes, st);
}

}  // namespace

extern "C" long long pg_attn_rows_scratch(const PgAttnRows* p) {
  long long need = 0;
  const int rc = attn_rows(p, &need, nullptr, 0, nullptr);
  return rc == PG_OK ? need : rc;
}

extern "C" int pg_attn_rows(const PgAttnRows* p, void* scratch, long long scratch_bytes, void* stream) { return attn_rows(p, nullptr, scratch, scratch_bytes, stream); }
