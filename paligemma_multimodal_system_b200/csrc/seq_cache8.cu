// The 8-bit paged cache (cache8.cuh): rows on their way in and out.
//
//   pg_attn_prepare_e4m3   the front end of softmax attention (pg_attn_prepare) whose keys and values leave as 8-bit codes
//   pg_kv_read_e4m3        the rows of entries of several tokens back into the activations' type, for prompt attention
#include "cache8.cuh"
#include "common.cuh"
#include "paligemma_b200.h"

using bf16 = __nv_bfloat16;

namespace {

__device__ __forceinline__ double wsum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const bf16* p) { return __bfloat162float(*p); }

// eight neighbouring elements as they lie in memory; VEC: on 16-byte boundaries
template <typename TA>
struct Eight {
  uint4 u[sizeof(TA) / 2];
  template <bool VEC>
  __device__ __forceinline__ void load(const TA* p) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(TA) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      TA* e = reinterpret_cast<TA*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(TA) / 2); ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = sizeof(TA) == 4 ? __uint_as_float(w[i]) : __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};
__device__ __forceinline__ void put8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void put8(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pg::pack_bf16(v[0], v[1]), pg::pack_bf16(v[2], v[3]), pg::pack_bf16(v[4], v[5]), pg::pack_bf16(v[6], v[7]));
}

constexpr float kDoubt = 0x1p-20f;  // no further are fp32 elements from the exact ones, relative to their size (12 half steps of 2^-24 without a turn, which cancels more in a few)
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float up) {
  return make_uint2(cache8::codes_of(x[0] * up, x[1] * up) | cache8::codes_of(x[2] * up, x[3] * up) << 16,
                    cache8::codes_of(x[4] * up, x[5] * up) | cache8::codes_of(x[6] * up, x[7] * up) << 16);
}
// to fp32 towards zero, the last bit set where something was cut off: what is rounded to fewer bits from here is rounded once
__device__ __forceinline__ float to_odd(double y) {
  const float f = __double2float_rz(y);
  return static_cast<double>(f) != y ? __uint_as_float(__float_as_uint(f) | 1u) : f;  // (NaN stays NaN)
}

using Prepare = PgPrepareE4m3;
static_assert(sizeof(PgPrepareE4m3) == 192 && sizeof(PgReadE4m3) == 112, "callers pack these structs by their sizes");

// A group of LG lanes holds a head vector, eight elements a lane; its mean square and its largest element are butterflies inside the group.  A CTA takes TOK tokens, whose cosines
// and sines (angles in double) are made once for all heads behind the first vectors' requests; four vectors of a group are under way together: one head of four tokens,
// which share its weights, or four heads of one token.
// Elements that a norm or a rotation computes are fp32; where that could choose the code beside the nearest (one in a million would be), the head's vector is marked and made again
// in double behind the loop, so that the codes are those of the exact elements -- but for one in some ten million that a rotation or a blend leaves small beside its parts, whose
// errors count by those (doubting by the parts: 37.7 us for the first size below against 34.4; 30.8 without any of it).  Inside the loop the second making cost 36.9: its registers
// are live beside four vectors'.
// What bounds it: for prompts instructions, then the bytes (a row is read once, 8-bit rows are half of bf16 ones); for a few rows the chain row -> sum -> largest -> codes.
// 7,796 bf16 rows of 32 + 8 + 8 heads of 64, normed and turned, in 34.4 us (2.6 of 6.6 TB/s; 28.8 into pages of bf16); 1,363 fp32 rows of 16 + 4 + 4 heads of 128 as they come in 12.4;
// 23 rows in 6.2.
template <typename TA, int LG, int TOK, bool VEC>
__global__ void __launch_bounds__(128, sizeof(TA) == 2 ? 7 : 5) attn_prepare_e4m3_kernel(const __grid_constant__ Prepare a) {
  constexpr int U = 4, NG = 128 / LG, HEADS = TOK == 1 ? U : 1;  // HEADS: head vectors of a round
  extern __shared__ __align__(16) double cs64[];  // [TOK][cos rot / 2 | sin rot / 2], behind them the same in fp32 and a bit per key or value head and token
  float* cs = reinterpret_cast<float*>(cs64 + (TOK * a.rot + 1) / 2 * 2);
  uint32_t* doubtful = reinterpret_cast<uint32_t*>(cs + TOK * a.rot);
  __shared__ double part[2][TOK][4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = tid % LG, group = tid / LG, d0 = 8 * l;
  const int t0 = blockIdx.x * TOK, nvec = a.H + 2 * a.G, half = a.rot / 2;
  const TA* qkv = static_cast<const TA*>(a.qkv);
  __shared__ long long kv_row[TOK], power_row[TOK];  // a token's row of codes, its byte of a page's first head
  pg::griddep_begin();
  if (tid < TOK) {
    const int t = min(t0 + tid, a.rows - 1), where = a.at[t], slot = where % a.page;
    const long long page = a.page_table[(long long)a.row_entry[t] * a.max_pages + where / a.page];
    kv_row[tid] = page * a.page + slot;
    power_row[tid] = page * a.G * a.page + slot;
  }
  Eight<TA> raw[U];
  const TA* rows[TOK];
#pragma unroll
  for (int k = 0; k < TOK; ++k) rows[k] = qkv + min(t0 + k, a.rows - 1) * a.ld + d0;
  auto request = [&](int vec0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int vec = TOK == 1 ? vec0 + u * NG : vec0;
      raw[u].zero();
      if (vec < nvec && d0 < (vec < a.H + a.G ? a.dim : a.vdim)) {
        const int off = vec < a.H + a.G ? vec * a.dim : a.v_from_k ? (vec - a.G) * a.dim : (a.H + a.G) * a.dim + (vec - a.H - a.G) * a.vdim;
        raw[u].template load<VEC>(rows[TOK == 1 ? 0 : u] + off);
      }
    }
  };
  request(group);
  for (int i = tid; i < (2 * a.G * TOK + 31) / 32; i += 128) doubtful[i] = 0u;
  for (int i = tid; i < TOK * half; i += 128) {
    const int k = i / half, j = i - k * half;
    double s, c;
    sincos((double)a.pos[min(t0 + k, a.rows - 1)] * a.freq[j], &s, &c);
    cs[k * a.rot + j] = static_cast<float>(cs64[k * a.rot + j] = a.rot_gain * c);
    cs[k * a.rot + half + j] = static_cast<float>(cs64[k * a.rot + half + j] = a.rot_gain * s);
  }
  if (a.norm_qk == 2) {  // one root mean square for all of q, one for all of k
    const int nq = a.H * a.dim, nk = a.G * a.dim;
#pragma unroll 1
    for (int k = 0; k < TOK; ++k) {
      const TA* row = qkv + (long long)min(t0 + k, a.rows - 1) * a.ld;
      double sq = 0.0, sk = 0.0;
      for (int d = tid; d < nq; d += 128) { const double x = ldf(row + d); sq = fma(x, x, sq); }
      for (int d = tid; d < nk; d += 128) { const double x = ldf(row + nq + d); sk = fma(x, x, sk); }
      sq = wsum(sq);
      sk = wsum(sk);
      if (lane == 0) { part[0][k][warp] = sq; part[1][k][warp] = sk; }
    }
  }
  __syncthreads();
  const bool turn8 = a.rot % 8 == 0 && half % 4 == 0;  // a lane's four pairs turn or do not, and lie on 16 bytes
  for (int vec0 = group; vec0 - group < nvec; vec0 += HEADS * NG) {
    Eight<TA> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = raw[u];
    request(vec0 + HEADS * NG);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int vec = vec0 + h * NG;
      const bool is_q = vec < a.H, is_k = !is_q && vec < a.H + a.G, is_v = !is_q && !is_k;
      const int n = is_v ? a.vdim : a.dim, head = is_q ? vec : is_k ? vec - a.H : vec - a.H - a.G;
      const float mean = 1.0f / (float)n;
      const bool mine = vec < nvec && d0 < n, quantised = __any_sync(0xffffffffu, !is_q);  // a group of this warp has a key or a value
      float w[8];
      const float* wp = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;  // NULL: a norm without a weight
      if (wp != nullptr && mine) {
        wp += a.norm_qk == 2 ? head * a.dim + d0 : d0;
        if (VEC) {
          const float4 lo = reinterpret_cast<const float4*>(wp)[0], hi = reinterpret_cast<const float4*>(wp)[1];
          w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = wp[i];
        }
      }
#pragma unroll
      for (int k = 0; k < TOK; ++k) {
        const int u = TOK == 1 ? h : k;
        const long long t = t0 + k;
        float x[8];
        now[u].get(x);
        float inv = 1.0f;
        if (a.norm_qk == 1 || a.norm_v) {  // (uniform: every lane takes part in the exchange)
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
#pragma unroll
          for (int o = LG / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (is_v ? a.norm_v != 0 : a.norm_qk == 1) inv = rsqrtf(s * mean + a.eps);
        }
        if (a.norm_qk == 2 && !is_v) {
          const double* p = part[is_q ? 0 : 1][k];
          inv = rsqrtf(static_cast<float>(p[0] + p[1] + p[2] + p[3]) / (float)((is_q ? a.H : a.G) * a.dim) + a.eps);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        if (mine) {
          if (wp != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= w[i];
          }
          if (!is_v && d0 < a.rot) {
            const float* ck = cs + k * a.rot + d0 / 2;
            float cv[4], sv[4];
            if (turn8) {
              const float4 c4 = *reinterpret_cast<const float4*>(ck), s4 = *reinterpret_cast<const float4*>(ck + half);
              cv[0] = c4.x, cv[1] = c4.y, cv[2] = c4.z, cv[3] = c4.w;
              sv[0] = s4.x, sv[1] = s4.y, sv[2] = s4.z, sv[3] = s4.w;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool turns = d0 + 2 * i < a.rot;
                cv[i] = turns ? ck[i] : 1.f;
                sv[i] = turns ? ck[half + i] : 0.f;
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float y = x[2 * i], z = x[2 * i + 1];
              x[2 * i] = y * cv[i] - z * sv[i];
              x[2 * i + 1] = z * cv[i] + y * sv[i];
            }
          }
          if (is_v && a.v_other != nullptr && t < a.rows) {
            const TA* o = static_cast<const TA*>(a.v_other) + t * a.ld_v_other + (long long)head * a.vdim + d0;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (1.0f - a.v_mix) * x[i] + a.v_mix * ldf(o + i);
          }
        }
        float top = 0.f;
        if (quantised) {
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));  // (passes over NaN)
#pragma unroll
          for (int o = LG / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (quantised && __any_sync(0xffffffffu, top == INFINITY)) {  // only finite elements count, infinities are kept as NaN
          uint32_t most = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) most = max(most, cache8::finite_magnitude(x[i]));
#pragma unroll
          for (int o = LG / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
          top = __uint_as_float(most);
          if (!is_q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fabsf(x[i]) < INFINITY ? x[i] : __uint_as_float(0x7fffffffu);
          }
        }
        if (!mine || t >= a.rows) continue;
        if (is_q) {
          put8(static_cast<TA*>(a.q_out) + t * (a.H * a.dim) + (head * a.dim + d0), x);
        } else {
          const uint32_t byte = cache8::power_of(__float_as_uint(top));
          const float up = cache8::inverse_of_power(byte);
          if (is_k ? a.norm_qk != 0 || d0 < a.rot : a.norm_v != 0 || a.v_other != nullptr) {  // (else it is what came)
            const uint2 more = codes8(x, up * (1.f + kDoubt)), less = codes8(x, up * (1.f - kDoubt));
            if (more.x != less.x || more.y != less.y ||
                cache8::power_of(__float_as_uint(top * (1.f + kDoubt))) != cache8::power_of(__float_as_uint(top * (1.f - kDoubt))))
              atomicOr(&doubtful[((vec - a.H) * TOK + k) / 32], 1u << ((vec - a.H) * TOK + k) % 32);
          }
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_k ? a.k_codes : a.v_codes) + kv_row[k] * (a.G * n) + (head * n + d0)) = codes8(x, up);
          if (l == 0) static_cast<uint8_t*>(is_k ? a.k_powers : a.v_powers)[power_row[k] + head * a.page] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
  // Codes that a little more or less would change, by elements in double.  The groups of a warp make the same vector, the first one writes it.
  __syncthreads();
  for (int word = warp; word < (2 * a.G * TOK + 31) / 32; word += 4) {
    for (uint32_t left = doubtful[word]; left != 0; left &= left - 1) {
      const int bit = 32 * word + __ffs(left) - 1, k = bit % TOK, vec = bit / TOK;
      const bool is_v = vec >= a.G;
      const int n = is_v ? a.vdim : a.dim, head = is_v ? vec - a.G : vec;
      const bool mine = d0 < n;
      Eight<TA> again;
      float x[8];
      double y[8], scale = 1.0;
      again.zero();
      if (mine) again.template load<VEC>(rows[k] + (is_v && !a.v_from_k ? (a.H + a.G) * a.dim + head * a.vdim : (a.H + head) * a.dim));
      again.get(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      if (is_v ? a.norm_v != 0 : a.norm_qk == 1) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fma(y[i], y[i], sum);
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        scale = 1.0 / sqrt(sum / n + static_cast<double>(a.eps));
      } else if (!is_v && a.norm_qk == 2) {
        const double* p = part[1][k];
        scale = 1.0 / sqrt((p[0] + p[1] + p[2] + p[3]) / (a.G * a.dim) + static_cast<double>(a.eps));
      }
      float top = 0.f;
      if (mine) {
        const float* wp = is_v || a.k_norm == nullptr ? nullptr : a.k_norm + (a.norm_qk == 2 ? head * a.dim + d0 : d0);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= wp != nullptr ? scale * wp[i] : scale;
        if (!is_v && d0 < a.rot) {
          const double* ck = cs64 + k * a.rot + d0 / 2;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (d0 + 2 * i >= a.rot) break;
            const double p = y[2 * i], r = y[2 * i + 1];
            y[2 * i] = p * ck[i] - r * ck[half + i];
            y[2 * i + 1] = r * ck[i] + p * ck[half + i];
          }
        }
        if (is_v && a.v_other != nullptr) {
          const TA* o = static_cast<const TA*>(a.v_other) + static_cast<long long>(t0 + k) * a.ld_v_other + (long long)head * a.vdim + d0;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = (1.0 - static_cast<double>(a.v_mix)) * y[i] + static_cast<double>(a.v_mix) * static_cast<double>(ldf(o + i));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = to_odd(y[i]);
          if (fabsf(x[i]) < INFINITY) top = fmaxf(top, fabsf(x[i]));
          else x[i] = __uint_as_float(0x7fffffffu);
        }
      }
#pragma unroll
      for (int o = LG / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!mine || lane >= LG) continue;
      const uint32_t byte = cache8::power_of(__float_as_uint(top));
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_v ? a.v_codes : a.k_codes) + kv_row[k] * (a.G * n) + (head * n + d0)) = codes8(x, cache8::inverse_of_power(byte));
      if (l == 0) static_cast<uint8_t*>(is_v ? a.v_powers : a.k_powers)[power_row[k] + head * a.page] = static_cast<uint8_t>(byte);
    }
  }
}

// 16 codes (bf16: two 16-byte pieces of output) or four (fp32: one) a thread and step, fp32 four steps under way together; a CTA's 16 rows lie in one page.  Rows behind an entry's last one up to the end of its last run of 64
// are zeros: whoever walks whole tiles of the scratch reads numbers.  What bounds it: the bytes, half again as many as it writes in bf16.
// 7,796 rows of 2 x 8 heads of 64 to bf16 in 8.3 us (2.9 of 6.6 TB/s).
constexpr int kReadRows = 16;
template <typename TO>
__global__ void __launch_bounds__(256) kv_read_e4m3_kernel(const __grid_constant__ PgReadE4m3 a) {
  constexpr int E = sizeof(TO) == 2 ? 16 : 4, U = sizeof(TO) == 2 ? 1 : 4;  // codes of a piece; pieces of a thread and round
  pg::griddep_begin();
  const int e = blockIdx.y, n = a.entry_n[e], len = a.entry_ctx[e] + n, j0 = blockIdx.x * kReadRows;
  const int end = (len + 63) / 64 * 64;  // the scratch has whole runs of 64 rows
  if (n <= 1 || j0 >= end) return;
  const bool is_k = blockIdx.z == 0;
  const int size = is_k ? a.dim : a.vdim, width = a.G * size, pieces = width / E;
  const long long id = j0 < len ? a.page_table[(long long)e * a.max_pages + j0 / a.page] : 0;
  const int slot0 = j0 % a.page, rows = min(kReadRows, end - j0), held = len - j0;
  const uint8_t* codes = static_cast<const uint8_t*>(is_k ? a.k_codes : a.v_codes) + (id * a.page + slot0) * width;
  const uint8_t* powers = static_cast<const uint8_t*>(is_k ? a.k_powers : a.v_powers) + id * a.G * a.page + slot0;
  TO* out = static_cast<TO*>(is_k ? a.k_out : a.v_out) + (a.dense_row0[e] + (long long)j0) * width;
  for (int i0 = threadIdx.x; i0 < rows * pieces; i0 += 256 * U) {
    uint32_t c[U][E / 4], byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u, r = i / pieces, at = (i - r * pieces) * E;
      byte[u] = 0;
#pragma unroll
      for (int y = 0; y < E / 4; ++y) c[u][y] = 0u;
      if (r < rows && r < held) {
        const uint8_t* p = codes + r * width + at;
        if constexpr (E == 16) {
          const uint4 w = *reinterpret_cast<const uint4*>(p);
          c[u][0] = w.x, c[u][1] = w.y, c[u][2] = w.z, c[u][3] = w.w;
        } else {
          c[u][0] = *reinterpret_cast<const uint32_t*>(p);
        }
        byte[u] = powers[at / size * a.page + r];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u;
      if (i >= rows * pieces) break;
      const float s = cache8::value_of_power(byte[u]);
      float v[E];
#pragma unroll
      for (int y = 0; y < E / 2; ++y) {
        const uint32_t two = cache8::halves_of(c[u][y / 2] >> (16 * (y % 2)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
        v[2 * y] = f.x * s;
        v[2 * y + 1] = f.y * s;
      }
      uint4* dst = reinterpret_cast<uint4*>(out + (long long)i * E);
      if constexpr (E == 16) {
#pragma unroll
        for (int y = 0; y < 16; y += 8)
          dst[y / 8] = make_uint4(pg::pack_bf16(v[y], v[y + 1]), pg::pack_bf16(v[y + 2], v[y + 3]), pg::pack_bf16(v[y + 4], v[y + 5]), pg::pack_bf16(v[y + 6], v[y + 7]));
      } else {
        dst[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int pg_attn_prepare_e4m3(const PgPrepareE4m3* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  Prepare a = *args;
  if (a.rows <= 0 || a.H <= 0 || a.G <= 0 || a.dim <= 0 || a.vdim <= 0 || a.rot < 0 || a.rot > a.dim || (a.rot & 1) || a.page <= 0 || a.max_pages <= 0) return PG_ERR_ARG;
  if (a.dim % 16 != 0 || a.vdim % 16 != 0 || a.dim > 256 || a.vdim > 256 || (a.v_from_k && a.vdim != a.dim) || a.norm_qk < 0 || a.norm_qk > 2) return PG_ERR_ARG;
  if (!aligned16(a.q_out) || !aligned16(a.k_codes) || !aligned16(a.v_codes) || a.k_codes == nullptr || a.v_codes == nullptr || a.k_powers == nullptr || a.v_powers == nullptr)
    return PG_ERR_ARG;
  if (a.at == nullptr) a.at = a.pos;
  const int rows = a.rows, rot_dims = a.rot, act_f32 = a.act_f32;
  const auto smem = [&](int tokens) { return static_cast<size_t>(tokens * rot_dims + 4) * 12 + static_cast<size_t>(2ll * a.G * tokens + 31) / 32 * 4; };
  const int lanes = (a.dim > a.vdim ? a.dim : a.vdim) / 8;
  const bool vec = aligned16(a.qkv) && a.ld % (act_f32 ? 4 : 8) == 0 && aligned16(a.q_norm) && aligned16(a.k_norm);
  const bool four = rows >= 16 * pg::num_sms();  // four tokens a CTA once that still fills the SMs
  pg_count_launch(1);
  cudaError_t rc;
#define PG_P8(TA, LG)                                                                                                                                       \
  rc = four ? (vec ? pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 4, true>, dim3((rows + 3) / 4), dim3(128), smem(4), st, a)   \
                   : pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 4, false>, dim3((rows + 3) / 4), dim3(128), smem(4), st, a)) \
            : (vec ? pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 1, true>, dim3(rows), dim3(128), smem(1), st, a)                 \
                   : pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 1, false>, dim3(rows), dim3(128), smem(1), st, a))
#define PG_P8T(TA)               \
  if (lanes <= 4) PG_P8(TA, 4);       \
  else if (lanes <= 8) PG_P8(TA, 8);  \
  else if (lanes <= 16) PG_P8(TA, 16); \
  else PG_P8(TA, 32)
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (act_f32) { PG_P8T(float); }
  else { PG_P8T(bf16); }
#undef PG_P8T
#undef PG_P8
  return rc == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}

extern "C" int pg_kv_read_e4m3(const PgReadE4m3* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgReadE4m3& a = *args;
  if (a.entries <= 0 || a.entries > 65535 || a.longest <= 0 || a.G <= 0 || a.dim <= 0 || a.vdim <= 0 || a.dim % 16 != 0 || a.vdim % 16 != 0 || a.page <= 0 || a.page % kReadRows != 0 || a.max_pages <= 0)
    return PG_ERR_ARG;
  if (!aligned16(a.k_codes) || !aligned16(a.v_codes) || !aligned16(a.k_out) || !aligned16(a.v_out)) return PG_ERR_ARG;
  const dim3 grid(((a.longest + 63) / 64 * 64 + kReadRows - 1) / kReadRows, a.entries, 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t rc = a.out_f32 ? pg::launch_kernel(kv_read_e4m3_kernel<float>, grid, dim3(256), 0, st, a) : pg::launch_kernel(kv_read_e4m3_kernel<bf16>, grid, dim3(256), 0, st, a);
  return rc == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
