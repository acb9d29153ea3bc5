// The 8-bit paged cache (cache8.cuh): rows on their way in and out.
//
//   pg_attn_prepare_e4m3   the front end of softmax attention (pg_attn_prepare) whose keys and values leave as 8-bit codes
//   pg_kv_read_e4m3        the rows of entries of several tokens back into the activations' type, for prompt attention
#include "cache8.cuh"
#include "common.cuh"
#include "paligemma_b200.h"

using bf16 = __nv_bfloat16;

namespace {

__device__ __forceinline__ float wsum(float v) {
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

struct Prepare {
  const void* qkv;
  long long ld;
  const int *pos, *at, *row_entry, *page_table;
  int max_pages, page;
  const double* freq;
  const float *qn, *kn;
  void* q_out;
  uint8_t *kc, *ke, *vc, *ve;
  int rows, H, G, dim, vdim, rot;
  float eps;
  int norm_qk, norm_v, v_from_k;
  float rot_gain;
  const void* v_other;
  long long ldvo;
  float v_mix;
};

// A group of LG lanes holds a head vector, eight elements a lane; its mean square and its largest element are butterflies inside the group.  A CTA takes TOK tokens, whose cosines
// and sines (angles in double) are made once for all heads behind the first vectors' requests; four vectors of a group are under way together: one head of four tokens,
// which share its weights, or four heads of one token.
// What bounds it: for prompts instructions, then the bytes (a row is read once, 8-bit rows are half of bf16 ones); for a few rows the chain row -> sum -> largest -> codes.
template <typename TA, int LG, int TOK, bool VEC>
__global__ void __launch_bounds__(128) attn_prepare_e4m3_kernel(const __grid_constant__ Prepare a) {
  constexpr int U = 4, NG = 128 / LG, HEADS = TOK == 1 ? U : 1;  // HEADS: head vectors of a round
  extern __shared__ __align__(16) float cs[];  // [TOK][cos rot / 2 | sin rot / 2]
  __shared__ float part[2][TOK][4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = tid % LG, group = tid / LG, d0 = 8 * l;
  const int t0 = blockIdx.x * TOK, nvec = a.H + 2 * a.G, half = a.rot / 2;
  const TA* qkv = static_cast<const TA*>(a.qkv);
  long long kv_row[TOK], power_row[TOK];  // the token's row of codes, its byte of a page's first head
#pragma unroll
  for (int k = 0; k < TOK; ++k) {  // (positions and pages are the host's)
    const int t = min(t0 + k, a.rows - 1), where = a.at[t], slot = where % a.page;
    const long long page = a.page_table[(long long)a.row_entry[t] * a.max_pages + where / a.page];
    kv_row[k] = page * a.page + slot;
    power_row[k] = page * a.G * a.page + slot;
  }
  pg::griddep_begin();
  Eight<TA> raw[U];
  auto request = [&](int vec0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int vec = TOK == 1 ? vec0 + u * NG : vec0, t = min(t0 + (TOK == 1 ? 0 : u), a.rows - 1);
      raw[u].zero();
      if (vec < nvec && d0 < (vec < a.H + a.G ? a.dim : a.vdim)) {
        const long long off = vec < a.H + a.G ? vec * a.dim : a.v_from_k ? (vec - a.G) * a.dim : (a.H + a.G) * a.dim + (vec - a.H - a.G) * a.vdim;
        raw[u].template load<VEC>(qkv + t * a.ld + off + d0);
      }
    }
  };
  request(group);
  for (int i = tid; i < TOK * half; i += 128) {
    const int k = i / half, j = i - k * half;
    double s, c;
    sincos((double)a.pos[min(t0 + k, a.rows - 1)] * a.freq[j], &s, &c);
    cs[k * a.rot + j] = a.rot_gain * (float)c;
    cs[k * a.rot + half + j] = a.rot_gain * (float)s;
  }
  if (a.norm_qk == 2) {  // one root mean square for all of q, one for all of k
    const int nq = a.H * a.dim, nk = a.G * a.dim;
#pragma unroll 1
    for (int k = 0; k < TOK; ++k) {
      const TA* row = qkv + (long long)min(t0 + k, a.rows - 1) * a.ld;
      float sq = 0.f, sk = 0.f;
      for (int d = tid; d < nq; d += 128) { const float x = ldf(row + d); sq = fmaf(x, x, sq); }
      for (int d = tid; d < nk; d += 128) { const float x = ldf(row + nq + d); sk = fmaf(x, x, sk); }
      sq = wsum(sq);
      sk = wsum(sk);
      if (lane == 0) { part[0][k][warp] = sq; part[1][k][warp] = sk; }
    }
  }
  __syncthreads();
  const bool turn8 = a.rot % 8 == 0 && half % 4 == 0;  // a lane's four pairs turn or do not, and lie on 16 bytes
  for (int vec0 = group; vec0 - group < nvec; vec0 += HEADS * NG) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].get(v[u]);
    request(vec0 + HEADS * NG);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int vec = vec0 + h * NG;
      const bool is_q = vec < a.H, is_k = !is_q && vec < a.H + a.G, is_v = !is_q && !is_k;
      const int n = is_v ? a.vdim : a.dim, head = is_q ? vec : is_k ? vec - a.H : vec - a.H - a.G;
      const bool mine = vec < nvec && d0 < n;
      float w[8];
      const float* wp = is_v ? nullptr : is_q ? a.qn : a.kn;  // NULL: a norm without a weight
      if (wp != nullptr && mine) {
        wp += a.norm_qk == 2 ? head * a.dim + d0 : d0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = wp[i];
      }
#pragma unroll
      for (int k = 0; k < TOK; ++k) {
        const int u = TOK == 1 ? h : k;
        const long long t = t0 + k;
        float(&x)[8] = v[u];
        float inv = 1.0f;
        if (a.norm_qk == 1 || a.norm_v) {  // (uniform: every lane takes part in the exchange)
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
#pragma unroll
          for (int o = LG / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (is_v ? a.norm_v != 0 : a.norm_qk == 1) inv = rsqrtf(s * (1.0f / (float)n) + a.eps);
        }
        if (a.norm_qk == 2 && !is_v) {
          const float* p = part[is_q ? 0 : 1][k];
          inv = rsqrtf((p[0] + p[1] + p[2] + p[3]) / (float)((is_q ? a.H : a.G) * a.dim) + a.eps);
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
            const TA* o = static_cast<const TA*>(a.v_other) + t * a.ldvo + (long long)head * a.vdim + d0;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (1.0f - a.v_mix) * x[i] + a.v_mix * ldf(o + i);
          }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));  // (passes over NaN)
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (__any_sync(0xffffffffu, top == INFINITY)) {  // only finite elements count, infinities are kept as NaN
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
          put8(static_cast<TA*>(a.q_out) + (t * a.H + head) * a.dim + d0, x);
        } else {
          const uint32_t byte = cache8::power_of(__float_as_uint(top));
          const float up = cache8::inverse_of_power(byte);
          uint2 codes;
          codes.x = cache8::codes_of(x[0] * up, x[1] * up) | cache8::codes_of(x[2] * up, x[3] * up) << 16;
          codes.y = cache8::codes_of(x[4] * up, x[5] * up) | cache8::codes_of(x[6] * up, x[7] * up) << 16;
          *reinterpret_cast<uint2*>((is_k ? a.kc : a.vc) + (kv_row[k] * a.G + head) * n + d0) = codes;
          if (l == 0) (is_k ? a.ke : a.ve)[power_row[k] + head * a.page] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
}

// 16 codes a thread and step.  Rows behind an entry's last one up to the end of its last page are zeros: whoever walks whole tiles of the scratch reads numbers.
constexpr int kReadRows = 16;
template <typename TO>
__global__ void __launch_bounds__(256) kv_read_e4m3_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ ke, const uint8_t* __restrict__ vc, const uint8_t* __restrict__ ve,
                                                           const int* __restrict__ page_table, int max_pages, int page, const int* __restrict__ dense_row0,
                                                           const int* __restrict__ entry_n, const int* __restrict__ entry_ctx, TO* __restrict__ k_out, TO* __restrict__ v_out,
                                                           int G, int dim, int vdim) {
  pg::griddep_begin();
  const int e = blockIdx.y, n = entry_n[e], len = entry_ctx[e] + n, j0 = blockIdx.x * kReadRows;
  const int end = (len + 63) / 64 * 64;  // the scratch has whole runs of 64 rows
  if (n <= 1 || j0 >= end) return;
  const bool is_k = blockIdx.z == 0;
  const int size = is_k ? dim : vdim, pieces = G * size / 16, per_head = size / 16;
  const uint8_t* codes = is_k ? kc : vc;
  const uint8_t* powers = is_k ? ke : ve;
  TO* out = (is_k ? k_out : v_out) + (dense_row0[e] + (long long)j0) * G * size;
  const int rows = min(kReadRows, end - j0);
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * pieces; i += 256) {
    const int r = i / pieces, p = i - r * pieces, j = j0 + r, head = p / per_head;
    uint4 c = make_uint4(0, 0, 0, 0);
    uint32_t byte = 127;
    if (j < len) {
      const long long pg_id = page_table[(long long)e * max_pages + j / page];
      const int slot = j % page;
      c = *reinterpret_cast<const uint4*>(codes + (pg_id * page + slot) * G * size + 16 * p);
      byte = powers[(pg_id * G + head) * page + slot];
    }
    const float s = cache8::value_of_power(byte);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    TO* dst = out + (long long)r * G * size + 16 * p;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t two = cache8::halves_of(w[2 * h + q / 2] >> (16 * (q & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
        v[2 * q] = f.x * s;
        v[2 * q + 1] = f.y * s;
      }
      put8(dst + 8 * h, v);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int pg_attn_prepare_e4m3(const void* qkv, long long ld, const int* pos, const int* at, const int* row_entry, const int* page_table, int max_pages, int page,
                                    const double* freq, const float* q_norm, const float* k_norm, void* q_out, void* k_codes, void* k_powers, void* v_codes, void* v_powers, int rows,
                                    int H, int G, int dim, int vdim, int rot_dims, float eps, int norm_qk, int norm_v, int v_from_k, float rot_gain, const void* v_other,
                                    long long ld_v_other, float v_mix, int act_f32, void* stream) {
  if (rows <= 0 || H <= 0 || G <= 0 || dim <= 0 || vdim <= 0 || rot_dims < 0 || rot_dims > dim || (rot_dims & 1) || page <= 0 || max_pages <= 0) return PG_ERR_ARG;
  if (dim % 16 != 0 || vdim % 16 != 0 || dim > 256 || vdim > 256 || (v_from_k && vdim != dim) || norm_qk < 0 || norm_qk > 2) return PG_ERR_ARG;
  if (!aligned16(q_out) || !aligned16(k_codes) || !aligned16(v_codes) || k_codes == nullptr || v_codes == nullptr || k_powers == nullptr || v_powers == nullptr) return PG_ERR_ARG;
  const Prepare a{qkv, ld, pos, at != nullptr ? at : pos, row_entry, page_table, max_pages, page, freq, q_norm, k_norm, q_out, static_cast<uint8_t*>(k_codes),
                  static_cast<uint8_t*>(k_powers), static_cast<uint8_t*>(v_codes), static_cast<uint8_t*>(v_powers), rows, H, G, dim, vdim, rot_dims, eps, norm_qk, norm_v, v_from_k,
                  rot_gain, v_other, ld_v_other, v_mix};
  const int lanes = (dim > vdim ? dim : vdim) / 8;
  const bool vec = aligned16(qkv) && ld % (act_f32 ? 4 : 8) == 0;
  const bool four = rows >= 16 * pg::num_sms();  // four tokens a CTA once that still fills the SMs
  pg_count_launch(1);
  cudaError_t rc;
#define PG_P8(TA, LG)                                                                                                                                       \
  rc = four ? (vec ? pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 4, true>, dim3((rows + 3) / 4), dim3(128), (size_t)(4 * rot_dims + 4) * 4, st, a)   \
                   : pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 4, false>, dim3((rows + 3) / 4), dim3(128), (size_t)(4 * rot_dims + 4) * 4, st, a)) \
            : (vec ? pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 1, true>, dim3(rows), dim3(128), (size_t)(rot_dims + 4) * 4, st, a)                 \
                   : pg::launch_dependent(attn_prepare_e4m3_kernel<TA, LG, 1, false>, dim3(rows), dim3(128), (size_t)(rot_dims + 4) * 4, st, a))
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

extern "C" int pg_kv_read_e4m3(const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers, const int* page_table, int max_pages, int page,
                               const int* dense_row0, const int* entry_n, const int* entry_ctx, void* k_out, void* v_out, int entries, int longest, int G, int dim, int vdim,
                               int out_f32, void* stream) {
  if (entries <= 0 || entries > 65535 || longest <= 0 || G <= 0 || dim <= 0 || vdim <= 0 || dim % 16 != 0 || vdim % 16 != 0 || page <= 0 || max_pages <= 0) return PG_ERR_ARG;
  if (!aligned16(k_codes) || !aligned16(v_codes) || !aligned16(k_out) || !aligned16(v_out)) return PG_ERR_ARG;
  const dim3 grid(((longest + 63) / 64 * 64 + kReadRows - 1) / kReadRows, entries, 2);
  auto go = [&](auto kern, auto t) {
    using TO = decltype(t);
    return pg::launch_kernel(kern, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(k_powers),
                             static_cast<const uint8_t*>(v_codes), static_cast<const uint8_t*>(v_powers), page_table, max_pages, page, dense_row0, entry_n, entry_ctx,
                             static_cast<TO*>(k_out), static_cast<TO*>(v_out), G, dim, vdim);
  };
  const cudaError_t rc = out_f32 ? go(kv_read_e4m3_kernel<float>, float()) : go(kv_read_e4m3_kernel<bf16>, bf16());
  return rc == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
