// Which drafted tokens stay: rows of target logits (and of the draft's) against given random numbers.
//
// A row decides by itself where the walk goes on from it (the header has the rules), so rows are judged at once, a cluster of CTAs a row, and the walks are
// pointer chases at the end, made by the last cluster.  Rows lie depth first in their entries and clusters are started in the order of the rows' places in their
// entries: one that finds that some row above it goes on elsewhere has nothing to do (256 rows beside a draft 281 -> 257 us, 48 trees 149 -> 111 when it came).
//
// After rejections the rest is r_j = (p - c_j q)+ / S_j: from r_j q is taken again, (p - c_j q)+ - S_j q = p - (c_j + S_j) q where that is positive, so c and S are
// two numbers and a rejection is one pass over the row, whatever came before it.
//
// The results are whole numbers that hang on running sums: a draw is wrong once a sum is off by the distance of u from a token's border.  Weights e^((x - m) / T) from
// 2^-16 on are therefore made in double, 2^(j / 256) from a table times a polynomial of degree 3 (error below 2e-13); smaller ones in fp32, where a run of 128 holds no other.
//
// The nucleus is a threshold on the logit: the entries above which at most top_p Z lies.  Entries below (1 - top_p) Z / V cannot belong to it.  The others are
// counted by mass into 1024 runs of the ordered bit patterns, in fixed point (sums do not hang on their order).  The entries of the run that holds the border go to
// all CTAs and are compared one by one; where they are many the run is divided again, until it is one pattern.
//
// Two passes over a row, one for its maximum and one, from L2, for its sum; the second leaves the entries that may belong to the nucleus in shared memory, in the
// order of their places, and everything behind it goes over those (over the row where they are too many).  The CTAs of a row meet three times: for the maximum, for the sums and the
// counted runs, for the run that holds the border and the mass above it; the one that holds the drawn token finishes alone.
//
// What bounds it: few rows, that chain (5 rows 29 us, of which 5 are passes; 35 with seven meetings); many rows, how fast an SM takes them from L2 (6.7 TB/s over all while their
// passes coincide) and the chains between: 256 rows of 257216 beside a draft 251 us, 1.2 TB/s of DRAM, 36 % of the issue slots.  Greedy walks have a kernel of their own, one pass: 104 rows
// 27 us, 17 of which their bytes take (with a cluster a row as well 32, some rows left out).
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 512, kPerSm = 2, kWarps = kThreads / 32, kRanks = 16, kBins = 1024, kCoarse = kBins / 32, kTable = 256, kList = 32;
constexpr int kRun = 128, kRuns = 4;  // entries that a warp takes at once, a float4 a lane; runs under way
// entries of a row that a warp can hold as candidates of the nucleus: what shared memory leaves is L1, where the registers' overflow lies (256 rows of 257216 beside a draft, us with
// 256, 384, 512: 279 -- some rows need more --, 253, 261; 624 of 32000 104, 106, 109)
constexpr int kHeld = 384;
constexpr int kDead = -2147483647 - 1;
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;

struct Entry {
  unsigned long long mass;
  uint32_t key;
  int warp;  // that holds it
};
struct Candidate {
  float x;
  int at;  // place in the CTA's share
};
// e^((x - m) / T) = 2^(x a + shift) with a = log2(e) / T and shift = -m a.  (The rounding of m a is in every weight alike.)  Entries below `cut` weigh nothing: they are 2^-1000 of
// the largest or outside the nucleus.
struct Scale {
  double a, shift;
  float cut;
  // for fp32: a and shift in two parts, shift's first a multiple of 2^-8; runs with an entry of `fine` or more are weighed in double (all where it is -inf: what equals m has the mass, or
  // `low` is past fp32's end)
  float a0, a1, s0, s1, fine, low;
};
struct Row {  // a row's distribution: weights / mass
  Scale s;
  double mass;
  float bound;  // entries from here on are the candidates in shared memory (listed)
  bool good, listed, held;  // held: nothing else weighs anything
};
struct How {  // what makes one of a row of logits
  double temperature, top_p, a;  // a: log2(e) / temperature
  double border;  // log(16 (1 - top_p) / V): where the border of the nucleus is looked for, see there
};
struct __align__(16) Shared {
  How how[2];                              // of the draft, of the target
  Row row[2];
  double table[kTable];                    // 2^(j / 256)
  double warp[kWarps];
  double all[2][kRanks], part[2][kRanks];  // doubles of every CTA, by turns
  double warp_part[kWarps];
  unsigned long long top[2][kRanks];       // a CTA's largest entry and what the threads' largest ones sum up to
  unsigned long long hist[kBins];          // mass of runs of bit patterns
  unsigned long long coarse[kRanks][kCoarse], fine[kRanks][32];
  Entry own[kList], list[kRanks][kList];   // entries of the run that holds the border
  int held_count[kWarps], listed[kRanks], over[2][kRanks];
  unsigned long long found_base;
  float largest[kWarps];
  int found, pick, state, last, own_listed;
  uint32_t least, top_key;
  int V, bits;
  Candidate held[kWarps][kHeld];           // (in the end the rows' outcomes)
};
PG_DEVINL uint32_t ordered(float x) {  // larger numbers have larger ones; both zeros alike, NaN above all
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
PG_DEVINL float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
PG_DEVINL float max_nan(float a, float b) {  // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

PG_DEVINL float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
using pg::max3;

PG_DEVINL uint32_t remote(const void* p, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(pg::smem_u32(p)), "r"(rank));
  return there;
}
PG_DEVINL void put64(const void* p, int rank, unsigned long long v) { asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory"); }
PG_DEVINL void put32(const void* p, int rank, int v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory"); }
PG_DEVINL unsigned long long get64(const void* p, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
PG_DEVINL int load_relaxed(const int* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

PG_DEVINL Scale scale_of(float m, double a, double temperature) {
  Scale s;
  s.a = a;
  s.shift = -static_cast<double>(m) * s.a;
  s.cut = nextafterf(__double2float_rd(static_cast<double>(m) - 1000.0 * kLn2 * temperature), INFINITY);
  const bool equals = !(fabs(s.shift) < 0x1p40);  // the float in front of m weighs less than 2^-1000 here: what equals m shares the mass
  if (equals) s.a = s.shift = 0.0, s.cut = m;
  s.a0 = static_cast<float>(s.a);
  s.a1 = static_cast<float>(s.a - s.a0);
  s.s0 = static_cast<float>(rint(s.shift * 256.0) / 256.0);
  s.s1 = static_cast<float>(s.shift - s.s0);
  s.low = static_cast<float>((-100.0 - s.shift) * kLn2 * temperature);
  s.fine = fabs(s.shift) < 0x1p15 && !equals && s.low > -INFINITY ? static_cast<float>(static_cast<double>(m) - 16.0 * kLn2 * temperature) : -INFINITY;
  return s;
}
PG_DEVINL double weight(const double* table, const Scale& s, float x) {
  const double t = fma(static_cast<double>(x), s.a, s.shift);
  constexpr double kRound = 6755399441055744.0 / kTable;  // 1.5 2^52 / 256: its last place is 1 / 256
  const double rounded = t + kRound, f = t - (rounded - kRound);  // |f| <= 1 / 512
  const int k = __double2loint(rounded);
  const double power = table[k & (kTable - 1)];
  constexpr double c1 = kLn2, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
  const double w = fma(f, fma(f, fma(f, c3, c2), c1), 1.0) * __hiloint2double(__double2hiint(power) + ((k >> 8) << 20), __double2loint(power));
  return x >= s.cut ? w : 0.0;
}
// The same for weights below 2^-16 in fp32, each off by 2^-23 and without a bias: together by 2^-23 sqrt(2^-16) of the whole at most.  The argument is divided exactly: s0 - k is, x a0 is
// inside the instruction.  Taylor's polynomial of degree 7, |f| <= 1 / 2 (error 5e-9 at the ends, 6e-10 on average).  Entries below `low` count as 2^-100.  Two at a time: issue slots
// are what bounds the pass.
struct Pairs {
  uint64_t a0, a1, s0, s1;
  float low;
  PG_DEVINL explicit Pairs(const Scale& s) : a0(pg::pair_of(s.a0, s.a0)), a1(pg::pair_of(s.a1, s.a1)), s0(pg::pair_of(s.s0, s.s0)), s1(pg::pair_of(s.s1, s.s1)) {
    low = s.low;
  }
  PG_DEVINL float2 operator()(float x, float y) const {
    constexpr double c1 = kLn2, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5, c6 = c5 * c1 / 6, c7 = c6 * c1 / 7;
    constexpr float kRound = 12582912.0f;  // 1.5 2^23
    auto both = [](double c) { return pg::pair_of(static_cast<float>(c), static_cast<float>(c)); };
    const uint64_t z = pg::pair_of(fmaxf(x, low), fmaxf(y, low));
    const uint64_t rounded = pg::add_pair(pg::fma_pair(z, a0, s0), both(kRound)), k = pg::add_pair(rounded, both(-kRound));
    const uint64_t f = pg::add_pair(pg::fma_pair(z, a0, pg::fma_pair(k, both(-1.0), s0)), pg::fma_pair(z, a1, s1));
    uint64_t p = pg::fma_pair(f, both(c7), both(c6));
    p = pg::fma_pair(f, p, both(c5)), p = pg::fma_pair(f, p, both(c4)), p = pg::fma_pair(f, p, both(c3));
    p = pg::fma_pair(f, p, both(c2)), p = pg::fma_pair(f, p, both(c1)), p = pg::fma_pair(f, p, both(1.0));
    return make_float2(__uint_as_float(pg::lo_of(p) + (pg::lo_of(rounded) << 23)), __uint_as_float(pg::hi_of(p) + (pg::hi_of(rounded) << 23)));
  }
};

PG_DEVINL bool is_fine(const Scale& s, float4 x) { return __any_sync(0xffffffffu, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= s.fine); }
// the sum of four entries of a run (whole warps); the run alone says in which form
PG_DEVINL double weights_sum(const double* table, const Scale& s, const Pairs& small, float4 x) {
  if (is_fine(s, x)) return (weight(table, s, x.x) + weight(table, s, x.y)) + (weight(table, s, x.z) + weight(table, s, x.w));
  const float2 u = small(x.x, x.y), v = small(x.z, x.w);
  return static_cast<double>(((x.x >= s.cut ? u.x : 0.0f) + (x.y >= s.cut ? u.y : 0.0f)) + ((x.z >= s.cut ? v.x : 0.0f) + (x.w >= s.cut ? v.y : 0.0f)));
}

struct Part {  // a CTA's share of a row: entries lo .. lo + n of it; warp w has seg from w seg on
  int lo, n, seg, rank, ranks;
};
struct Source {  // a share in global memory (behind the first pass: in L2)
  const float* x;
  bool aligned;
  PG_DEVINL Source(const float* row, int lo) : x(row + lo), aligned((reinterpret_cast<uintptr_t>(row + lo) & 15) == 0) {}
  PG_DEVINL float4 four(int i, int n) const {  // entries i .. i + 3 of n, -inf behind
    if (aligned && i + 4 <= n) return __ldg(reinterpret_cast<const float4*>(x + i));
    return make_float4(i < n ? x[i] : -INFINITY, i + 1 < n ? x[i + 1] : -INFINITY, i + 2 < n ? x[i + 2] : -INFINITY, i + 3 < n ? x[i + 3] : -INFINITY);
  }
};

// f(first place, four entries) over entries begin .. end of the share, a warp's runs; whole warps
template <typename F>
PG_DEVINL void each4(const Part& p, const Source& s, int begin, int end, F f) {
  const int lane = threadIdx.x % 32;
  int i = begin;
  if (s.aligned)
    for (; i + kRun * kRuns <= end; i += kRun * kRuns) {
      const float4* from = reinterpret_cast<const float4*>(s.x + i) + lane;
      float4 x[kRuns];
#pragma unroll
      for (int k = 0; k < kRuns; ++k) x[k] = __ldg(from + k * (kRun / 4));
#pragma unroll
      for (int k = 0; k < kRuns; ++k) f(i + k * kRun + 4 * lane, x[k]);
    }
#pragma unroll 1
  for (; i < end; i += kRun) f(i + 4 * lane, s.four(i + 4 * lane, end));
}
template <typename F>
PG_DEVINL void each4(const Part& p, const Source& s, F f) {
  const int warp = threadIdx.x / 32;
  each4(p, s, warp * p.seg, min((warp + 1) * p.seg, p.n), f);
}

PG_DEVINL float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

PG_DEVINL unsigned long long warp_max(unsigned long long key) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  return key;
}

// The row's largest entry as an ordered pattern (a NaN above all), known to all CTAs, and in `whole` the sum of the largest entries' weights of all threads, scale being log2(e) / T:
// less than the row's.
PG_DEVINL uint32_t row_top(Shared& sh, const Part& p, const Source& s, int& turn, const double& scale, float& whole) {
  float best = -INFINITY;  // this thread's largest
  each4(p, s, [&](int, float4 x) { best = max_nan(max_nan(best, x.x, x.y), x.z, x.w); });
  const uint32_t key = __reduce_max_sync(0xffffffffu, ordered(best));
  uint32_t* mine = reinterpret_cast<uint32_t*>(sh.warp);
  __syncthreads();  // (the sums before have been read)
  if (threadIdx.x % 32 == 0) mine[threadIdx.x / 32] = key;
  __syncthreads();
  const float a = static_cast<float>(scale);  // (behind a barrier: the first row's may have been written just now)
  const uint32_t here = __reduce_max_sync(0xffffffffu, mine[threadIdx.x % kWarps]);
  float some = ex2((best - unordered(here)) * a);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) some += __shfl_xor_sync(0xffffffffu, some, o);
  if (threadIdx.x % 32 == 0) sh.largest[threadIdx.x / 32] = some;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < p.ranks) {
    some = 0.0f;
    for (int w = 0; w < kWarps; ++w) some += sh.largest[w];
    put64(&sh.top[turn][p.rank], threadIdx.x, static_cast<unsigned long long>(here) << 32 | __float_as_uint(some));
  }
  pg::cluster_sync_all();
  uint32_t top = 0;
  for (int r = 0; r < p.ranks; ++r) top = max(top, static_cast<uint32_t>(sh.top[turn][r] >> 32));
  whole = 0.0f;
  const float m = unordered(top);
  for (int r = 0; r < p.ranks; ++r) whole += __uint_as_float(static_cast<uint32_t>(sh.top[turn][r])) * ex2((unordered(static_cast<uint32_t>(sh.top[turn][r] >> 32)) - m) * a);
  turn ^= 1;
  return top;
}
PG_DEVINL bool is_distribution(uint32_t top) { return top > ordered(-INFINITY) && top < ordered(INFINITY); }

// What the warps have summed: theirs in sh.warp, the CTAs' in sh.all[turn] (until the next but one), the whole as the result.  The order of additions is fixed.  `over` of any
// thread becomes all CTAs'; `part`: a second sum.  counted: the runs of sh.hist go along, 32 at a time.
PG_DEVINL void share_coarse(Shared& sh, const Part& p) {
  const int lane = threadIdx.x % 32;
  for (int c = threadIdx.x / 32; c < kCoarse; c += kWarps) {
    unsigned long long v = sh.hist[c * 32 + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane < p.ranks) put64(&sh.coarse[p.rank][c], lane, v);
  }
}
PG_DEVINL double share_sums(Shared& sh, const Part& p, int& turn, double sum, bool over = false, double* part = nullptr, bool counted = false) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (part != nullptr) *part += __shfl_xor_sync(0xffffffffu, *part, o);
  }
  over = __syncthreads_or(over);  // (and the sums before have been read)
  if (lane == 0) {
    sh.warp[warp] = sum;
    if (part != nullptr) sh.warp_part[warp] = *part;
  }
  if (counted) share_coarse(sh, p);
  __syncthreads();
  if (warp == 0) {
    double all = lane < kWarps ? sh.warp[lane] : 0.0, all_part = part != nullptr && lane < kWarps ? sh.warp_part[lane] : 0.0;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      if (part != nullptr) all_part += __shfl_xor_sync(0xffffffffu, all_part, o);
    }
    all = __shfl_sync(0xffffffffu, all, 0);
    all_part = __shfl_sync(0xffffffffu, all_part, 0);
    if (lane < p.ranks) {
      put64(&sh.all[turn][p.rank], lane, __double_as_longlong(all));
      if (part != nullptr) {
        put64(&sh.part[turn][p.rank], lane, __double_as_longlong(all_part));
        put32(&sh.over[turn][p.rank], lane, over);
      }
    }
  }
  pg::cluster_sync_all();
  double total = 0.0;
  for (int r = 0; r < p.ranks; ++r) total += sh.all[turn][r];
  if (part != nullptr) {
    *part = 0.0;
    for (int r = 0; r < p.ranks; ++r) *part += sh.over[turn][r] ? NAN : sh.part[turn][r];
  }
  turn ^= 1;
  return total;
}

// Sums over the row: f(place, four entries) is their sum
template <typename F>
PG_DEVINL double row_mass(Shared& sh, const Part& p, const Source& s, int& turn, F f) {
  double sum = 0.0;
  each4(p, s, [&](int i, float4 x) { sum += f(i, x); });
  return share_sums(sh, p, turn, sum);
}
// and over the candidates: f(candidate)
template <typename F>
PG_DEVINL double held_mass(Shared& sh, const Part& p, int& turn, F f) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  double sum = 0.0;
  for (int i = lane; i < sh.held_count[warp]; i += 32) sum += f(sh.held[warp][i]);
  return share_sums(sh, p, turn, sum);
}

// Where u times the whole lies among n sums (n <= 32, one a lane): the first whose running sum is above `rest`, else the last with any mass; `run` becomes what lies in
// front of it.  -1 where none has any.  Whole warps; every lane has the result.
PG_DEVINL int place_among(double mine, int n, double rest, double& run) {
  const int lane = threadIdx.x % 32;
  double incl = lane < n ? mine : 0.0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double before = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += before;
  }
  const uint32_t some = __ballot_sync(0xffffffffu, lane < n && mine > 0.0), past = __ballot_sync(0xffffffffu, run + incl > rest) & some;
  const int at = past ? __ffs(past) - 1 : 31 - __clz(some);
  run += __shfl_sync(0xffffffffu, incl - (lane < n ? mine : 0.0), at & 31);
  return at;
}

// The token at u times the whole, whose sums are in sh.warp and sh.all (`turn` behind them): the first place whose running sum is above that.  Known to the CTA that holds it,
// `owner`, alone.  (Where rounding leaves no border behind u: the last place with any mass.)  find(warp, rest, run) gives the place from the share's first entry on, within that warp's
// part where that has any mass.  Where no sum is above zero the token is -1.
template <typename F>
PG_DEVINL int share_draw(Shared& sh, const Part& p, int turn, double total, float u, int& owner, F find) {
  const int lane = threadIdx.x % 32;
  double rest = static_cast<double>(u) * total, run = 0.0;
  owner = max(place_among(lane < p.ranks ? sh.all[turn ^ 1][lane] : 0.0, p.ranks, rest, run), 0);
  if (owner != p.rank) return -1;
  const int mine = place_among(lane < kWarps ? sh.warp[lane] : 0.0, kWarps, rest, run);
  if (mine < 0) return -1;  // (the same in the whole CTA)
  __syncthreads();  // (the warps' sums have been read)
  const int place = find(mine, rest, run);
  if (static_cast<int>(threadIdx.x) / 32 == mine && lane == 0) sh.pick = p.lo + place;
  __syncthreads();
  return sh.pick;
}
// (next: see next_with_mass.)
template <typename F, typename N>
PG_DEVINL int row_draw(Shared& sh, const Part& p, const Source& s, int turn, double total, float u, int& owner, F f, N next) {
  return share_draw(sh, p, turn, total, u, owner, [&](int mine, double rest, double run) {
    // all warps sum pieces of that warp's part, which then looks for the piece, the lane and the entry
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, begin = mine * p.seg, end = min(begin + p.seg, p.n);
    const int piece = (end - begin + kWarps * kRun - 1) / (kWarps * kRun) * kRun, from = min(begin + warp * piece, end), to = min(from + piece, end);
    double sum = 0.0;
    for (int i = from; i < to; i += kRun) {
      double w[4];
      f(i + 4 * lane, s.four(i + 4 * lane, to), w);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.warp[warp] = sum;
    __syncthreads();
    int place = -1, last = 0;
    if (warp == mine) {
      const int at = place_among(lane < kWarps ? sh.warp[lane] : 0.0, kWarps, rest, run);
      if (at < 0) return next(p.lo + end) - p.lo;
      const int begin2 = min(begin + at * piece, end), end2 = min(begin2 + piece, end);
      for (int i = begin2; i < end2 && place < 0; i += kRun) {
        double w[4];
        f(i + 4 * lane, s.four(i + 4 * lane, end2), w);
        const double four = (w[0] + w[1]) + (w[2] + w[3]);
        double all = four;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        const uint32_t some = __ballot_sync(0xffffffffu, four > 0.0);
        if (some == 0) continue;
        const int l0 = 31 - __clz(some), k0 = w[3] > 0.0 ? 3 : w[2] > 0.0 ? 2 : w[1] > 0.0 ? 1 : 0;
        last = i + 4 * l0 + __shfl_sync(0xffffffffu, k0, l0);
        if (run + all > rest) {
          double before = run;
          const int l = place_among(four, 32, rest, before);
          int k = -1, behind = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            before += w[j];
            if (w[j] > 0.0) {
              behind = j;
              if (k < 0 && before > rest) k = j;
            }
          }
          place = i + 4 * l + __shfl_sync(0xffffffffu, k < 0 ? behind : k, l);
        }
        run += all;
      }
    }
    return place < 0 ? last : place;
  });
}
template <typename F>
PG_DEVINL int held_draw(Shared& sh, const Part& p, int turn, double total, float u, int& owner, F f) {
  return share_draw(sh, p, turn, total, u, owner, [&](int mine, double rest, double run) {
    const int lane = threadIdx.x % 32;
    int place = -1, last = 0;
    if (static_cast<int>(threadIdx.x) / 32 == mine)
      for (int i = 0; i < sh.held_count[mine] && place < 0; i += 32) {
        const bool there = i + lane < sh.held_count[mine];
        const double w = there ? f(sh.held[mine][i + lane]) : 0.0;
        const uint32_t some = __ballot_sync(0xffffffffu, w > 0.0);
        if (some == 0) continue;
        double all = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        double before = run;
        const int l = run + all > rest ? place_among(w, 32, rest, before) : 31 - __clz(some);
        if (run + all > rest) place = sh.held[mine][i + l].at;
        last = sh.held[mine][i + l].at;
        run += all;
      }
    return place < 0 ? last : place;
  });
}

// An entry below this has (1 - top_p) z / V at most: even all of them together are not what the nucleus leaves out.
PG_DEVINL float least_of(float m, double z, double top_p, double temperature, int V) {
  const float x = __double2float_rd(static_cast<double>(m) + log((1.0 - top_p) * z / V) * temperature);
  return x - (fabsf(x) * 3e-7f + 1e-37f);
}

// Runs of bit patterns from hi down to lo, 1024 at most
struct Runs {
  uint32_t hi, lo;
  int shift;
  PG_DEVINL Runs(uint32_t hi_, uint32_t lo_) : hi(hi_), lo(lo_) { shift = hi - lo < kBins ? 0 : 32 - __clz(hi - lo) - 10; }
  PG_DEVINL int of(float x) const { return static_cast<int>((hi - ordered(x)) >> shift); }
};
PG_DEVINL void count_begin(Shared& sh) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
  if (threadIdx.x == 0) sh.own_listed = 0;
}

// Least entry of the nucleus.  z: the whole mass, `bits`: of the fixed point, each(f): f of every entry that may belong, runs: of these.  HELD: they are the candidates, counted already, and the
// mass of what is kept is left behind as share_sums leaves it (`mass`; < 0: it has to be summed).
template <bool HELD, typename E>
PG_DEVINL float nucleus(Shared& sh, const Part& p, const Scale& s, Runs runs, double z, double top_p, int bits, int& turn, double& mass, E each) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const double one = static_cast<double>(1ull << bits), border = top_p * z * one;
  unsigned long long base = 0;  // mass above the runs
  mass = -1.0;
  for (bool counted = HELD;; counted = false) {
    uint32_t &hi = runs.hi, &lo = runs.lo;
    const int shift = runs.shift;
    if (!counted) {
      __syncthreads();
      count_begin(sh);
      __syncthreads();
      const float least = unordered(lo), most = unordered(hi);
      each([&](float x) {
        if (x >= least && x <= most) atomicAdd(&sh.hist[runs.of(x)], static_cast<unsigned long long>(weight(sh.table, s, x) * one));
      });
      __syncthreads();
      share_coarse(sh, p);
      pg::cluster_sync_all();
    }
    int bin = 0;
#pragma unroll
    for (int step = 0; step < 2; ++step) {  // 32 runs of 32, then one of them
      if (step == 1) {
        for (int r = warp; r < p.ranks; r += kWarps) sh.fine[r][lane] = get64(sh.hist + bin * 32 + lane, r);
        __syncthreads();
      }
      if (warp == 0) {
        unsigned long long v = 0;
        for (int r = 0; r < p.ranks; ++r) v += step == 0 ? sh.coarse[r][lane] : sh.fine[r][lane];
        unsigned long long incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long before = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += before;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, static_cast<double>(base + incl) > border);
        const int at = past ? __ffs(past) - 1 : 31;
        if (lane == at) sh.found = past ? at : -1, sh.found_base = base + incl - v;
      }
      __syncthreads();
      if (sh.found < 0) break;  // (the border lies behind everything that may belong)
      base = sh.found_base;
      bin = bin * 32 + sh.found;
    }
    if (sh.found < 0) return unordered(lo);
    hi -= static_cast<uint32_t>(bin) << shift;
    if (shift == 0) return unordered(hi);
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    // the run's entries to all CTAs; where they are few it is decided at once
    const float run_least = unordered(lo), run_most = unordered(hi);
    double above = 0.0;
    each([&](float x) {
      if (x > run_most) {
        if (HELD) above += weight(sh.table, s, x);
      } else if (x >= run_least) {
        const int at = atomicAdd(&sh.own_listed, 1);
        if (at < kList) {
          sh.own[at].mass = static_cast<unsigned long long>(weight(sh.table, s, x) * one);
          sh.own[at].key = ordered(x);
          sh.own[at].warp = warp;
        }
      }
    });
    if (HELD) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (lane == 0) sh.warp[warp] = above;
    }
    __syncthreads();
    const int own = sh.own_listed;
    if (HELD) {
      above = lane < kWarps ? sh.warp[lane] : 0.0;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    }
    for (int r = warp; r < p.ranks; r += kWarps) {
      if (lane < min(own, kList)) {
        put64(&sh.list[p.rank][lane].mass, r, sh.own[lane].mass);
        put32(&sh.list[p.rank][lane].key, r, static_cast<int>(sh.own[lane].key));
      }
      if (lane == 0) {
        put32(&sh.listed[p.rank], r, own);
        if (HELD) put64(&sh.all[turn][p.rank], r, __double_as_longlong(above));
      }
    }
    if (threadIdx.x == 0) sh.least = hi;
    pg::cluster_sync_all();
    bool few = true;
    for (int r = 0; r < p.ranks; ++r) few = few && sh.listed[r] <= kList;
    if (few) {  // an entry belongs if what is above it does not pass the border
      for (int mine = warp; mine < p.ranks; mine += kWarps) {
        if (lane >= sh.listed[mine]) continue;
        const uint32_t key = sh.list[mine][lane].key;
        unsigned long long above = base;
        for (int r = 0; r < p.ranks; ++r)
          for (int i = 0; i < sh.listed[r]; ++i)
            if (sh.list[r][i].key > key) above += sh.list[r][i].mass;
        if (static_cast<double>(above) <= border) atomicMin(&sh.least, key);
      }
      __syncthreads();
      const uint32_t cut = sh.least;
      if (HELD) {  // what is kept of the run, beside what lies above it
        for (int r = warp; r < p.ranks; r += kWarps) {
          unsigned long long kept = lane < sh.listed[r] && sh.list[r][lane].key >= cut ? sh.list[r][lane].mass : 0ull;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
          if (lane == 0) sh.all[turn][r] += static_cast<double>(kept) / one;
        }
        if (warp == kWarps - 1 && lane < kWarps) {
          unsigned long long kept = 0;
          for (int i = 0; i < own; ++i) kept += sh.own[i].warp == lane && sh.own[i].key >= cut ? sh.own[i].mass : 0ull;
          sh.warp[lane] += static_cast<double>(kept) / one;
        }
        __syncthreads();
        mass = 0.0;
        for (int r = 0; r < p.ranks; ++r) mass += sh.all[turn][r];
        turn ^= 1;
      }
      return unordered(cut);
    }
    runs = Runs(hi, lo);
  }
}

struct Nucleus {
  double mass;  // of what is kept; < 0: not known
  float cut;
  int turn;
};
// (Out of line, like `distribution`: what they hold is not held in the loops over a row.)
__device__ __noinline__ Nucleus held_nucleus(Shared& sh, const Part p, const Scale s, const Runs runs, const double z, const double top_p, const int bits, int turn) {
  Nucleus r;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  r.cut = nucleus<true>(sh, p, s, runs, z, top_p, bits, turn, r.mass, [&](auto f) {
    for (int i = lane; i < sh.held_count[warp]; i += 32) f(sh.held[warp][i].x);
  });
  r.turn = turn;
  return r;
}
__device__ __noinline__ Nucleus row_nucleus(Shared& sh, const Part p, const Source x, const Scale s, const Runs runs, const double z, const double top_p, const int bits, int turn) {
  Nucleus r;
  r.cut = nucleus<false>(sh, p, s, runs, z, top_p, bits, turn, r.mass, [&](auto f) { each4(p, x, [&](int, float4 x) { f(x.x), f(x.y), f(x.z), f(x.w); }); });
  r.turn = turn;
  return r;
}

// The distribution of a row to sh.row[which]; its sums of the kept weights are left behind for a draw.  Returns `turn`.  (Once in the program: its loops are long.  By value: what has
// an address is loaded anew for every entry.  What lives longer than the loops lies in shared memory: they take all registers.)
PG_DEVINL int distribution(Shared& sh, const Part p, const Source s, const int which, int turn) {
  count_begin(sh);
  float some;
  const uint32_t top = row_top(sh, p, s, turn, sh.how[which].a, some);
  if (!is_distribution(top)) {
    if (threadIdx.x == 0) sh.row[which].good = false;
    __syncthreads();
    return turn;
  }
  const double temperature = sh.how[which].temperature;
  if (threadIdx.x == 0) sh.top_key = top;
  __syncthreads();  // (a warp without entries reads it at once)
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const float m = unordered(top);
  Scale sc = scale_of(m, sh.how[which].a, temperature);
  const bool in_fp32 = sc.fine > -INFINITY;
  const double whole = logf(fmaxf(1.0f, 0.99f * some));  // small is what is below 2^-16 of e^whole
  if (in_fp32) sc.fine += static_cast<float>(whole * temperature);
  // Candidates, in the order of their places: what is not small, and what probably belongs to the nucleus (an entry at its border weighs many times the mean of those outside;
  // sixteen times in most rows).
  float bound = sc.fine;
  if (sh.how[which].top_p < 1.0) bound = fminf(bound, static_cast<float>(static_cast<double>(m) + (sh.how[which].border + whole) * temperature));
  bound = fmaxf(bound, sc.cut);  // (the same number in all CTAs)
  int held = 0;
  double sum = 0.0;
  const Pairs small(sc);
  if (in_fp32)
    each4(p, s, [&](int i, float4 x) {
      float2 u = small(x.x, x.y), v = small(x.z, x.w);
      if (__any_sync(0xffffffffu, max3(fmaxf(x.x, x.y), x.z, x.w) >= bound)) {
        const float xs[4] = {x.x, x.y, x.z, x.w};
        u.x = x.x >= bound ? 0.0f : u.x, u.y = x.y >= bound ? 0.0f : u.y, v.x = x.z >= bound ? 0.0f : v.x, v.y = x.w >= bound ? 0.0f : v.y;
        int is = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) is |= xs[k] >= bound ? 1 << k : 0;
        const uint32_t front = (1u << lane) - 1, any = __ballot_sync(0xffffffffu, is != 0);
        int at = held + __popc(any & front), all = __popc(any);
        if (__any_sync(0xffffffffu, (is & (is - 1)) != 0)) {  // (a lane with several)
          const int count = __popc(is);
          const uint32_t b0 = __ballot_sync(0xffffffffu, count & 1), b1 = __ballot_sync(0xffffffffu, count & 2), b2 = __ballot_sync(0xffffffffu, count & 4);
          at = held + __popc(b0 & front) + 2 * __popc(b1 & front) + 4 * __popc(b2 & front);
          all = __popc(b0) + 2 * __popc(b1) + 4 * __popc(b2);
        }
        for (; is != 0; is &= is - 1, ++at) {
          const int k = __ffs(is) - 1;
          if (at < kHeld) sh.held[warp][at] = Candidate{k == 0 ? x.x : k == 1 ? x.y : k == 2 ? x.z : x.w, i + k};
        }
        held += all;
      }
      sum += static_cast<double>((u.x + u.y) + (v.x + v.y));
    });
  const bool over = !in_fp32 || held > kHeld;
  held = min(held, kHeld);
  if (lane == 0) sh.held_count[warp] = held;
  __syncwarp();
  double part = 0.0;
  const double top_p = sh.how[which].top_p;
  const int bits = sh.bits;
  const uint32_t top_key = sh.top_key;
  const Runs runs(top_key, ordered(bound));
  const double one = static_cast<double>(1ull << bits);
  for (int i = lane; i < held; i += 32) {
    const float x = sh.held[warp][i].x;
    const double w = weight(sh.table, sc, x);
    part += w;
    if (top_p < 1.0) atomicAdd(&sh.hist[runs.of(x)], static_cast<unsigned long long>(w * one));
  }
  double mass = share_sums(sh, p, turn, sum + part, over, &part, top_p < 1.0);
  bool listed = part == part, kept = false;  // (NaN: some warp had no room)
  auto sum_of = [&](int, float4 x) { return weights_sum(sh.table, sc, small, x); };
  if (!listed) mass = row_mass(sh, p, s, turn, sum_of);
  if (top_p < 1.0) {
    kept = listed && part > top_p * mass * (1.0 + 1e-9);  // the border lies among the candidates
    if (kept) {
      const Nucleus k = held_nucleus(sh, p, sc, runs, mass, top_p, bits, turn);
      sc.cut = k.cut, turn = k.turn, mass = k.mass;
      if (mass < 0.0) mass = held_mass(sh, p, turn, [&](const Candidate& c) { return weight(sh.table, sc, c.x); });
    } else {
      listed = false;
      const float floor_x = least_of(unordered(top_key), mass, top_p, sh.how[which].temperature, sh.V);
      const Nucleus k = row_nucleus(sh, p, s, sc, Runs(top_key, floor_x == floor_x ? min(ordered(fmaxf(floor_x, sc.cut)), top_key) : ordered(sc.cut)), mass, top_p, bits, turn);
      sc.cut = k.cut, turn = k.turn;
      mass = row_mass(sh, p, s, turn, sum_of);
    }
  }
  if (threadIdx.x == 0) {
    Row& r = sh.row[which];
    r.s = sc, r.mass = mass, r.bound = bound;
    r.good = true, r.listed = listed, r.held = kept;
  }
  __syncthreads();
  return turn;
}

// A part's sum may come from entries that weigh nothing in double: masked ones count as 2^-100 in fp32, and what the draft leaves is rounded otherwise there.  Then the token is this: the
// first from `from` on, around the row's end, with any mass in p or, beside a draft's row, in max(pf wp - qf wq, 0).  -1: there is none.  A warp; out of line, since it is hardly ever needed.
__device__ __noinline__ int next_with_mass(const Shared& sh, const float* logits, const float* draft, const double pf, const double qf, const int V, const int from) {
  const int lane = threadIdx.x % 32;
  const Source target(logits, 0), other(draft != nullptr ? draft : logits, 0);
  auto mass = [&](float y, float z) {
    const double w = weight(sh.table, sh.row[1].s, y);
    return draft == nullptr ? w : __dsub_rn(__dmul_rn(pf, w), __dmul_rn(qf, weight(sh.table, sh.row[0].s, z)));
  };
#pragma unroll 1
  for (int round = 0; round < 2; ++round)
#pragma unroll 1
    for (int i = round == 0 ? from : 0, to = round == 0 ? V : from; i < to; i += kRun) {
      const float4 y = target.four(i + 4 * lane, to), z = other.four(i + 4 * lane, to);
      const int is = (mass(y.x, z.x) > 0.0 ? 1 : 0) | (mass(y.y, z.y) > 0.0 ? 2 : 0) | (mass(y.z, z.z) > 0.0 ? 4 : 0) | (mass(y.w, z.w) > 0.0 ? 8 : 0);
      const uint32_t some = __ballot_sync(0xffffffffu, is != 0);
      if (some) return __shfl_sync(0xffffffffu, i + 4 * lane + __ffs(is) - 1, __ffs(some) - 1);
    }
  return -1;
}

PG_DEVINL float unit_number(float u) { return fminf(fmaxf(u, 0.0f), 1.0f - 0x1p-24f); }  // (a NaN is 0)

struct Family {  // parents and tokens of an entry; those of the 32 rows behind v lie in the lanes
  const int *parents, *tokens;
  int v, n, up, token;
  PG_DEVINL void look() {
    const int j = v + 1 + threadIdx.x % 32;
    up = j < n ? parents[j] : -1;
    token = j < n ? tokens[j] : 0;
  }
  // first row from `i` on (i > v) whose parent is v, n where there is none; x: its token.  Whole warps.
  PG_DEVINL int child(int i, int& x) const {
    for (int i0 = i; i0 < n;) {
      const int base = i0 <= v + 32 ? v + 1 : i0, j = base + threadIdx.x % 32;
      const bool near = base == v + 1;
      const uint32_t is = __ballot_sync(0xffffffffu, j >= i0 && j < n && (near ? up : parents[j]) == v);
      if (is) {
        const int l = __ffs(is) - 1;
        x = near ? __shfl_sync(0xffffffffu, token, l) : tokens[base + l];
        return base + l;
      }
      i0 = base + 32;
    }
    return n;
  }
  PG_DEVINL int with(int t) const {  // first child that carries t, or n
    int x = 0;
    for (int i = child(v + 1, x); i < n; i = child(i + 1, x))
      if (x == t) return i;
    return n;
  }
};

// Whether nothing that is decided yet leads past row v: all the way up, since rows that nothing leads to are judged as well while that is not known.  A warp; the parents and outcomes
// of the 32 rows in front of v lie in its lanes.
PG_DEVINL bool may_be_reached(const int* parents, const int* outcome, int v) {
  const int j = v - 1 - static_cast<int>(threadIdx.x % 32);
  const int ups = j >= 0 ? parents[j] : -1, saids = j >= 0 ? load_relaxed(outcome + j) : 0;
  int row = v, up = parents[v];
  for (;;) {
    if (up < 0 || up >= row) return false;
    const int l = v - 1 - up;
    const int said = l < 32 ? __shfl_sync(0xffffffffu, saids, l) : load_relaxed(outcome + up);
    if (said != 0 && said != row) return false;
    if (up == 0) return true;
    row = up;
    up = l < 32 ? __shfl_sync(0xffffffffu, ups, l) : parents[up];
  }
}

__global__ void __launch_bounds__(kThreads, kPerSm) verify_kernel(const PgVerify a, int share, int bits) {
  extern __shared__ __align__(16) char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x;
  int finisher = 0;  // the CTA that knows the outcome
  pg::cluster_arrive();
  const int v = item / a.entries, e = item % a.entries;  // the entries' first rows come first
  const int n = a.n[e];
  const long long row0 = a.row0[e], row = row0 + v;
  bool live = v < n && row0 >= 0 && row0 + n <= a.rows;
  int* outcome = a.outcome + row0;
  Family fam;
  fam.parents = a.parents + row0, fam.tokens = a.tokens + row0, fam.v = v, fam.n = n;
  pg::cluster_wait();  // (the others run: their shared memory is there)
  if (live && v > 0) {
    if (rank == 0 && tid < 32) {  // one look for all: what the parent decides may come in between
      const bool reached = may_be_reached(fam.parents, outcome, v);
      if (tid < static_cast<int>(ranks)) put32(&sh.state, tid, reached);
    }
    pg::cluster_sync_all();
    live = sh.state != 0;
    if (!live && rank == 0 && tid == 0) outcome[v] = kDead;
  }
  if (live) {
    Part p;
    p.rank = rank, p.ranks = ranks;
    p.lo = min(rank * share, a.V);
    p.n = min(share, a.V - p.lo);
    p.seg = (share + kWarps * kRun - 1) / (kWarps * kRun) * kRun;
    int turn = 0, to = 0, x = 0;  // to: the child, or -2 - token where the walk ends
    const float *logits = a.logits + row * a.ld, *draft = a.draft + row * a.draft_ld;
    const Source target(logits, p.lo);
    fam.look();
    if (tid >= kTable && tid < kTable + 2) {
      const bool draft = tid == kTable;
      const double temperature = draft ? a.draft_temperature : a.temperature, top_p = draft ? a.draft_top_p : a.top_p;
      if (!draft || a.draft != nullptr) sh.how[tid - kTable] = How{temperature, top_p, kLog2e / temperature, top_p < 1.0 ? log(16.0 * (1.0 - top_p) / a.V) : 0.0};
      sh.V = a.V, sh.bits = bits;
    }
    if (tid < kTable) sh.table[tid] = exp2(static_cast<double>(tid) / kTable);  // (read behind the first barriers of row_top)
    const float u = unit_number(a.uniforms[2 * row + 1]);
    const Source other(draft, p.lo);
    int child = a.draft != nullptr ? fam.child(v + 1, x) : n;
    bool good = true;
#pragma unroll 1
    for (int which = child < n ? 0 : 1; which < 2 && good; ++which) {
      turn = distribution(sh, p, which == 0 ? other : target, which, turn);
      good = sh.row[which].good;
    }
    if (!good) {
      to = -1;
    } else {
      const Row &t = sh.row[1], &q = sh.row[child < n ? 0 : 1];
      const Scale ts = t.s, qs = q.s;
      double mass = t.mass, c = 0.0, left = 1.0, pf = 0.0, qf = 0.0;
      // max(p - c q, 0); both products rounded alike, so that equal ones leave nothing
      auto rest_of = [&](double wt, double wq) { return fmax(__dsub_rn(__dmul_rn(pf, wt), __dmul_rn(qf, wq)), 0.0); };
      auto rest4 = [&](int i, float4 y, double (&w)[4]) {
        const float4 z = other.four(i, p.n);
        w[0] = rest_of(weight(sh.table, ts, y.x), weight(sh.table, qs, z.x)), w[1] = rest_of(weight(sh.table, ts, y.y), weight(sh.table, qs, z.y));
        w[2] = rest_of(weight(sh.table, ts, y.z), weight(sh.table, qs, z.z)), w[3] = rest_of(weight(sh.table, ts, y.w), weight(sh.table, qs, z.w));
      };
      const float bound = t.bound;
      const bool quick = child < n && t.listed && qs.fine > -INFINITY;
      const Pairs small_t(ts), small_q(qs);
      float pf0 = 0.0f, pf1 = 0.0f, qf0 = 0.0f, qf1 = 0.0f;  // the factors in two parts
      auto rest_sum = [&](int i, float4 y) {
        if (!quick) {
          double w[4];
          rest4(i, y, w);
          return (w[0] + w[1]) + (w[2] + w[3]);
        }
        const float4 z = other.four(i, p.n);  // (what is not small is added from the candidates; what p has not is not there, whatever q has)
        const float2 t0 = small_t(y.x, y.y), t1 = small_t(y.z, y.w), q0 = small_q(z.x, z.y), q1 = small_q(z.z, z.w);
        const float ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w}, wt[4] = {t0.x, t0.y, t1.x, t1.y}, wq[4] = {q0.x, q0.y, q1.x, q1.y};
        float w = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float b = zs[k] >= qs.cut ? wq[k] : 0.0f;
          const float left_over = __fsub_rn(fmaf(wt[k], pf0, __fmul_rn(wt[k], pf1)), fmaf(b, qf0, __fmul_rn(b, qf1)));
          w += ys[k] < bound && ys[k] >= ts.cut ? fmaxf(left_over, 0.0f) : 0.0f;
        }
        return static_cast<double>(w);
      };
      auto rest1 = [&](const Candidate& k) { return k.x >= ts.cut ? rest_of(weight(sh.table, ts, k.x), weight(sh.table, qs, other.x[k.at])) : 0.0; };
      auto rest_mass = [&]() {
        double sum = 0.0;
        each4(p, target, [&](int i, float4 y) { sum += rest_sum(i, y); });
        if (quick)
          for (int i = tid % 32; i < sh.held_count[tid / 32]; i += 32) sum += rest1(sh.held[tid / 32][i]);
        return share_sums(sh, p, turn, sum);
      };
      while (child < n) {
        if (x >= 0 && x < a.V) {  // (what is no token was drawn from nothing: it takes nothing away)
          const double pt = weight(sh.table, ts, logits[x]) / mass, qt = weight(sh.table, qs, draft[x]) / q.mass;
          const bool stays = static_cast<double>(unit_number(a.uniforms[2 * (row0 + child)])) * qt * left < __dsub_rn(pt, __dmul_rn(c, qt));
          if (stays) break;
          c += left;
          pf = 1.0 / mass, qf = c / q.mass;
          pf0 = static_cast<float>(pf), pf1 = static_cast<float>(pf - pf0), qf0 = static_cast<float>(qf), qf1 = static_cast<float>(qf - qf0);
          left = t.held ? held_mass(sh, p, turn, rest1) : rest_mass();
          if (!(left > 0.0)) break;
        }
        child = fam.child(child + 1, x);
      }
      if (child < n && left > 0.0) {
        to = child;
      } else {
        int token;
        auto behind = [&](int from) { return next_with_mass(sh, logits, c > 0.0 && left > 0.0 ? draft : nullptr, pf, qf, a.V, from); };
        if (c > 0.0 && left > 0.0) {
          token = t.held ? held_draw(sh, p, turn, left, u, finisher, rest1) : row_draw(sh, p, target, turn, left, u, finisher, rest4, behind);
        } else {
          auto one = [&](const Candidate& k) { return weight(sh.table, ts, k.x); };
          auto four = [&](int, float4 y, double (&w)[4]) {
            w[0] = weight(sh.table, ts, y.x), w[1] = weight(sh.table, ts, y.y), w[2] = weight(sh.table, ts, y.z), w[3] = weight(sh.table, ts, y.w);
          };
          if (c > 0.0) mass = t.held ? held_mass(sh, p, turn, one) : row_mass(sh, p, target, turn, [&](int, float4 y) { return weights_sum(sh.table, ts, small_t, y); });
          token = t.held ? held_draw(sh, p, turn, mass, u, finisher, one) : row_draw(sh, p, target, turn, mass, u, finisher, four, behind);
        }
        const int next = a.draft == nullptr && rank == finisher ? fam.with(token) : n;
        to = next < n ? next : -2 - token;
      }
    }
    if (rank == finisher && tid == 0) outcome[v] = to;
  }
  // the last cluster walks
  if (rank == finisher) {
    if (tid == 0) {
      __threadfence();
      sh.last = atomicAdd(a.outcome + a.rows, 1) == static_cast<int>(gridDim.x / ranks) - 1;
      __threadfence();
    }
    __syncthreads();
    if (sh.last) {
      const bool fits = a.rows <= static_cast<int>(sizeof(sh.held) / sizeof(int));  // (the candidates are not needed any more)
      int* held = reinterpret_cast<int*>(sh.held);
      if (fits)
        for (int i = tid; i < a.rows; i += kThreads) held[i] = load_relaxed(a.outcome + i);
      __syncthreads();
      for (int w = tid; w < a.entries; w += kThreads) {
        const int m = a.n[w], first = a.row0[w];
        int* path = a.path + w * a.path_ld;
        int at = 0, kept = 0, next = -1;
        if (m > 0 && m <= a.path_ld && first >= 0 && first + m <= a.rows) {
          for (;;) {
            path[kept++] = at;
            const int said = fits ? held[first + at] : load_relaxed(a.outcome + first + at);
            if (said <= at || said >= m) {
              next = said < 0 && said != kDead ? -2 - said : -1;
              break;
            }
            at = said;
          }
        }
        a.kept[w] = kept;
        a.next[w] = next;
        for (int i = kept; i < a.path_ld; ++i) path[i] = -1;
      }
    }
  }
  // (what the CTAs hand one another lies in front of a barrier that all have passed)
}

// Greedy walks: one pass over all rows of the step, cut into pieces that the CTAs share evenly; (largest entry, lowest place) of a row meet in one word each.  The CTA that is through
// last walks, a warp an entry: 32 rows of it in the lanes.
constexpr int kPiece = 4 * kThreads;  // (two CTAs an SM, four loads a thread: 27 us; three or four, eight loads: 27, 29, 29)
__global__ void __launch_bounds__(kThreads, kPerSm) greedy_kernel(const PgVerify a, int pieces, long long all) {
  __shared__ int last;
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(a.outcome);
  const int tid = threadIdx.x, lane = tid % 32;
  const long long end = all * (blockIdx.x + 1) / gridDim.x;
  for (long long u = all * blockIdx.x / gridDim.x; u < end;) {
    const long long row = u / pieces;
    const int p0 = static_cast<int>(u % pieces), p1 = static_cast<int>(min(static_cast<long long>(pieces), p0 + (end - u)));
    const int hi = static_cast<int>(min(static_cast<long long>(a.V), static_cast<long long>(p1) * kPiece));
    const Source s(a.logits + row * a.ld, 0);
    float best = -INFINITY;
    int i = p0 * kPiece + 4 * tid, run = i;  // run: the first four that hold it
    auto take = [&](int at, float4 x) {
      const float four = max_nan(max_nan(x.x, x.y), x.z, x.w);
      if (four > best) run = at;
      best = max_nan(best, four);  // (where that is a NaN the place does not matter)
    };
    if (s.aligned)
      for (; i + 3LL * kPiece + 4 <= hi; i += 4 * kPiece) {
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __ldg(reinterpret_cast<const float4*>(s.x + i + k * kPiece));
#pragma unroll
        for (int k = 0; k < 4; ++k) take(i + k * kPiece, x[k]);
      }
    for (; i < hi; i += kPiece) take(i, s.four(i, hi));
    unsigned long long key = 0;
    if (run < hi) {
      const float4 x = s.four(run, hi);
      const int at = run + (x.x == best ? 0 : x.y == best ? 1 : x.z == best ? 2 : 3);
      key = static_cast<unsigned long long>(ordered(best)) << 32 | static_cast<uint32_t>(~at);
    }
    key = warp_max(key);
    if (lane == 0) atomicMax(keys + row, key);
    u += p1 - p0;
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    last = atomicAdd(a.outcome + 2 * static_cast<long long>(a.rows), 1) == static_cast<int>(gridDim.x) - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  for (int e = tid / 32; e < a.entries; e += kWarps) {
    const int m = a.n[e], row0 = a.row0[e];
    int* path = a.path + e * a.path_ld;
    int kept = 0, next = -1;
    if (m > 0 && m <= a.path_ld && row0 >= 0 && row0 + static_cast<long long>(m) <= a.rows) {
      int base = 0, up = 0, token = 0, said = -1;  // rows base .. base + 31: what they follow, carry and say
      auto look = [&](int b) {
        base = b;
        const int j = b + lane;
        if (j >= m) return;
        const unsigned long long key = __ldcg(keys + row0 + j);
        up = a.parents[row0 + j], token = a.tokens[row0 + j];
        said = is_distribution(static_cast<uint32_t>(key >> 32)) ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
      };
      look(0);
      for (int at = 0;;) {
        if (lane == 0) path[kept] = at;
        ++kept;
        const int t = __shfl_sync(0xffffffffu, said, at - base);
        uint32_t is = 0;
        if (t >= 0)
          for (int b = (at + 1) / 32 * 32; b < m && is == 0; b += 32) {
            if (b != base) look(b);
            const int j = b + lane;
            is = __ballot_sync(0xffffffffu, j > at && j < m && up == at && token == t);
          }
        if (is == 0) {
          next = t;
          break;
        }
        at = base + __ffs(is) - 1;
      }
    }
    if (lane == 0) a.kept[e] = kept, a.next[e] = next;
    for (long long i = kept + lane; i < a.path_ld; i += 32) path[i] = -1;
  }
}

}  // namespace

extern "C" int pg_verify_drafts(const PgVerify* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgVerify& a = *args;
  auto sound = [](double temperature, double top_p) { return temperature > 0.0 && temperature < INFINITY && kLog2e / temperature < 1e30 && top_p >= 0.0 && top_p <= 1.0; };
  if (a.logits == nullptr || a.tokens == nullptr || a.parents == nullptr || a.row0 == nullptr || a.n == nullptr || a.path == nullptr || a.kept == nullptr || a.next == nullptr ||
      a.outcome == nullptr || (reinterpret_cast<uintptr_t>(a.outcome) & 7) || a.entries <= 0 || a.rows <= 0 || a.max_n <= 0 || a.V <= 0 || a.ld < a.V || a.path_ld < a.max_n || (a.draft != nullptr && (a.draft_ld < a.V || a.uniforms == nullptr)) ||
      !sound(a.temperature, a.top_p) || (a.draft != nullptr && !sound(a.draft_temperature, a.draft_top_p)) || a.V > 0x7fffff00 / 2)
    return PG_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  pg_count_launch(1);
  if (a.uniforms == nullptr) {
    const int pieces = (a.V + kPiece - 1) / kPiece;
    const long long all = static_cast<long long>(a.rows) * pieces, most = static_cast<long long>(kPerSm) * pg::num_sms();
    if (cudaMemsetAsync(a.outcome, 0, sizeof(int) * (2 * static_cast<size_t>(a.rows) + 1), st) != cudaSuccess) return PG_ERR_CUDA;
    greedy_kernel<<<static_cast<unsigned>(all < most ? all : most), kThreads, 0, st>>>(a, pieces, all);
    return cudaGetLastError() == cudaSuccess ? PG_OK : PG_ERR_CUDA;
  }
  const long long items = static_cast<long long>(a.entries) * a.max_n;
  // CTAs that share a row: so many that a warp's candidates have room, and more while all of them stay within nine an SM.  (us with fewer, as taken, more: 5 rows of 257216 with 4, 8, 16
  // CTAs 42, 32, 29; 256 beside a draft with 4, 8 257, 308; 624 of 32000 with 1, 2, 4 132, 111, 131.)
  int ranks = 1;
  while (ranks < kRanks && a.V / ranks > 65536) ranks *= 2;
  while (ranks < kRanks && items * ranks * 2 <= 9LL * pg::num_sms() && a.V / (ranks * 2) >= 4 * kThreads) ranks *= 2;
  if (items * ranks > 0x7fffffff) return PG_ERR_ARG;
  const int share = ((a.V + ranks - 1) / ranks + 3) / 4 * 4;
  int bits = 62;
  while ((1ll << (62 - bits)) < a.V) --bits;  // V weights of at most 1 stay below 2^62
  static bool configured[pg::kMaxDevices] = {};
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared)) != cudaSuccess ||
        cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  if (cudaMemsetAsync(a.outcome, 0, sizeof(int) * (static_cast<size_t>(a.rows) + 1), st) != cudaSuccess) return PG_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel, a, share, bits) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
