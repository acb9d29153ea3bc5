// Which drafted tokens stay: rows of target logits (and of the draft's) against given random numbers.
//
// A row decides by itself where the walk goes on from it (the header has the rules), so all rows are judged at once, a cluster of CTAs a row, and the walks are
// pointer chases at the end, made by the last cluster.  Rows lie depth first in their entries and clusters are started in the order of the rows' places in their
// entries: one that finds its parent decided for another child has nothing to do.
//
// After rejections the rest is r_j = (p - c_j q)+ / S_j: from r_j q is taken again, (p - c_j q)+ - S_j q = p - (c_j + S_j) q where that is positive, so c and S are
// two numbers and a rejection is one pass over the row, whatever came before it.
//
// The results are whole numbers that hang on running sums: a draw is wrong once a sum is off by the distance of u from a token's border.  Weights are therefore
// e^((x - m) / T) in double, 2^(j / 64) from a table times a polynomial of degree 4 (error below 1e-13), nine operations of the double pipe, half of fp32's rate.
//
// The nucleus is a threshold on the logit: the entries above which at most top_p Z lies.  Entries below (1 - top_p) Z / V cannot belong to it.  The others are
// counted by mass into 1024 runs of the ordered bit patterns, in fixed point (sums do not hang on their order), and the run that holds the border is divided
// again until a run is one pattern: at most three rounds of one cluster barrier, and few entries take part.
//
// A CTA keeps its share of the row in shared memory: one read of global memory, whatever follows.
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kRanks = 16, kBins = 1024, kCoarse = kBins / 32, kTable = 64;
constexpr int kShare = 16384;      // entries of a row that a CTA keeps where that many CTAs do (64 KB: three CTAs an SM)
constexpr int kMostShare = 49152;  // and at most (192 KB)
constexpr int kDead = -2147483647 - 1;
constexpr double kLog2e = 1.4426950408889634;

struct __align__(16) Shared {
  double table[kTable];                    // 2^(j / 64)
  double warp[kWarps];
  double all[2][kRanks];                   // one double of every CTA, by turns
  unsigned long long key[2][kRanks];
  unsigned long long hist[2][kBins];       // mass of runs of bit patterns, by turns
  unsigned long long coarse[2][kCoarse];
  unsigned long long gather[kRanks][32];
  unsigned long long found_base;
  int found, pick, state, last;
};

static_assert(sizeof(Shared) % 16 == 0, "a share of a row starts on a 16-byte boundary");

PG_DEVINL uint32_t ordered(float x) {  // larger numbers have larger ones; both zeros alike, NaN above all
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
PG_DEVINL float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }

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

struct Scale {
  double m, a;  // maximum, log2(e) / T
};
// e^((x - m) / T) for x <= m (the difference of two floats first: it stays right for the smallest temperatures)
PG_DEVINL double weight(const double* table, Scale s, float x) {
  const double t = (static_cast<double>(x) - s.m) * s.a;
  if (!(t > -1000.0)) return 0.0;  // (-inf too)
  constexpr double kRound = 6755399441055744.0 / kTable;  // 1.5 2^52 / 64: its last place is 1 / 64
  const double rounded = t + kRound, f = t - (rounded - kRound);  // |f| <= 1 / 128
  const int k = __double2loint(rounded);
  constexpr double c1 = 0.6931471805599453, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c1 * c1 * c1 * c1 / 24;
  const double p = fma(f, fma(f, fma(f, fma(f, c4, c3), c2), c1), 1.0) * table[k & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));
}

struct Part {  // a CTA's share of a row: entries lo .. lo + n of it in xs; warp w has seg from w seg on
  float* xs;
  int lo, n, seg, rank, ranks;
};

PG_DEVINL void load_share(const Part& p, const float* row) {
  const float* src = row + p.lo;
  const uint32_t dst = pg::smem_u32(p.xs);
  const int whole = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? p.n / 4 * 4 : 0;
  for (int i = 4 * threadIdx.x; i < whole; i += 4 * kThreads) pg::cp_async16(dst + 4 * i, src + i, true);
  for (int i = whole + threadIdx.x; i < p.n; i += kThreads)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * i), "l"(src + i) : "memory");
  pg::cp_async_commit();
}

// (largest entry, lowest place) of the row as one number, known to all CTAs
PG_DEVINL unsigned long long row_top(Shared& sh, const Part& p, int& turn) {
  uint32_t best = 0;
  int at = 0;
  for (int i = threadIdx.x; i < p.n; i += kThreads) {
    const uint32_t k = ordered(p.xs[i]);
    if (k > best) best = k, at = i;
  }
  unsigned long long key = p.n > 0 ? static_cast<unsigned long long>(best) << 32 | static_cast<uint32_t>(~(p.lo + at)) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  unsigned long long* mine = reinterpret_cast<unsigned long long*>(sh.warp);
  if (threadIdx.x % 32 == 0) mine[threadIdx.x / 32] = key;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < p.ranks) {
    for (int w = 0; w < kWarps; ++w) key = mine[w] > key ? mine[w] : key;
    put64(&sh.key[turn][p.rank], threadIdx.x, key);
  }
  pg::cluster_sync_all();
  unsigned long long top = 0;
  for (int r = 0; r < p.ranks; ++r) top = sh.key[turn][r] > top ? sh.key[turn][r] : top;
  turn ^= 1;
  return top;
}
PG_DEVINL bool is_distribution(unsigned long long top) {
  const uint32_t k = static_cast<uint32_t>(top >> 32);
  return k > ordered(-INFINITY) && k < ordered(INFINITY);
}

// Sums of f over the row: the warps' in sh.warp, the CTAs' in sh.all[turn] (until the next but one), the whole as the result.  The order of additions is fixed.
template <typename F>
PG_DEVINL double row_mass(Shared& sh, const Part& p, int& turn, F f) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int lo = min(warp * p.seg, p.n), hi = min(lo + p.seg, p.n);
  double sum = 0.0;
  for (int i = lo + lane; i < hi; i += 32) sum += f(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();  // (the sums before have been read)
  if (lane == 0) sh.warp[warp] = sum;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < p.ranks) {
    double all = 0.0;
    for (int w = 0; w < kWarps; ++w) all += sh.warp[w];
    put64(&sh.all[turn][p.rank], threadIdx.x, __double_as_longlong(all));
  }
  pg::cluster_sync_all();
  double total = 0.0;
  for (int r = 0; r < p.ranks; ++r) total += sh.all[turn][r];
  turn ^= 1;
  return total;
}

// The token at u times the whole of f, whose sums row_mass has left (`turn` behind it): the first place whose running sum is above that.  Known to all CTAs.
template <typename F>
PG_DEVINL int row_draw(Shared& sh, const Part& p, int turn, double total, float u, F f) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  double rest = static_cast<double>(u) * total, run = 0.0;
  int owner = -1, behind = -1;
  for (int r = 0; r < p.ranks; ++r) {  // (where rounding leaves no border behind u: the last one with any mass)
    const double m = sh.all[turn ^ 1][r];
    if (m > 0.0) behind = r;
    if (owner < 0 && run + m > rest) owner = r;
    if (owner < 0) run += m;
  }
  if (owner < 0) owner = behind;
  if (owner == p.rank) {
    int mine = -1, other = -1;
    for (int w = 0; w < kWarps; ++w) {
      const double m = sh.warp[w];
      if (m > 0.0) other = w;
      if (mine < 0 && run + m > rest) mine = w;
      if (mine < 0) run += m;
    }
    if (mine < 0) mine = other;
    if (warp == mine) {
      const int lo = min(warp * p.seg, p.n), hi = min(lo + p.seg, p.n);
      int place = -1, last = -1;
      for (int i0 = lo; i0 < hi && place < 0; i0 += 32) {
        const double w = i0 + lane < hi ? f(i0 + lane) : 0.0;
        double incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double before = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += before;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, w > 0.0), past = __ballot_sync(0xffffffffu, run + incl > rest) & some;
        if (some) last = i0 + 31 - __clz(some);
        if (past) place = i0 + __ffs(past) - 1;
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (place < 0) place = last;
      if (lane < p.ranks) put32(&sh.pick, lane, p.lo + place);
    }
  }
  pg::cluster_sync_all();
  return sh.pick;
}

// Least ordered pattern of the nucleus.  z: the whole mass, `bits`: of the fixed point.
PG_DEVINL uint32_t nucleus(Shared& sh, const Part& p, Scale s, uint32_t top, double z, double top_p, double temperature, int V, int bits, int& turn) {
  const double least = static_cast<double>(unordered(top)) + log((1.0 - top_p) * z / V) * temperature;
  float floor_x = __double2float_rd(least);
  floor_x -= fabsf(floor_x) * 3e-7f + 1e-37f;
  uint32_t hi = top, lo = floor_x == floor_x ? min(ordered(floor_x), top) : 0u;
  const double one = static_cast<double>(1ull << bits), border = top_p * z * one;
  unsigned long long base = 0;  // mass above hi
  for (;;) {
    const uint32_t range = hi - lo;
    const int shift = range < kBins ? 0 : 32 - __clz(range) - 10;
    unsigned long long* hist = sh.hist[turn];
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.n; i += kThreads) {
      const float x = p.xs[i];
      const uint32_t k = ordered(x);
      if (k >= lo && k <= hi) atomicAdd(&hist[(hi - k) >> shift], static_cast<unsigned long long>(weight(sh.table, s, x) * one));
    }
    __syncthreads();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int c = warp; c < kCoarse; c += kWarps) {
      unsigned long long v = hist[c * 32 + lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) sh.coarse[turn][c] = v;
    }
    pg::cluster_sync_all();
    int bin = 0;
#pragma unroll
    for (int step = 0; step < 2; ++step) {  // 32 runs of 32, then one of them
      const unsigned long long* from = step == 0 ? sh.coarse[turn] : hist + bin * 32;
      if (warp < p.ranks) sh.gather[warp][lane] = get64(from + lane, warp);
      __syncthreads();
      if (warp == 0) {
        unsigned long long v = 0;
        for (int r = 0; r < p.ranks; ++r) v += sh.gather[r][lane];
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
    const int found = sh.found;
    turn ^= 1;
    if (found < 0) return lo;
    hi -= static_cast<uint32_t>(bin) << shift;
    if (shift == 0) return hi;
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
  }
}

struct Row {  // a row's distribution: weight / mass where the pattern is `least` or above
  Scale s;
  uint32_t least;
  double mass;
};

PG_DEVINL double kept_weight(const double* table, const Row& r, float x) { return ordered(x) >= r.least ? weight(table, r.s, x) : 0.0; }

// max(p - c q, 0) of one entry; both products rounded alike, so that equal ones leave nothing
PG_DEVINL double rest_weight(const double* table, const Row& t, double pf, float x, const Row& q, double qf, float y) {
  return fmax(__dsub_rn(__dmul_rn(pf, kept_weight(table, t, x)), __dmul_rn(qf, kept_weight(table, q, y))), 0.0);
}

// The distribution of the row in xs; its sums of the kept weights are left behind for a draw.
PG_DEVINL bool distribution(Shared& sh, const Part& p, double temperature, double top_p, int V, int bits, Row& r, int& turn) {
  const unsigned long long top = row_top(sh, p, turn);
  if (!is_distribution(top)) return false;
  r.s.a = kLog2e / temperature;
  r.s.m = unordered(static_cast<uint32_t>(top >> 32));
  r.least = 0;
  r.mass = row_mass(sh, p, turn, [&](int i) { return weight(sh.table, r.s, p.xs[i]); });
  if (top_p < 1.0) {
    r.least = nucleus(sh, p, r.s, static_cast<uint32_t>(top >> 32), r.mass, top_p, temperature, V, bits, turn);
    r.mass = row_mass(sh, p, turn, [&](int i) { return kept_weight(sh.table, r, p.xs[i]); });
  }
  return true;
}

PG_DEVINL float unit_number(float u) { return fminf(fmaxf(u, 0.0f), 1.0f - 0x1p-24f); }  // (a NaN is 0)

// first row behind `v` (exclusive) from `i` on whose parent is v; n where there is none.  Whole warps.
PG_DEVINL int next_child(const int* parents, int v, int i, int n) {
  for (int i0 = i; i0 < n; i0 += 32) {
    const int j = i0 + threadIdx.x % 32;
    const uint32_t is = __ballot_sync(0xffffffffu, j < n && parents[j] == v);
    if (is) return i0 + __ffs(is) - 1;
  }
  return n;
}

// first child of v that carries `token`, or n
PG_DEVINL int child_with(const int* parents, const int* tokens, int v, int n, int token) {
  for (int i = next_child(parents, v, v + 1, n); i < n; i = next_child(parents, v, i + 1, n))
    if (tokens[i] == token) return i;
  return n;
}

__global__ void __launch_bounds__(kThreads) verify_kernel(const PgVerify a, int share, int bits) {
  extern __shared__ __align__(16) char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  float* xs = reinterpret_cast<float*>(raw + sizeof(Shared));
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int rank = pg::cluster_ctarank(), item = blockIdx.x / ranks, tid = threadIdx.x;
  if (tid < kTable) sh.table[tid] = exp2(static_cast<double>(tid) / kTable);
  const int v = item / a.entries, e = item % a.entries;  // the entries' first rows come first
  const int n = a.n[e];
  const long long row0 = a.row0[e], row = row0 + v;
  bool live = v < n && row0 >= 0 && row0 + n <= a.rows;
  int* outcome = a.outcome + row0;
  const int* parents = a.parents + row0;
  const int* tokens = a.tokens + row0;
  if (live && v > 0) {
    if (rank == 0 && tid < 32) {  // one look for all: what the parent decides may come in between
      int said = 0;
      if (tid == 0) {
        const int up = parents[v];
        said = up >= 0 && up < v ? load_relaxed(outcome + up) : kDead;
      }
      said = __shfl_sync(0xffffffffu, said, 0);
      if (tid < static_cast<int>(ranks)) put32(&sh.state, tid, said == 0 || said == v);
    }
    pg::cluster_sync_all();
    live = sh.state != 0;
    if (!live && rank == 0 && tid == 0) outcome[v] = kDead;
  }
  if (live) {
    Part p;
    p.xs = xs, p.rank = rank, p.ranks = ranks;
    p.lo = min(rank * share, a.V);
    p.n = min(share, a.V - p.lo);
    p.seg = (share + kThreads - 1) / kThreads * 32;
    int turn = 0, to = 0;  // to: the child, or -2 - token where the walk ends
    const float* logits = a.logits + row * a.ld;
    auto wait = [&]() {
      pg::cp_async_wait<0>();
      __syncthreads();
    };
    if (a.uniforms == nullptr) {
      load_share(p, logits);
      wait();
      const unsigned long long top = row_top(sh, p, turn);
      const int token = is_distribution(top) ? static_cast<int>(~static_cast<uint32_t>(top)) : -1;
      const int child = token >= 0 ? child_with(parents, tokens, v, n, token) : n;
      to = child < n ? child : -2 - token;
    } else {
      const float u = unit_number(a.uniforms[2 * row + 1]);
      int child = a.draft != nullptr ? next_child(parents, v, v + 1, n) : n;
      Row t, q;
      bool good = true;
      const float* draft = a.draft + row * a.draft_ld;
      if (child < n) {
        load_share(p, draft);
        wait();
        good = distribution(sh, p, a.draft_temperature, a.draft_top_p, a.V, bits, q, turn);
        __syncthreads();  // (xs has been read)
      }
      if (good) {
        load_share(p, logits);
        wait();
        good = distribution(sh, p, a.temperature, a.top_p, a.V, bits, t, turn);
      }
      if (!good) {
        to = -1;
      } else {
        double c = 0.0, left = 1.0;
        while (child < n) {
          const int x = tokens[child];
          if (x >= 0 && x < a.V) {  // (what is no token was drawn from nothing: it takes nothing away)
            const double pt = kept_weight(sh.table, t, logits[x]) / t.mass, qt = kept_weight(sh.table, q, draft[x]) / q.mass;
            const bool stays = static_cast<double>(unit_number(a.uniforms[2 * (row0 + child)])) * qt * left < __dsub_rn(pt, __dmul_rn(c, qt));
            if (stays) break;
            c += left;
            const double pf = 1.0 / t.mass, qf = c / q.mass;
            left = row_mass(sh, p, turn, [&](int i) { return rest_weight(sh.table, t, pf, xs[i], q, qf, draft[p.lo + i]); });
            if (!(left > 0.0)) break;
          }
          child = next_child(parents, v, child + 1, n);
        }
        if (child < n && left > 0.0) {
          to = child;
        } else {
          int token;
          if (c > 0.0 && left > 0.0) {
            const double pf = 1.0 / t.mass, qf = c / q.mass;
            token = row_draw(sh, p, turn, left, u, [&](int i) { return rest_weight(sh.table, t, pf, xs[i], q, qf, draft[p.lo + i]); });
          } else {
            auto f = [&](int i) { return kept_weight(sh.table, t, xs[i]); };
            if (c > 0.0) t.mass = row_mass(sh, p, turn, f);
            token = row_draw(sh, p, turn, t.mass, u, f);
          }
          child = a.draft == nullptr ? child_with(parents, tokens, v, n, token) : n;
          to = child < n ? child : -2 - token;
        }
      }
    }
    if (rank == 0 && tid == 0) outcome[v] = to;
  }
  // the last cluster walks
  if (rank == 0) {
    if (tid == 0) {
      __threadfence();
      sh.last = atomicAdd(a.outcome + a.rows, 1) == static_cast<int>(gridDim.x / ranks) - 1;
      __threadfence();
    }
    __syncthreads();
    if (sh.last) {
      const bool fits = a.rows <= share;
      int* held = reinterpret_cast<int*>(xs);
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
  pg::cluster_sync_all();  // nobody leaves while its memory is read
}

}  // namespace

extern "C" int pg_verify_drafts(const PgVerify* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgVerify& a = *args;
  auto sound = [](double temperature, double top_p) { return temperature > 0.0 && temperature < INFINITY && kLog2e / temperature < 1e30 && top_p >= 0.0 && top_p <= 1.0; };
  if (a.logits == nullptr || a.tokens == nullptr || a.parents == nullptr || a.row0 == nullptr || a.n == nullptr || a.path == nullptr || a.kept == nullptr || a.next == nullptr ||
      a.outcome == nullptr || a.entries <= 0 || a.rows <= 0 || a.max_n <= 0 || a.V <= 0 || a.ld < a.V || a.path_ld < a.max_n || (a.draft != nullptr && (a.draft_ld < a.V || a.uniforms == nullptr)) ||
      !sound(a.temperature, a.top_p) || (a.draft != nullptr && !sound(a.draft_temperature, a.draft_top_p)) || a.V > kRanks * kMostShare)
    return PG_ERR_ARG;
  const long long items = static_cast<long long>(a.entries) * a.max_n;
  int ranks = 1;
  while (ranks < kRanks && (a.V + ranks - 1) / ranks > kShare) ranks *= 2;
  while (ranks < kRanks && items * ranks * 2 <= pg::num_sms() && a.V / (ranks * 2) >= 4 * kThreads) ranks *= 2;  // few rows: more CTAs for each
  if (items * ranks > 0x7fffffff) return PG_ERR_ARG;
  const int share = ((a.V + ranks - 1) / ranks + 3) / 4 * 4;
  int bits = 62;
  while ((1ll << (62 - bits)) < a.V) --bits;  // V weights of at most 1 stay below 2^62
  const size_t smem = sizeof(Shared) + sizeof(float) * share;
  static bool configured[pg::kMaxDevices] = {};
  bool& done = configured[pg::current_device()];
  if (!done) {
    if (cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared) + 4 * kMostShare) != cudaSuccess ||
        cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
      cudaGetLastError();
      return PG_ERR_CUDA;
    }
    done = true;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(a.outcome, 0, sizeof(int) * (static_cast<size_t>(a.rows) + 1), st) != cudaSuccess) return PG_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  pg_count_launch(1);
  return cudaLaunchKernelEx(&cfg, verify_kernel, a, share, bits) == cudaSuccess ? PG_OK : PG_ERR_CUDA;
}
