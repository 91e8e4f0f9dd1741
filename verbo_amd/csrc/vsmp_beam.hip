// One step of beam search (k_beam): a row's log of the sum of exponentials and its largest logits in one pass, then,
// in the group's last part, the best continuations over its rows.
#include <cfloat>

#include "vsmp_beam.hpp"
#include "vsmp_keys.hpp"
#include "vsmp_logits.hpp"
#include "vsmp_rows.hpp"

namespace vsmp {
namespace {

constexpr int kNt = 256;       // threads per workgroup
constexpr int kW = kNt / 64;   // its waves

// ---- lists of 64 in a wave, an entry a lane -------------------------------------------------------------

// The value of the lane D away (lane ^ D).
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0u, v, 0xB1, 0xF, 0xF, false);  // quads: 1 0 3 2
  if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0u, v, 0x4E, 0xF, 0xF, false);  // 2 3 0 1
  if constexpr (D == 4) {  // eight lanes the other way round (^ 7), then each quad (^ 3)
    const uint32_t m = __builtin_amdgcn_update_dpp(0u, v, 0x141, 0xF, 0xF, false);
    return __builtin_amdgcn_update_dpp(0u, m, 0x1B, 0xF, 0xF, false);
  }
  if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xF, 0xF, false);  // rows of 16 turned by 8
  if constexpr (D == 16) {  // the first: the even rows' values in both rows of a pair, the second: the odd rows'
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if constexpr (D == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int D>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v, int lane) {
  return static_cast<uint64_t>(lane_xor<D>(static_cast<uint32_t>(v >> 32), lane)) << 32 | lane_xor<D>(static_cast<uint32_t>(v), lane);
}

// A continuation as two whole numbers that have its order: its score; then its beam (the lowest first), logit and token
// (6, 32 and 20 bits). That of nothing comes after all others.
struct Cand {
  uint64_t s, t;
};
__device__ __forceinline__ bool before(uint32_t a, uint32_t b) { return a > b; }
__device__ __forceinline__ bool before(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) {
  return a.s > b.s || (a.s == b.s && a.t > b.t);
}
template <int D>
__device__ __forceinline__ Cand lane_xor(const Cand& c, int lane) {
  return {lane_xor<D>(c.s, lane), lane_xor<D>(c.t, lane)};
}
__device__ __forceinline__ Cand none() { return {0u, 0u}; }
static_assert(kBeamMax <= 64 && kOpVocab <= 1 << 20, "a continuation's beam and token");

__device__ __forceinline__ uint64_t ord_f64(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double f64_ord(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7FFFFFFFFFFFFFFFull : ~k));
}

// One exchange of a sorting network: with the lane D away, the lane keeps the earlier or the later of the two.
template <int D, class T>
__device__ __forceinline__ void exchange(T& v, int lane, bool earlier) {
  const T o = lane_xor<D>(v, lane);
  if (before(o, v) == earlier) v = o;  // (of equal entries it does not matter which)
}
// Of each run of 2 K lanes that rises and falls, or falls and rises, the order within it: blocks of `block` lanes in turn
// one way and the other.
template <int K, class T>
__device__ __forceinline__ void merge_runs(T& v, int lane, int block, bool last_first) {
  exchange<K>(v, lane, (((lane & block) == 0) == ((lane & K) == 0)) != last_first);
  if constexpr (K > 1) merge_runs<K / 2>(v, lane, block, last_first);
}
// Sorted over the wave: lane 0 first, or with `last_first` lane 63.
template <class T>
__device__ __forceinline__ void sort64(T& v, int lane, bool last_first) {
  merge_runs<1>(v, lane, 2, last_first);
  merge_runs<2>(v, lane, 4, last_first);
  merge_runs<4>(v, lane, 8, last_first);
  merge_runs<8>(v, lane, 16, last_first);
  merge_runs<16>(v, lane, 32, last_first);
  merge_runs<32>(v, lane, 64, last_first);
}
// The first 64 of a sorted list and of one sorted the other way round, sorted.
template <class T>
__device__ __forceinline__ void merge64(T& v, const T& reversed, int lane) {
  if (before(reversed, v)) v = reversed;
  merge_runs<32>(v, lane, 64, false);
}

template <class T>
__device__ __forceinline__ T agent_load(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ void agent_store(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ bool finite(float v) { return __builtin_isfinite(v); }
// How many of the n entries at p come before c, eight at a time; entries up to the next eight are there.
template <class T>
__device__ __forceinline__ int count_before(const T* p, int n, const T& c) {
  int rank = 0;
  for (int i = 0; i < n; i += 8) {
    T o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = p[i + k];
#pragma unroll
    for (int k = 0; k < 8; ++k) rank += i + k < n && before(o[k], c) ? 1 : 0;
  }
  return rank;
}
// How many of the lanes' flags below this one are set.
__device__ __forceinline__ int below(unsigned long long at) {
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(at >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(at), 0u)));
}

// ---- k_beam ----------------------------------------------------------------------------------------------

constexpr int kCands = 256;    // continuations that the last part ranks side by side
constexpr int kWait = 144;     // logits that a wave has collected: 64 that wait, 64 more or 64 in order, a row's last 7

// One part of a row: a step of four 16-byte groups a thread at a time, the next in flight; what a row has beyond whole
// groups, a lane each, in the end. Each wave collects in LDS the logits that reach its bound, below which none can be
// among the part's N largest that are no stop tokens. The bound is at first the N-th largest of the lanes' maxima over the
// first step, stop tokens left out of account: few more logits reach it. It is sharpened to the N-th of what waits as more
// comes, and to the least of the keys that a quarter of N of each wave's logits reach, which the waves tell each other.
// Where 64 wait, the wave sorts them into a list over its lanes, whose N-th is the bound from then on. In the end the
// waves' logits that reach the largest of their bounds are ranked by comparing each with each, a thread each: mostly they
// are few more than N.
//
// The last part of a group ranks its rows' lists by score in the same way: the N-th largest first entry of the lists (of
// those of a wave's threads; several of each list where there are few) is a bound for all entries. Where more entries than
// kCands reach it (many equal ones) each wave merges lists in order instead, and the first wave the waves'.
//
// Many fp32 rows are bound by the logits' read: 64 groups of 8 rows of 128,256 49.4 us (5.3 TB/s; 8 vector instructions a
// logit, the waves wait for memory half of their time). bf16 by vector instructions: 64 of 16 of 151,936 73 us (4.3 TB/s; 13 a
// logit at N = 16, active in a third of each wave's time, with four waves a SIMD; 80 us with each wave's own bound). f16
// of the same size takes 94 us with as many instructions: the waves wait for loads two thirds of their time. A few rows are bound by latencies that follow one another: one
// group of 4 rows of 49,152 fp32 10.4 us, of which the logits' load and sums take about 3, a part's ranks and their way to
// memory 2, the ticket 1, the last part's loads 1, and its sums, bound and ranks 3. Every workgroup runs most of the code
// once; loops stay rolled where they hardly turn, and nothing is divided by what is not a constant. Sorting networks and
// merges by shuffles through LDS, in the place of bounds and ranks, took 24.6 and 80 us.
//
// Groups of few entries (a.alone) are ended by one wave without a barrier: 24 groups of 5 rows of 50,257 f16 14.4 us, 16.0
// with four.
template <class E>
__global__ __launch_bounds__(kNt, 4) void k_beam(BeamArgs a) {
  constexpr int N = 16 / E::kSize, G = 4;
  constexpr int kStep = kNt * N * G;
  union Shared {
    struct {
      uint64_t wait[kW][kWait], list[kW * kWait];
    } part;
    struct {
      Cand cand[kCands];
      Cand end[kBeamMax * kBeamStops];
      unsigned char lists[kNt];
    } group;
    Cand merge[kW][kBeamMax];
  };
  __shared__ Shared sh;
  __shared__ float s_m[kW], s_s[kW];
  __shared__ double s_lse[kBeamMax], s_score[kBeamMax];
  __shared__ uint32_t s_bound[kW], s_share[kW];
  __shared__ int s_wait[kW], s_n, s_lists, s_end, s_ended, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = static_cast<int>(blockIdx.x), group = static_cast<int>(blockIdx.z);
  const int first = group * a.W, row = first + static_cast<int>(blockIdx.y);  // the group's first row, and this one
  const int lo = part * a.L, hi = min(a.V, lo + a.L), whole = hi & ~(N - 1);
  const char* x = static_cast<const char*>(a.x) + row * a.ld * E::kSize;
  const int stop = lane < a.n_stop ? a.stops[lane] : -1;  // a lane each
  // A key that a wave's share of N, a quarter, of its logits reach: the least of the waves' is one that N of the part's reach.
  const int share = (a.N + kW - 1) / kW;
  if (tid < kW) s_share[tid] = 0u;
  if (tid == 0) s_n = 0;
  __syncthreads();

  Lse z{-INFINITY, 0.0f};
  int waiting = 0;               // logits that the wave has collected
  uint64_t best = 0;             // the lane's entry of the wave's list; 0: none
  uint32_t sure = 0;             // a key that N of its logits reach, no stop tokens among them; 0: none known
  if (finite(a.scores[row])) {
    float bound = -FLT_MAX;
    const int skip = __popcll(__ballot(stop >= lo && stop < hi));  // stop tokens in this part
    Raw<E, N> r[G];
    auto load = [&](int e0) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int e = e0 + N * (tid + g * kNt);
        if (e < whole) {
          r[g].load(x, e);
        } else {
          constexpr float kNone[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
          float v[N];
#pragma unroll
          for (int k = 0; k < N; ++k) v[k] = kNone[k];
          r[g].set(v);
        }
      }
    };
    load(lo);
    float rest = -INFINITY;
    if (tid < hi - whole) rest = E::get(x, whole + tid);
    // i: the wave's logits that reach the bound, u the lane's of token e, go to those that wait
    auto collect = [&](float u, int e, bool take) {
      for (int i = 0; i < a.n_stop; ++i) take = take && e != __builtin_amdgcn_readlane(stop, i);
      const unsigned long long at = __ballot(take);
      if (take) sh.part.wait[wv][waiting + below(at)] = comp(ord_key(u), static_cast<uint32_t>(e));
      waiting += __popcll(at);
    };
    int known = 64;              // of those that wait, how many the bound takes into account
    uint32_t mine = 0;           // what the wave has published
    auto publish = [&](uint32_t key) {
      mine = max(mine, key);
      if (lane == 0) __hip_atomic_store(&s_share[wv], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    auto shared = [&]() {        // (what it has of the others may be old: a smaller key, which is as true)
      uint32_t k[kW];
#pragma unroll
      for (int w = 0; w < kW; ++w) k[w] = __hip_atomic_load(&s_share[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      return min(min(k[0], k[1]), min(k[2], k[3]));
    };
    auto sharpen = [&]() {       // the N-th of the first 64 that wait
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      uint32_t top = lane < waiting ? static_cast<uint32_t>(sh.part.wait[wv][lane] >> 32) : 0u;
      sort64(top, lane, false);
      const uint32_t nth = __builtin_amdgcn_readlane(top, a.N - 1);
      sure = max(sure, nth);
      known = waiting;
      publish(__builtin_amdgcn_readlane(top, share - 1));
    };
    for (int e0 = lo; e0 < whole; e0 += kStep) {
      float v[G * N], gm[G];
#pragma unroll
      for (int k = 0; k < G * N; ++k) v[k] = r[k / N].get(k % N);
      if (e0 + kStep < whole) load(e0 + kStep);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        gm[g] = v[g * N];
#pragma unroll
        for (int k = 1; k < N; ++k) gm[g] = fmaxf(gm[g], v[g * N + k]);
      }
      const float mx = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
      const float m = fmaxf(z.m, mx), rel = m == -INFINITY ? 0.0f : m;  // of -inf alone: exp(-inf - 0) = 0, and NaN stays
      // exp(x - rel) as 2^(x log2e - r), one operation less a logit. r is rel log2e rounded, off by d, and the sum's 2^d is
      // made good by its first two terms: below 2^14 d is at most 2^-11, and the third one 2^-24
      const float r2 = rel * kLog2e;
      float s = 0.0f;
      if (!__ballot(!(fabsf(r2) < 16384.0f))) {
#pragma unroll
        for (int k = 0; k < G * N; ++k) s += __builtin_amdgcn_exp2f(fmaf(v[k], kLog2e, -r2));
        s = fmaf(s, -0.693147181f * fmaf(rel, kLog2e, -r2), s);
      } else {  // large, as where all of a lane's logits are masked by a finite number, or infinite
#pragma unroll
        for (int k = 0; k < G * N; ++k) s += exp_rel(v[k], rel);
      }
      z = {m, fmaf(z.s, exp_rel(z.m, rel), s)};
      if (e0 == lo && a.N + skip <= 64) {
        uint32_t top = ord_key(mx == mx ? mx : -INFINITY);
        sort64(top, lane, false);
        const uint32_t few = __builtin_amdgcn_readlane(top, share + skip - 1);
        top = __builtin_amdgcn_readlane(top, a.N + skip - 1);
        known = a.N;
        if (key_val(few) > -INFINITY) publish(few);
        if (key_val(top) > -INFINITY) {
          bound = key_val(top);
          sure = top;
        }
      }
      // (equal logits of other waves may come after this wave's, so that those stay)
      if (const uint32_t k = shared()) bound = fmaxf(bound, key_val(k));
      if (!__ballot(mx >= bound)) continue;
      uint32_t hits = 0;  // the lane's logits that reach the bound, a bit each
#pragma unroll
      for (int k = 0; k < G * N; ++k) hits |= v[k] >= bound ? 1u << k : 0u;
      while (__ballot(hits != 0u)) {  // one of each lane's at a time
        const int i = __ffs(static_cast<int>(hits)) - 1;
        float u[G * N];  // halved by the bits of i
#pragma unroll
        for (int k = 0; k < G * N; ++k) u[k] = v[k];
#pragma unroll
        for (int d = G * N / 2; d; d >>= 1)
#pragma unroll
          for (int k = 0; k < d; ++k) u[k] = i & d ? u[k + d] : u[k];
        collect(u[0], e0 + N * (tid + (i / N) * kNt) + i % N, hits != 0u && u[0] >= bound);
        hits &= hits - 1u;
        if (waiting <= 64) continue;
        // the first 64 of those that wait go into the list
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        uint64_t w = sh.part.wait[wv][lane];
        const uint64_t left = sh.part.wait[wv][64 + lane];
        waiting -= 64;
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        if (lane < waiting) sh.part.wait[wv][lane] = left;
        sort64(w, lane, true);
        merge64(best, w, lane);
        const uint32_t nth = __builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), a.N - 1);
        if (nth) {
          sure = max(sure, nth);
          bound = fmaxf(bound, key_val(nth));
          known = 0;
        }
        publish(__builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), share - 1));
      }
      if (waiting > known + max(4, a.N / 2)) sharpen();
      // what comes in later steps has higher tokens: among equal logits it is behind those that N have reached
      if (sure) bound = fmaxf(bound, next_up(key_val(sure)));
    }
    sure = max(sure, shared());
    if (whole < hi && wv == 0) {
      const float m = fmaxf(z.m, rest), rel = m == -INFINITY ? 0.0f : m;
      z = {m, z.s * exp_rel(z.m, rel) + exp_rel(rest, rel)};
      collect(rest, whole + lane, rest >= bound);
    }
    if (waiting > known + 8) sharpen();
    const int listed = min(__popcll(__ballot(best != 0ull)), a.N);
    if (lane < listed) sh.part.wait[wv][waiting + lane] = best;
    waiting += listed;
  }
  // the waves' sums and logits as the part's
  z = wave_lse(z);
  if (lane == 0) {
    s_m[wv] = z.m;
    s_s[wv] = z.s;
    s_bound[wv] = sure;
    s_wait[wv] = waiting;
  }
  __syncthreads();
  const int slot = row * a.P + part;
  const int lists = a.W * a.P, entries = lists * a.N;  // at most kNt lists (beam_parts)
  const unsigned long long* keys = a.s.key + static_cast<long long>(first) * a.P * a.N;
  const int n_ends = a.end_token ? a.W * a.n_stop : 0;
  // pieces of both ways to go on from here
  auto part_sum = [&](float* m) {
    *m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kW; ++w) s += static_cast<double>(*m == -INFINITY ? s_s[w] : s_s[w] * exp_rel(s_m[w], *m));
    return s;
  };
  auto last_of_group = [&]() {  // one thread: whether the group's other parts are done
    const unsigned t = __hip_atomic_fetch_add(&a.s.tick[group * kBeamPad], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (static_cast<int>(t) != lists - 1) return 0;
    agent_store(&a.s.tick[group * kBeamPad], 0u);
    return 1;
  };
  auto stop_logit = [&](int i, int* b, int* t) {  // of beam b's row, of the stop token t
    *b = static_cast<int>(divide(static_cast<uint32_t>(i), static_cast<uint32_t>(a.n_stop), a.m_stop));
    *t = a.stops[i - *b * a.n_stop];
    return E::get(static_cast<const char*>(a.x) + (first + *b) * a.ld * E::kSize, *t);
  };
  auto keep_lse = [&](int b, float top, double s, float sc) {  // NaN for a row that is not live
    const double lse = static_cast<double>(top) + log(s);
    s_lse[b] = finite(sc) && __builtin_isfinite(lse) ? lse : NAN;
    s_score[b] = static_cast<double>(sc);
  };
  const int heads = lists << a.log_j;  // the lists' first entries, 2^log_j of each
  auto head_of = [&](int i) { return agent_load(&keys[(i >> a.log_j) * a.N + (i & ((1 << a.log_j) - 1))]); };
  auto beam_of = [&](int l) { return static_cast<int>(divide(static_cast<uint32_t>(l), static_cast<uint32_t>(a.P), a.m_parts)); };
  auto entry = [&](uint64_t key, int b) {
    const double lse = s_lse[b];
    if (!key || lse != lse) return none();
    return Cand{ord_f64(s_score[b] + (static_cast<double>(comp_val(key)) - lse)),
                static_cast<uint64_t>(63 - b) << 52 | key >> 32 << 20 | (key & 0xFFFFFu)};
  };
  auto end_entry = [&](float u, int b, int t) { return u > -INFINITY ? entry(comp(ord_key(u), static_cast<uint32_t>(t)), b) : none(); };
  // its score as fp32 below it, next to zero as well; a key (0: nothing). From such a key a bound for scores
  auto below_score = [&](const Cand& c) { return c.s ? ord_key(static_cast<float>(f64_ord(c.s))) - 2u : 0u; };
  auto score_bound = [&](uint32_t k) { return k ? ord_f64(static_cast<double>(key_val(k))) : static_cast<uint64_t>(1); };
  auto put = [&](int* token, int* parent, float* score, int at, const Cand& c) {
    const long long o = static_cast<long long>(group) * a.N + at;
    int b = at;
    while (b >= a.W) b -= a.W;
    token[o] = c.s ? static_cast<int>(~static_cast<uint32_t>(c.t) & 0xFFFFFu) : -1;
    parent[o] = a.row0 + first + (c.s ? 63 - static_cast<int>(c.t >> 52) : b);
    score[o] = c.s ? static_cast<float>(f64_ord(c.s)) : -INFINITY;
  };

  if (a.alone) {  // small groups: the first wave does the rest by itself, without waiting for others
    if (wv != 0) return;
    const uint32_t most = max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3]));
    int n = 0;
    uint64_t has[kW];
#pragma unroll
    for (int w = 0; w < kW; ++w) has[w] = lane < s_wait[w] ? sh.part.wait[w][lane] : 0ull;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      uint64_t key = has[w];
      for (int i = lane;;) {
        const bool take = key != 0 && key >> 32 >= most;
        const unsigned long long at = __ballot(take);
        if (take) sh.part.list[n + below(at)] = key;
        n += __popcll(at);
        i += 64;
        if (i - lane >= s_wait[w]) break;
        key = i < s_wait[w] ? sh.part.wait[w][i] : 0ull;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll 1
    for (int t = lane; t < max(n, a.N); t += 64) {
      const uint64_t key = t < n ? sh.part.list[t] : 0ull;
      const int rank = t < n ? count_before(sh.part.list, n, key) : t;
      if (rank < a.N) agent_store(&a.s.key[slot * a.N + rank], static_cast<unsigned long long>(key));
    }
    float m;
    double s = part_sum(&m);
    int last = 0;
    if (lane == 0) {
      agent_store(&a.s.max[slot], m);
      agent_store(&a.s.sum[slot], s);
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (lane == 0) last = last_of_group();
    if (!__builtin_amdgcn_readfirstlane(last)) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    constexpr int kOwn = kNt / 64;
    uint64_t key[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) key[k] = lane + 64 * k < entries ? agent_load(&keys[lane + 64 * k]) : 0ull;
    const uint64_t head = lane < heads ? head_of(lane) : 0ull;
    const int b = lane >> a.log_s, p = lane & ((1 << a.log_s) - 1);
    float sc = 0.0f, end_x = -INFINITY;
    int end_b = 0, end_t = 0;
    m = -INFINITY;
    s = 0.0;
    if (b < a.W && p < a.P) {
      m = agent_load(&a.s.max[(first + b) * a.P + p]);
      s = agent_load(&a.s.sum[(first + b) * a.P + p]);
      sc = a.scores[first + b];
    }
    if (lane < n_ends) end_x = stop_logit(lane, &end_b, &end_t);
    float top = m;
    if (a.log_s > 0) top = fmaxf(top, __uint_as_float(lane_xor<1>(__float_as_uint(top), lane)));
    if (a.log_s > 1) top = fmaxf(top, __uint_as_float(lane_xor<2>(__float_as_uint(top), lane)));
    if (a.log_s > 2) top = fmaxf(top, __uint_as_float(lane_xor<4>(__float_as_uint(top), lane)));
    if (a.log_s > 3) top = fmaxf(top, __uint_as_float(lane_xor<8>(__float_as_uint(top), lane)));
    if (a.log_s > 4) top = fmaxf(top, __uint_as_float(lane_xor<16>(__float_as_uint(top), lane)));
    if (a.log_s > 5) top = fmaxf(top, __uint_as_float(lane_xor<32>(__float_as_uint(top), lane)));
    if (m != -INFINITY) s *= static_cast<double>(exp_rel(m, top));  // (a sum at -inf is 0 or NaN)
    auto f64 = [](uint64_t v) { return __longlong_as_double(static_cast<long long>(v)); };
    auto u64 = [](double v) { return static_cast<uint64_t>(__double_as_longlong(v)); };
    if (a.log_s > 0) s += f64(lane_xor<1>(u64(s), lane));
    if (a.log_s > 1) s += f64(lane_xor<2>(u64(s), lane));
    if (a.log_s > 2) s += f64(lane_xor<4>(u64(s), lane));
    if (a.log_s > 3) s += f64(lane_xor<8>(u64(s), lane));
    if (a.log_s > 4) s += f64(lane_xor<16>(u64(s), lane));
    if (a.log_s > 5) s += f64(lane_xor<32>(u64(s), lane));
    if (b < a.W && p == 0) keep_lse(b, top, s, sc);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    // the N-th of the lists' first entries: a bound for all entries
    uint32_t t = lane < heads ? below_score(entry(head, beam_of(lane >> a.log_j))) : 0u;
    sort64(t, lane, false);
    const uint64_t bound = score_bound(__builtin_amdgcn_readlane(t, a.N - 1));
    Cand c[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int l = static_cast<int>(divide(static_cast<uint32_t>(min(lane + 64 * k, entries - 1)), static_cast<uint32_t>(a.N), a.m_n));
      c[k] = entry(key[k], beam_of(l));
    }
    int c_n = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const unsigned long long at = __ballot(c[k].s >= bound);
      if (c[k].s >= bound) sh.group.cand[c_n + below(at)] = c[k];
      c_n += __popcll(at);
    }
    const Cand end = end_entry(end_x, end_b, end_t);
    const unsigned long long at = __ballot(end.s >= bound);
    if (end.s >= bound) sh.group.end[below(at)] = end;
    const int ends = __popcll(at);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll 1
    for (int i = lane; i < max(c_n, a.N); i += 64) {
      const Cand o = i < c_n ? sh.group.cand[i] : none();
      const int rank = i < c_n ? count_before(sh.group.cand, c_n, o) : i;
      if (rank < a.N) put(a.token, a.parent, a.score, rank, o);
    }
    if (!a.end_token) return;
    bool ended = false;
    if (end.s >= bound) {
      const int rank = count_before(sh.group.end, ends, end);
      ended = rank + count_before(sh.group.cand, c_n, end) < a.N;
      if (ended) put(a.end_token, a.end_parent, a.end_score, rank, end);
    }
    const int n_end = __popcll(__ballot(ended));
    if (lane >= n_end && lane < a.N) put(a.end_token, a.end_parent, a.end_score, lane, none());
    if (lane == 0) a.n_end[group] = n_end;
    return;
  }

  {
    const uint32_t most = max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3]));
    auto give = [&](uint64_t key) {
      const bool take = key != 0 && key >> 32 >= most;
      const unsigned long long at = __ballot(take);
      if (!at) return;
      int to = 0;
      if (lane == 0) to = atomicAdd(&s_n, __popcll(at));
      to = __builtin_amdgcn_readfirstlane(to) + below(at);
      if (take) sh.part.list[to] = key;
    };
#pragma unroll 1
    for (int i = lane; i < (waiting + 63 & ~63); i += 64) give(i < waiting ? sh.part.wait[wv][i] : 0ull);
  }
  __syncthreads();
  // hand over through the device's memory: agent-scope stores, completed before the ticket is taken; the part
  // with the group's last ticket reads them with agent-scope loads after an acquire, and clears the ticket
  const int n = s_n;
#pragma unroll 1
  for (int t = tid; t < max(n, a.N); t += kNt) {
    const uint64_t key = t < n ? sh.part.list[t] : 0ull;
    const int rank = t < n ? count_before(sh.part.list, n, key) : t;
    if (rank < a.N) agent_store(&a.s.key[slot * a.N + rank], static_cast<unsigned long long>(key));
  }
  if (wv == kW - 1) {  // (the last wave has no logits to rank, mostly)
    float m;
    const double s = part_sum(&m);
    if (lane == 0) {
      agent_store(&a.s.max[slot], m);
      agent_store(&a.s.sum[slot], s);
    }
  }
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (tid == 0) {
    s_last = last_of_group();
    s_n = s_lists = s_end = s_ended = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const bool few = entries <= kNt;  // an entry a thread

  // what does not wait for the rows' sums is loaded first
  const uint64_t mine = few && tid < entries ? agent_load(&keys[tid]) : 0ull;
  const uint64_t head = tid < heads ? head_of(tid) : 0ull;
  float end_x = -INFINITY;
  int end_b = 0, end_t = 0;
  if (tid < n_ends) end_x = stop_logit(tid, &end_b, &end_t);
  // lse of each row, its parts side by side in lanes; NaN for a row that is not live
#pragma unroll 1
  for (int i0 = 0; i0 < a.W << a.log_s; i0 += kNt) {
    const int b = (i0 + tid) >> a.log_s, p = (i0 + tid) & ((1 << a.log_s) - 1);
    float m = -INFINITY, sc = 0.0f;
    double s = 0.0;
    if (b < a.W && p < a.P) {
      m = agent_load(&a.s.max[(first + b) * a.P + p]);
      s = agent_load(&a.s.sum[(first + b) * a.P + p]);
      sc = a.scores[first + b];
    }
    float top = m;
#pragma unroll 1
    for (int d = 1 << a.log_s >> 1; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (m != -INFINITY) s *= static_cast<double>(exp_rel(m, top));  // (a sum at -inf is 0 or NaN)
#pragma unroll 1
    for (int d = 1 << a.log_s >> 1; d; d >>= 1) s += __shfl_xor(s, d);
    if (b < a.W && p == 0) keep_lse(b, top, s, sc);
  }
  __syncthreads();
  // the N-th of the first entries that a wave's threads have, their scores as fp32 below them: the largest of the
  // waves' is a bound for all entries
  uint32_t top = tid < heads ? below_score(entry(head, beam_of(tid >> a.log_j))) : 0u;
  if (wv * 64 < heads) sort64(top, lane, false);
  if (lane == a.N - 1) s_bound[wv] = top;
  __syncthreads();
  const uint64_t bound = score_bound(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])));
  // the stop tokens' continuations; N others come before those that do not reach the bound
#pragma unroll 1
  for (int i = tid; i < n_ends; i += kNt) {
    if (i >= kNt) end_x = stop_logit(i, &end_b, &end_t);
    const Cand c = end_entry(end_x, end_b, end_t);
    if (c.s >= bound) sh.group.end[atomicAdd(&s_end, 1)] = c;
  }
  // the entries that reach it: of all lists, or of those whose first one does
  int some = lists;
  if (!few) {
    if (tid < lists && entry(agent_load(&keys[tid * a.N]), beam_of(tid)).s >= bound)
      sh.group.lists[atomicAdd(&s_lists, 1)] = static_cast<unsigned char>(tid);
    __syncthreads();
    some = s_lists;
  }
#pragma unroll 1
  for (int i = tid; i < some * a.N; i += kNt) {
    const int at = static_cast<int>(divide(static_cast<uint32_t>(i), static_cast<uint32_t>(a.N), a.m_n));
    const int l = few ? at : sh.group.lists[at];
    const Cand c = entry(few ? mine : agent_load(&keys[l * a.N + (i - at * a.N)]), beam_of(l));
    if (c.s >= bound) {
      const int to = atomicAdd(&s_n, 1);
      if (to < kCands) sh.group.cand[to] = c;
    }
  }
  __syncthreads();
  int c_n = s_n;  // continuations in sh.group.cand, the first N among them
  const int ends = s_end;
  if (c_n > kCands) {
    Cand c = none();
    __syncthreads();
#pragma unroll 1
    for (int l = wv; l < lists; l += kW) {
      const int b = beam_of(l);
      if (entry(agent_load(&keys[l * a.N]), b).s < bound) continue;
      uint64_t k = 0;
      if (63 - lane < a.N) k = agent_load(&keys[l * a.N + 63 - lane]);
      merge64(c, entry(k, b), lane);
    }
    sh.merge[wv][lane] = c;
    __syncthreads();
    if (wv == 0)
#pragma unroll 1
      for (int w = 1; w < kW; ++w) merge64(c, sh.merge[w][63 - lane], lane);
    __syncthreads();
    if (wv == 0) sh.group.cand[lane] = c;
    c_n = a.N;
    __syncthreads();
  }
#pragma unroll 1
  for (int t = tid; t < max(c_n, a.N); t += kNt) {
    const Cand c = t < c_n ? sh.group.cand[t] : none();
    const int rank = t < c_n ? count_before(sh.group.cand, c_n, c) : t;
    if (rank < a.N) put(a.token, a.parent, a.score, rank, c);
  }
  if (!a.end_token) return;
  // an end is one of the first N of all if fewer come before it, ends or not; those that do are among the candidates.
  // (The second wave begins with them: the first has the others to rank, mostly.)
  int ended = 0;
#pragma unroll 1
  for (int t = (tid - 64) & (kNt - 1); t < ends; t += kNt) {
    const Cand c = sh.group.end[t];
    int rank = count_before(sh.group.cand, c_n, c);
    if (rank >= a.N) continue;
    const int among = count_before(sh.group.end, ends, c);
    if (rank + among >= a.N) continue;
    put(a.end_token, a.end_parent, a.end_score, among, c);
    ++ended;
  }
  if (ended) atomicAdd(&s_ended, ended);
  __syncthreads();
#pragma unroll 1
  for (int t = s_ended + tid; t < a.N; t += kNt) put(a.end_token, a.end_parent, a.end_score, t, none());
  if (tid == 0) a.n_end[group] = s_ended;
}

}  // namespace

// Workgroups of four a CU or fewer, each of whole steps. Measured for one, two, four and eight a CU, us: 64 x 8 x 128,256
// fp32 52.8, 52.7, 50.0, 55.7; 16 x 16 x 128,256 bf16 44.9, 31.6, 29.5, 34.8; 24 x 5 x 50,257 f16 23.3, 18.4, 15.4, 15.4; 200 x
// 5 x 50,257 fp32 41.6, 41.6, 41.5, 49.0 (1,000 rows: one part each; two, more than four a CU, 49.5). No more lists than
// threads in the group's last part: 1 x 8 x 151,936 in 32 parts a row 13.6, in 38 16.0.
void beam_parts(int B, int W, int V, int dtype, int cus, int* P, int* L) {
  const int step = kNt * 4 * (dtype == VSMP_F32 ? 4 : 8);
  const int steps = (V + step - 1) / step;
  int p = 4 * cus / B;
  if (p > steps) p = steps;
  if (p > kNt / W) p = kNt / W;  // the group's last part reads a list a thread
  if (p > 64) p = 64;            // and a row's sums side by side in a wave
  if (p > kBeamSlots / B) p = kBeamSlots / B;
  if (p < 1) p = 1;
  *L = (steps + p - 1) / p * step;
  *P = (V + *L - 1) / *L;
}

void launch_beam(BeamArgs a, int dtype, hipStream_t st) {
  a.m_parts = 0xFFFFFFFFu / static_cast<uint32_t>(a.P);
  a.m_n = 0xFFFFFFFFu / static_cast<uint32_t>(a.N);
  a.m_stop = a.n_stop ? 0xFFFFFFFFu / static_cast<uint32_t>(a.n_stop) : 0u;
  a.log_s = 0;
  while (1 << a.log_s < a.P) ++a.log_s;
  // as many first entries of each list as make a sharp bound: few lists have most of the best
  const int lists = a.W * a.P;
  a.alone = a.W << a.log_s <= 64 && lists * a.N <= kNt && lists <= 64 && a.W * a.n_stop <= 64 && a.N <= 16;
  a.log_j = 0;
  while (2 << a.log_j <= a.N && lists << a.log_j <= (a.alone ? 64 : kNt) / 2) ++a.log_j;
  const dim3 grid(static_cast<unsigned>(a.P), static_cast<unsigned>(a.W), static_cast<unsigned>(a.G));
  if (dtype == VSMP_F32)
    hipLaunchKernelGGL(k_beam<F32>, grid, dim3(kNt), 0, st, a);
  else if (dtype == VSMP_BF16)
    hipLaunchKernelGGL(k_beam<Bf16>, grid, dim3(kNt), 0, st, a);
  else
    hipLaunchKernelGGL(k_beam<F16>, grid, dim3(kNt), 0, st, a);
}

}  // namespace vsmp
