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
// How many of the lanes' flags below this one are set.
__device__ __forceinline__ int below(unsigned long long at) {
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(at >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(at), 0u)));
}

// ---- k_beam ----------------------------------------------------------------------------------------------

constexpr int kCands = 256;  // continuations that the last part ranks side by side

// One part of a row: a step of four 16-byte groups a thread at a time, the next in flight. Each wave collects in LDS the
// logits that reach its bound, below which none can be among the part's N largest that are no stop tokens. The bound
// is at first the N-th largest (or one below it) of the lanes' maxima over the first step: the least of the maxima of
// as many groups of lanes, stop tokens' groups left out of account. Where 64 have collected, the wave sorts them into a
// list over its lanes, whose N-th is the bound from then on. In the end the waves' logits that reach the largest of their
// bounds are ranked by comparing each with each, a thread each: mostly they are few more than N.
//
// The last part of a group ranks its rows' lists by score in the same way: the N-th largest first entry of the lists (of
// those of a wave's threads) is a bound for all entries. Where more entries than kCands reach it (many equal
// ones) each wave merges lists in order instead, and the first wave the waves'.
template <class E>
__global__ __launch_bounds__(kNt) void k_beam(BeamArgs a) {
  constexpr int N = 16 / E::kSize, G = 4;
  constexpr int kStep = kNt * N * G;
  union Shared {
    struct {
      uint64_t wait[kW][128], list[kNt];
    } part;
    struct {
      Cand cand[kCands];
      Cand end[kBeamMax * kBeamStops];
    } group;
    Cand merge[kW][kBeamMax];
  };
  __shared__ Shared sh;
  __shared__ float s_m[kW];
  __shared__ double s_s[kW], s_lse[kBeamMax], s_score[kBeamMax];
  __shared__ uint64_t s_bound[kW];
  __shared__ int s_wait[kW], s_n, s_end, s_ended, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.P));
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.P));
  const int group = row / a.W;
  const int lo = part * a.L, hi = min(a.V, lo + a.L);
  const char* x = static_cast<const char*>(a.x) + row * a.ld * E::kSize;

  auto is_stop = [&](int t) {
    bool s = false;
    for (int i = 0; i < a.n_stop; ++i) s |= t == a.stops[i];
    return s;
  };

  Lse z{-INFINITY, 0.0f};
  int waiting = 0;               // logits that the wave has collected
  uint32_t sure = 0;             // a key that N of its logits reach, no stop tokens among them; 0: none known
  if (finite(a.scores[row])) {
    uint64_t best = 0;           // the lane's entry of the wave's list; 0: none
    bool listed = false;
    float bound = -FLT_MAX;
    int skip = 0;                // stop tokens in this part
    for (int i = 0; i < a.n_stop; ++i) skip += a.stops[i] >= lo && a.stops[i] < hi ? 1 : 0;
    auto flush = [&]() {         // the first 64 of those that wait go into the list
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      const int n = min(waiting, 64);
      uint64_t v = lane < n ? sh.part.wait[wv][lane] : 0ull;
      const uint64_t rest = sh.part.wait[wv][64 + lane];
      waiting -= n;
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      if (lane < waiting) sh.part.wait[wv][lane] = rest;
      sort64(v, lane, true);
      merge64(best, v, lane);
      listed = true;
      const uint32_t nth = __builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), a.N - 1);
      if (nth) {
        sure = nth;
        bound = fmaxf(bound, key_val(nth));
      }
    };
    Raw<E, N> r[G];
    auto load = [&](int e0) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int e = e0 + N * (tid + g * kNt);
        if (e + N <= hi) {
          r[g].load(x, e);
        } else {  // the row's end: its last elements one by one, then -inf
          float v[N];
#pragma unroll
          for (int k = 0; k < N; ++k) v[k] = e + k < hi ? E::get(x, e + k) : -INFINITY;
          r[g].set(v);
        }
      }
    };
    load(lo);
    for (int e0 = lo; e0 < hi; e0 += kStep) {
      float v[G][N], gm[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < N; ++k) v[g][k] = r[g].get(k);
      if (e0 + kStep < hi) load(e0 + kStep);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        gm[g] = v[g][0];
#pragma unroll
        for (int k = 1; k < N; ++k) gm[g] = fmaxf(gm[g], v[g][k]);
      }
      const float mx = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
      const float m = fmaxf(z.m, mx), rel = m == -INFINITY ? 0.0f : m;  // of -inf alone: exp(-inf - 0) = 0, and NaN stays
      float s = z.s * exp_rel(z.m, rel);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < N; ++k) s += exp_rel(v[g][k], rel);
      z = {m, s};
      if (e0 == lo && a.N + skip <= 64) {
        // groups of 64 / M lanes, M >= N + skip: their maxima, and the least of those
        const int M = a.N + skip;
        float t = mx == mx ? mx : -INFINITY;
        auto with = [&](float o, bool within) { t = within ? fmaxf(t, o) : fminf(t, o); };
        with(__uint_as_float(lane_xor<32>(__float_as_uint(t), lane)), M <= 32);
        with(__uint_as_float(lane_xor<16>(__float_as_uint(t), lane)), M <= 16);
        with(__uint_as_float(lane_xor<8>(__float_as_uint(t), lane)), M <= 8);
        with(__uint_as_float(lane_xor<4>(__float_as_uint(t), lane)), M <= 4);
        with(__uint_as_float(lane_xor<2>(__float_as_uint(t), lane)), M <= 2);
        with(__uint_as_float(lane_xor<1>(__float_as_uint(t), lane)), M <= 1);
        if (t > -INFINITY) {
          bound = t;
          sure = ord_key(t);
        }
      }
      if (__ballot(mx >= bound)) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (!__ballot(gm[g] >= bound)) continue;
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int e = e0 + N * (tid + g * kNt) + k;
            bool take = v[g][k] >= bound;
            if (!__ballot(take)) continue;
            take = take && !is_stop(e);
            const unsigned long long at = __ballot(take);
            const int pos = waiting + below(at);
            if (take) sh.part.wait[wv][pos] = comp(ord_key(v[g][k]), static_cast<uint32_t>(e));
            waiting += __popcll(at);
            if (waiting > 64) flush();
          }
        }
        // what comes in later steps has higher tokens: among equal logits it is behind those that N have reached
        if (sure) bound = fmaxf(bound, next_up(key_val(sure)));
      }
    }
    if (listed) {  // in order, so that no more than N of them count
      flush();
      if (waiting) flush();
      waiting = __popcll(__ballot(best != 0 && lane < a.N));
      if (lane < waiting) sh.part.wait[wv][lane] = best;
    }
  }
  // the waves' sums and logits as the part's
  z = wave_lse(z);
  if (lane == 0) {
    s_m[wv] = z.m;
    s_s[wv] = static_cast<double>(z.s);
    s_bound[wv] = sure;
    s_wait[wv] = waiting;
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  const int slot = row * a.P + part;
  {
    const uint64_t most = max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3]));
    const uint64_t key = lane < s_wait[wv] ? sh.part.wait[wv][lane] : 0ull;
    const bool take = key != 0 && key >> 32 >= most;
    const unsigned long long at = __ballot(take);
    int first = 0;
    if (lane == 0 && at) first = atomicAdd(&s_n, __popcll(at));
    first = __builtin_amdgcn_readfirstlane(first);
    if (take) sh.part.list[first + below(at)] = key;
  }
  __syncthreads();
  // hand over through the device's memory: agent-scope stores, completed before the ticket is taken; the part
  // with the group's last ticket reads them with agent-scope loads after an acquire, and clears the ticket
  const int n = s_n;
  if (tid < n) {
    const uint64_t key = sh.part.list[tid];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += sh.part.list[i] > key ? 1 : 0;
    if (rank < a.N) agent_store(&a.s.key[slot * a.N + rank], static_cast<unsigned long long>(key));
  } else if (tid < a.N) {
    agent_store(&a.s.key[slot * a.N + tid], 0ull);
  }
  if (tid == 0) {
    float m = s_m[0];
#pragma unroll
    for (int w = 1; w < kW; ++w) m = fmaxf(m, s_m[w]);
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kW; ++w) s += m == -INFINITY ? s_s[w] : s_s[w] * static_cast<double>(exp_rel(s_m[w], m));
    agent_store(&a.s.max[slot], m);
    agent_store(&a.s.sum[slot], s);
  }
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (tid == 0) {
    const unsigned t = __hip_atomic_fetch_add(&a.s.tick[group * kBeamPad], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = static_cast<int>(t) == a.W * a.P - 1;
    s_n = s_end = s_ended = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  if (tid == 0) agent_store(&a.s.tick[group * kBeamPad], 0u);
  const int first = group * a.W;  // the group's first row
  const int lists = a.W * a.P, entries = lists * a.N;
  const unsigned long long* keys = a.s.key + static_cast<long long>(first) * a.P * a.N;

  // what does not wait for the rows' sums is loaded first
  constexpr int kAhead = 4;
  uint64_t key[kAhead], head[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int e = tid + k * kNt;
    key[k] = e < entries ? agent_load(&keys[e]) : 0ull;
    head[k] = e < lists ? agent_load(&keys[e * a.N]) : 0ull;
  }
  // lse of each row, its parts side by side in lanes; NaN for a row that is not live
  int S = 1;
  while (S < a.P) S <<= 1;
  for (int i = tid; i < a.W * S + kNt - 1 - (a.W * S - 1) % kNt; i += kNt) {
    const int b = i / S, p = i % S;
    float m = -INFINITY, sc = 0.0f;
    double s = 0.0;
    if (b < a.W && p < a.P) {
      m = agent_load(&a.s.max[(first + b) * a.P + p]);
      s = agent_load(&a.s.sum[(first + b) * a.P + p]);
      sc = a.scores[first + b];
    }
    float top = m;
    for (int d = S >> 1; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (m != top) s *= m == -INFINITY ? 1.0 : exp(static_cast<double>(m) - static_cast<double>(top));  // (a sum at -inf is 0 or NaN)
    for (int d = S >> 1; d; d >>= 1) s += __shfl_xor(s, d);
    if (b < a.W && p == 0) {
      const double lse = static_cast<double>(top) + log(s);
      s_lse[b] = finite(sc) && __builtin_isfinite(lse) ? lse : NAN;
      s_score[b] = static_cast<double>(sc);
    }
  }
  __syncthreads();
  auto entry = [&](uint64_t key, int b) {
    const double lse = s_lse[b];
    if (!key || lse != lse) return none();
    return Cand{ord_f64(s_score[b] + (static_cast<double>(comp_val(key)) - lse)),
                static_cast<uint64_t>(63 - b) << 52 | key >> 32 << 20 | (key & 0xFFFFFu)};
  };
  auto put = [&](int* token, int* parent, float* score, int at, const Cand& c, bool there) {
    const long long o = static_cast<long long>(group) * a.N + at;
    token[o] = there ? static_cast<int>(~static_cast<uint32_t>(c.t) & 0xFFFFFu) : -1;
    parent[o] = a.row0 + first + (there ? 63 - static_cast<int>(c.t >> 52) : at % a.W);
    score[o] = there ? static_cast<float>(f64_ord(c.s)) : -INFINITY;
  };
  // the N-th of the first entries that a wave's threads have: the largest of the waves' is a bound for all entries
  uint64_t bound;
  {
    uint64_t top = 0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint64_t s = tid + k * kNt < lists ? entry(head[k], (tid + k * kNt) / a.P).s : 0ull;
      top = s > top ? s : top;
    }
    for (int l = tid + kAhead * kNt; l < lists; l += kNt) {
      const uint64_t s = entry(agent_load(&keys[l * a.N]), l / a.P).s;
      top = s > top ? s : top;
    }
    if (wv * 64 < lists) sort64(top, lane, false);
    if (lane == a.N - 1) s_bound[wv] = top;
    __syncthreads();
    bound = max(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])), static_cast<uint64_t>(1));
  }
  // the stop tokens' continuations; N others come before those that do not reach the bound
  if (a.end_token) {
    for (int i = tid; i < a.W * a.n_stop; i += kNt) {
      const int b = i / a.n_stop, t = a.stops[i % a.n_stop];
      const float u = E::get(static_cast<const char*>(a.x) + (first + b) * a.ld * E::kSize, t);
      const Cand c = u > -INFINITY ? entry(comp(ord_key(u), static_cast<uint32_t>(t)), b) : none();
      if (c.s >= bound) sh.group.end[atomicAdd(&s_end, 1)] = c;
    }
  }
  auto collect = [&](uint64_t key, int e) {
    const Cand c = key ? entry(key, e / (a.P * a.N)) : none();
    const bool take = c.s >= bound;
    const unsigned long long at = __ballot(take);
    if (!at) return;
    int to = 0;
    if (lane == 0) to = atomicAdd(&s_n, __popcll(at));
    to = __builtin_amdgcn_readfirstlane(to) + below(at);
    if (take && to < kCands) sh.group.cand[to] = c;
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (k * kNt < entries) collect(key[k], min(tid + k * kNt, entries - 1));
  for (int e0 = kAhead * kNt; e0 < entries; e0 += kAhead * kNt) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) key[k] = e0 + tid + k * kNt < entries ? agent_load(&keys[e0 + tid + k * kNt]) : 0ull;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (e0 + k * kNt < entries) collect(key[k], min(e0 + tid + k * kNt, entries - 1));
  }
  __syncthreads();
  int c_n = s_n;  // continuations in sh.group.cand, the first N among them
  const int ends = s_end;
  if (c_n > kCands) {
    Cand c = none();
    __syncthreads();
    for (int l = wv; l < lists; l += kW) {
      const Cand top = entry(agent_load(&keys[l * a.N]), l / a.P);
      if (top.s < bound) continue;
      uint64_t k = 0;
      if (63 - lane < a.N) k = agent_load(&keys[l * a.N + 63 - lane]);
      merge64(c, entry(k, l / a.P), lane);
    }
    sh.merge[wv][lane] = c;
    __syncthreads();
    if (wv == 0)
      for (int w = 1; w < kW; ++w) merge64(c, sh.merge[w][63 - lane], lane);
    __syncthreads();
    if (wv == 0) sh.group.cand[lane] = c;
    c_n = a.N;
    __syncthreads();
  }
  for (int t = tid; t < max(c_n, a.N); t += kNt) {
    if (t >= c_n) {
      put(a.token, a.parent, a.score, t, none(), false);
      continue;
    }
    const Cand c = sh.group.cand[t];
    int rank = 0;
    for (int i = 0; i < c_n; ++i) rank += before(sh.group.cand[i], c) ? 1 : 0;
    if (rank < a.N) put(a.token, a.parent, a.score, rank, c, true);
  }
  if (!a.end_token) return;
  // an end is one of the first N of all if fewer come before it, ends or not; those that do are among the candidates
  int mine = 0;
  for (int t = tid; t < ends; t += kNt) {
    const Cand c = sh.group.end[t];
    int others = 0, rank = 0;
    for (int i = 0; i < c_n; ++i) others += before(sh.group.cand[i], c) ? 1 : 0;
    if (others >= a.N) continue;
    for (int i = 0; i < ends; ++i) rank += before(sh.group.end[i], c) ? 1 : 0;
    if (others + rank >= a.N) continue;
    put(a.end_token, a.end_parent, a.end_score, rank, c, true);
    ++mine;
  }
  if (mine) atomicAdd(&s_ended, mine);
  __syncthreads();
  for (int t = s_ended + tid; t < a.N; t += kNt) put(a.end_token, a.end_parent, a.end_score, t, none(), false);
  if (tid == 0) a.n_end[group] = s_ended;
}

}  // namespace

void beam_parts(int B, int V, int dtype, int cus, int* P, int* L) {
  const int step = kNt * 4 * (dtype == VSMP_F32 ? 4 : 8);
  const int steps = (V + step - 1) / step;
  int p = (4 * cus + B - 1) / B;
  if (p > steps) p = steps;
  if (p > 64) p = 64;  // a lane each reads their results
  if (p > kBeamSlots / B) p = kBeamSlots / B;
  if (p < 1) p = 1;
  *L = (steps + p - 1) / p * step;
  *P = (V + *L - 1) / *L;
}

void launch_beam(const BeamArgs& a, int dtype, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.G) * static_cast<unsigned>(a.W) * static_cast<unsigned>(a.P));
  if (dtype == VSMP_F32)
    hipLaunchKernelGGL(k_beam<F32>, grid, dim3(kNt), 0, st, a);
  else if (dtype == VSMP_BF16)
    hipLaunchKernelGGL(k_beam<Bf16>, grid, dim3(kNt), 0, st, a);
  else
    hipLaunchKernelGGL(k_beam<F16>, grid, dim3(kNt), 0, st, a);
}

}  // namespace vsmp
