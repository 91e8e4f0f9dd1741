// One step of beam search (k_beam): a row's log of the sum of exponentials and its largest logits in one pass, then,
// in the group's last part, the best continuations over its rows.
#include <cfloat>

#include "vsmp_beam.hpp"
#include "vsmp_keys.hpp"
#include "vsmp_rows.hpp"

namespace vsmp {
namespace {

constexpr int kNt = 256;       // threads per workgroup
constexpr int kW = kNt / 64;   // its waves

// ---- lists of 64 in a wave, an entry a lane -------------------------------------------------------------

__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int d) { return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)); }
__device__ __forceinline__ uint64_t lane_xor(uint64_t v, int d) {
  return static_cast<uint64_t>(lane_xor(static_cast<uint32_t>(v >> 32), d)) << 32 | lane_xor(static_cast<uint32_t>(v), d);
}

// A continuation: its score as a whole number in the scores' order, its row's composite (logit, token), its beam.
// That of nothing comes after all others.
struct Cand {
  uint64_t s, key;
  uint32_t beam;
};
__device__ __forceinline__ bool before(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ bool before(uint32_t a, uint32_t b) { return a > b; }
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) {
  return a.s > b.s || (a.s == b.s && (a.beam < b.beam || (a.beam == b.beam && a.key > b.key)));
}
__device__ __forceinline__ Cand lane_xor(const Cand& c, int d) { return {lane_xor(c.s, d), lane_xor(c.key, d), lane_xor(c.beam, d)}; }
__device__ __forceinline__ Cand none() { return {0u, 0u, 0xFFFFFFFFu}; }

__device__ __forceinline__ uint64_t ord_f64(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double f64_ord(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7FFFFFFFFFFFFFFFull : ~k));
}

// One exchange of a sorting network: with the lane d away, the lane keeps the earlier or the later of the two.
template <class T>
__device__ __forceinline__ void exchange(T& v, int d, bool earlier) {
  const T o = lane_xor(v, d);
  if (before(o, v) == earlier) v = o;  // (of equal entries it does not matter which)
}
// Sorted over the wave: lane 0 first, or with `last_first` lane 63.
template <class T>
__device__ __forceinline__ void sort64(T& v, int lane, bool last_first) {
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) exchange(v, j, ((lane & k & 63) == 0) == ((lane & j) == 0) ? !last_first : last_first);
}
// The first 64 of a sorted list and of one sorted the other way round, sorted.
template <class T>
__device__ __forceinline__ void merge64(T& v, const T& reversed, int lane) {
  if (before(reversed, v)) v = reversed;
#pragma unroll
  for (int j = 32; j; j >>= 1) exchange(v, j, (lane & j) == 0);
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

// ---- k_beam ----------------------------------------------------------------------------------------------

// One part of a row: a step of four 16-byte groups a thread at a time, the next in flight. Each wave keeps its N
// largest logits that are no stop tokens, a sorted list over its lanes, and a bound: no logit below it can be among
// them. Logits that reach the bound wait in LDS until there are 64, which are then sorted and merged into the list.
// The first bound is the N-th largest of the lanes' maxima over the first step (the stop tokens' lanes left out of
// account): so many logits reach it.
//
// The last part of a group ranks its rows' lists by score. A list whose first entry does not reach the N-th of all
// first entries has none of the best N; of the others, every wave merges some, and the first wave the waves'.
template <class E>
__global__ __launch_bounds__(kNt) void k_beam(BeamArgs a) {
  constexpr int N = 16 / E::kSize, G = 4;
  constexpr int kStep = kNt * N * G;
  __shared__ uint64_t s_wait[kW][128];
  __shared__ float s_m[kW];
  __shared__ double s_s[kW];
  __shared__ uint64_t s_list[kW][kBeamMax];
  __shared__ Cand s_cand[kW][kBeamMax];
  __shared__ double s_lse[kBeamMax];
  __shared__ int s_last;
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
  uint64_t best = 0;        // the lane's entry of the list; 0: none
  if (finite(a.scores[row])) {
    int skip = 0;           // stop tokens in this part
    for (int i = 0; i < a.n_stop; ++i) skip += a.stops[i] >= lo && a.stops[i] < hi ? 1 : 0;
    float bound = -FLT_MAX;
    int waiting = 0;
    auto flush = [&]() {    // the first 64 that wait go into the list
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      const int n = min(waiting, 64);
      uint64_t v = lane < n ? s_wait[wv][lane] : 0ull;
      const uint64_t rest = s_wait[wv][64 + lane];
      waiting -= n;
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      if (lane < waiting) s_wait[wv][lane] = rest;
      sort64(v, lane, true);
      merge64(best, v, lane);
      const uint32_t nth = __builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), a.N - 1);
      if (nth) bound = fmaxf(bound, key_val(nth));
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
      if (e0 == lo) {
        uint32_t top = ord_key(mx == mx ? mx : -INFINITY);
        sort64(top, lane, false);
        const int n = a.N + skip;
        if (n <= 64) bound = fmaxf(bound, key_val(__builtin_amdgcn_readlane(top, n - 1)));
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
            const int pos = waiting + static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(at >> 32),
                                                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(at), 0u)));
            if (take) s_wait[wv][pos] = comp(ord_key(v[g][k]), static_cast<uint32_t>(e));
            waiting += __popcll(at);
            if (waiting >= 64) flush();
          }
        }
        if (e0 == lo && waiting) flush();
        // what comes in later steps has higher tokens: among equal logits it is behind those of the list
        const uint32_t nth = __builtin_amdgcn_readlane(static_cast<uint32_t>(best >> 32), a.N - 1);
        if (nth) bound = fmaxf(bound, next_up(key_val(nth)));
      }
    }
    if (waiting) flush();
  }
  // the waves' sums and lists as the part's
  z = wave_lse(z);
  if (lane == 0) {
    s_m[wv] = z.m;
    s_s[wv] = static_cast<double>(z.s);
  }
  s_list[wv][lane] = best;
  __syncthreads();
  const int slot = row * a.P + part;
  if (wv == 0) {
    float m = s_m[0];
#pragma unroll
    for (int w = 1; w < kW; ++w) m = fmaxf(m, s_m[w]);
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kW; ++w) s += m == -INFINITY ? s_s[w] : s_s[w] * static_cast<double>(exp_rel(s_m[w], m));
#pragma unroll
    for (int w = 1; w < kW; ++w) merge64(best, s_list[w][63 - lane], lane);
    // hand over through the device's memory: agent-scope stores, completed before the ticket is taken; the part
    // with the group's last ticket reads them with agent-scope loads after an acquire, and clears the ticket
    if (lane < a.N) agent_store(&a.s.key[slot * kBeamMax + lane], static_cast<unsigned long long>(best));
    if (lane == 0) {
      agent_store(&a.s.max[slot], m);
      agent_store(&a.s.sum[slot], s);
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (lane == 0) {
      const unsigned n = __hip_atomic_fetch_add(&a.s.tick[group * kBeamPad], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = static_cast<int>(n) == a.W * a.P - 1;
    }
  }
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  if (tid == 0) agent_store(&a.s.tick[group * kBeamPad], 0u);
  const int first = group * a.W;  // the group's first row

  // lse of each row, its parts side by side in lanes; NaN for a row that is not live
  int S = 1;
  while (S < a.P) S <<= 1;
  for (int i = tid; i < a.W * S + kNt - 1 - (a.W * S - 1) % kNt; i += kNt) {
    const int b = i / S, p = i % S;
    float m = -INFINITY;
    double s = 0.0;
    if (b < a.W && p < a.P) {
      m = agent_load(&a.s.max[(first + b) * a.P + p]);
      s = agent_load(&a.s.sum[(first + b) * a.P + p]);
    }
    float top = m;
    for (int d = S >> 1; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (m != -INFINITY) s *= exp(static_cast<double>(m) - static_cast<double>(top));  // (+inf: NaN)
    for (int d = S >> 1; d; d >>= 1) s += __shfl_xor(s, d);
    if (b < a.W && p == 0) {
      const float sc = a.scores[first + b];
      const double lse = static_cast<double>(top) + log(s);
      s_lse[b] = finite(sc) && __builtin_isfinite(lse) ? lse : NAN;
    }
  }
  __syncthreads();
  auto entry = [&](uint64_t key, int b) {
    const double lse = s_lse[b];
    if (!key || lse != lse) return none();
    return Cand{ord_f64(static_cast<double>(a.scores[first + b]) + (static_cast<double>(comp_val(key)) - lse)), key, static_cast<uint32_t>(b)};
  };
  const int lists = a.W * a.P;
  // the N-th of all lists' first entries (of each thread's best, where there are more lists than threads)
  uint64_t bound;
  {
    uint64_t head = 0;
    for (int l = tid; l < lists; l += kNt) {
      const uint64_t s = entry(agent_load(&a.s.key[(first * a.P + l) * static_cast<long long>(kBeamMax)]), l / a.P).s;
      head = s > head ? s : head;
    }
    sort64(head, lane, false);
    s_list[wv][lane] = head;
    __syncthreads();
    head = s_list[0][lane];
#pragma unroll
    for (int w = 1; w < kW; ++w) merge64(head, s_list[w][63 - lane], lane);
    bound = __shfl(static_cast<unsigned long long>(head), a.N - 1);
    if (!bound) bound = 1;  // fewer lists than that: all with an entry
  }
  Cand c = none();
  for (int l0 = wv * 64; l0 < lists; l0 += kNt) {
    const int l = l0 + lane;
    uint64_t s = 0;
    if (l < lists) s = entry(agent_load(&a.s.key[(first * a.P + l) * static_cast<long long>(kBeamMax)]), l / a.P).s;
    for (unsigned long long todo = __ballot(s >= bound); todo; todo &= todo - 1ull) {
      const int at = l0 + __ffsll(static_cast<long long>(todo)) - 1;
      uint64_t key = 0;
      if (63 - lane < a.N) key = agent_load(&a.s.key[(first * a.P + at) * static_cast<long long>(kBeamMax) + 63 - lane]);
      merge64(c, entry(key, at / a.P), lane);
    }
  }
  s_cand[wv][lane] = c;
  __syncthreads();
  if (wv != 0) return;
#pragma unroll
  for (int w = 1; w < kW; ++w) merge64(c, s_cand[w][63 - lane], lane);
  auto put = [&](int* token, int* parent, float* score, const Cand& c, bool there) {
    if (lane >= a.N) return;
    const long long o = static_cast<long long>(group) * a.N + lane;
    token[o] = there ? comp_idx(c.key) : -1;
    parent[o] = a.row0 + first + (there ? static_cast<int>(c.beam) : lane % a.W);
    score[o] = there ? static_cast<float>(f64_ord(c.s)) : -INFINITY;
  };
  put(a.token, a.parent, a.score, c, c.s != 0);
  if (!a.end_token) return;
  // the stop tokens' continuations, and how many of both kinds come before each
  s_cand[0][lane] = c;
  Cand end = none();
  for (int i0 = 0; i0 < a.W * a.n_stop; i0 += 64) {
    const int i = i0 + lane;
    Cand v = none();
    if (i < a.W * a.n_stop) {
      const int b = i / a.n_stop;
      int t = 0;
      for (int k = 0; k < a.n_stop; ++k) t = k == i % a.n_stop ? a.stops[k] : t;
      const float u = E::get(static_cast<const char*>(a.x) + (first + b) * a.ld * E::kSize, t);
      if (u > -INFINITY) v = entry(comp(ord_key(u), static_cast<uint32_t>(t)), b);
    }
    sort64(v, lane, true);
    merge64(end, v, lane);
  }
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  int rank = lane;
  for (int i = 0; i < a.N; ++i) rank += before(s_cand[0][i], end) ? 1 : 0;
  const bool there = end.s != 0 && rank < a.N;
  put(a.end_token, a.end_parent, a.end_score, end, there);
  const int n = __popcll(__ballot(there));
  if (lane == 0) a.n_end[group] = n;
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
