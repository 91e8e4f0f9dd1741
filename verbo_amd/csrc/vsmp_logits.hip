// Logits adjusted before the pick (k_adjust), and log-probabilities and ranks of given tokens
// (k_logprobs). Both read a row once; rows are cut into parts so that few rows fill the chip.
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

constexpr int kNt = 256;  // threads per workgroup

// ---- loads -------------------------------------------------------------------------------------------

// Rows start where their element type allows, so that a row of a bf16 matrix with an odd number of
// columns may start at any even address: gfx950 takes global loads and stores of any size there. What is
// read once is read with the non-temporal hint.
struct F32 {
  static constexpr int kSize = 4;
  __device__ static float get(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
};
struct Bf16 {
  static constexpr int kSize = 2;
  __device__ static float from(uint32_t h) { return __uint_as_float(h << 16); }
  __device__ static uint32_t bits(float v) { return __float_as_uint(v) >> 16; }
  __device__ static float get(const void* p, long long i) { return from(static_cast<const uint16_t*>(p)[i]); }
};
struct F16 {
  static constexpr int kSize = 2;
  __device__ static float from(uint32_t h) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h))); }
  __device__ static uint32_t bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
  __device__ static float get(const void* p, long long i) { return from(static_cast<const uint16_t*>(p)[i]); }
};

// N consecutive logits from element i on, N * size = 8 or 16 bytes.
template <class E, int N>
struct Raw {
  static constexpr int kWords = N * E::kSize / 4;
  uint32_t w[kWords];
  typedef uint32_t vec __attribute__((ext_vector_type(kWords), aligned(E::kSize)));
  __device__ void load(const void* p, long long i) {
    const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec*>(static_cast<const char*>(p) + i * E::kSize));
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = v[k];
  }
  __device__ void set(const float (&v)[N]) {  // of values that get() gave, or infinities
    if constexpr (E::kSize == 4) {
#pragma unroll
      for (int k = 0; k < N; ++k) w[k] = __float_as_uint(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < N; k += 2) w[k / 2] = E::bits(v[k]) | E::bits(v[k + 1]) << 16;
    }
  }
  __device__ float get(int k) const {
    if constexpr (E::kSize == 4)
      return __uint_as_float(w[k]);
    else
      return E::from(k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xFFFFu);
  }
};

__device__ __forceinline__ int sum64(int v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// ---- k_adjust ------------------------------------------------------------------------------------------

constexpr uint32_t kSeen = 0x80000000u;  // a slot's mark of a prompt id; the bits below count generated ones

// One part of kAdjustParts logits, 16 per thread as four groups of four. The part's histories are
// counted in LDS, a word per logit (integer atomics, so that the order does not matter); the last
// entry that biases a logit is the largest index + 1 in a second array. Each thread's logits are in
// flight while the lists are read. An element without a mark costs its LDS read alone. Logits of four
// that the mask forbids are not read.
//
// Many rows are bound by the logits' read and the output's write: 512 x 128,256 f16 without histories 74 us
// (5.3 TB/s), 256 x 151,936 fp32 53 us (5.8 TB/s), with 512 ids of history a row 55 us. Histories are read by every
// part of their row: 512 x 128,256 f16 with 5,000 ids a row 104 us. Few rows are bound by loads that follow one
// another: mask row, mask words, logits, penalties and offsets, ids, biases. 64 x 151,936 with 40 tokens allowed a
// row 16.0 us, 20.2 where forbidden logits are read too.
template <class E, bool BIAS>
__global__ __launch_bounds__(kNt) void k_adjust(AdjustArgs a) {
  __shared__ __align__(16) uint32_t s_cnt[kAdjustParts];
  __shared__ __align__(16) uint32_t s_bias[BIAS ? kAdjustParts : 4];
  __shared__ int s_left;
  const int tid = threadIdx.x;
  const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.P));
  const int lo = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.P)) * kAdjustParts;
  const int len = min(kAdjustParts, a.V - lo);
  const char* in = static_cast<const char*>(a.in) + (row * a.ldi + lo) * E::kSize;
  float* out = a.out + row * a.ldo + lo;

  uint32_t allow[4] = {0xFu, 0xFu, 0xFu, 0xFu};
  if (a.mask) {
    const int m = a.mask_row ? a.mask_row[row] : row;
    if (m >= 0) {
      const uint32_t* words = a.mask + (m < a.n_masks ? m : 0) * a.ldm + (lo >> 5);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = 4 * (tid + g * kNt);
        allow[g] = m < a.n_masks && e < len ? (words[e >> 5] >> (e & 31)) & 0xFu : 0u;
      }
    }
  }
  Raw<E, 4> x[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int e = 4 * (tid + g * kNt);
    x[g] = {};
    if (e + 4 <= len && allow[g]) x[g].load(in, e);
  }

  const vsmp_penalty pen = a.pen ? a.pen[row] : a.shared;
  int h0 = 0, h1 = 0, hp = 0;  // the window, and where in the history generated ids begin
  if (a.hist && (pen.repeat != 1.0f || pen.presence != 0.0f || pen.frequency != 0.0f)) {
    const int seq = a.slot ? a.slot[row] : row;
    h0 = a.hist_off[seq];
    h1 = a.hist_len ? h0 + a.hist_len[seq] : a.hist_off[seq + 1];
    int window = pen.window;
    if (a.hist_len) {  // what a sequence's region holds beyond its repeat_last depends on when it was cut last
      const int most = a.seq_params[seq].repeat_last;
      if (most > 0 && (window <= 0 || window > most)) window = most;
    }
    hp = h0;
    if (a.prompt_len) hp += min(max(max(a.prompt_len[row], 0) - (a.hist_len ? a.gone[seq] : 0), 0), max(h1 - h0, 0));
    if (window > 0 && h1 - h0 > window) h0 = h1 - window;
  }
  int b0 = 0, b1 = 0;
  if (BIAS) {
    b0 = a.bias_off[row];
    b1 = a.bias_off[row + 1];
  }
  const bool counted = h1 > h0, biased = BIAS && b1 > b0;
  if (counted || biased) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      *reinterpret_cast<uint4*>(&s_cnt[4 * (tid + g * kNt)]) = make_uint4(0u, 0u, 0u, 0u);
      if (BIAS) *reinterpret_cast<uint4*>(&s_bias[4 * (tid + g * kNt)]) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    auto count = [&](uint32_t id, int i) {
      const uint32_t d = id - static_cast<uint32_t>(lo);
      if (d < static_cast<uint32_t>(len)) {
        if (i < hp)
          atomicOr(&s_cnt[d], kSeen);
        else
          atomicAdd(&s_cnt[d], 1u);
      }
    };
    // eight ids a thread in flight; the last few one by one
    int i = h0;
    for (; h1 - i >= 8 * kNt; i += 8 * kNt) {
      typedef uint32_t ids4 __attribute__((ext_vector_type(4), aligned(4)));
      const int i0 = i + 4 * tid, i1 = i0 + 4 * kNt;
      const ids4 u = *reinterpret_cast<const ids4*>(a.hist + i0), w = *reinterpret_cast<const ids4*>(a.hist + i1);
#pragma unroll
      for (int k = 0; k < 4; ++k) count(u[k], i0 + k);
#pragma unroll
      for (int k = 0; k < 4; ++k) count(w[k], i1 + k);
    }
    if (i < h1) {
      uint32_t u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = tid + k * kNt < h1 - i ? static_cast<uint32_t>(a.hist[i + tid + k * kNt]) : 0xFFFFFFFFu;
#pragma unroll
      for (int k = 0; k < 8; ++k) count(u[k], i + tid + k * kNt);
    }
    if (BIAS) {
      for (int i = b0 + tid; i < b1; i += kNt) {
        const unsigned d = static_cast<unsigned>(a.bias_ids[i]) - static_cast<unsigned>(lo);
        if (d < static_cast<unsigned>(len)) atomicMax(&s_bias[d], static_cast<uint32_t>(i - b0) + 1u);
      }
    }
    __syncthreads();
  }

  int left = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int e = 4 * (tid + g * kNt);
    if (e >= len) continue;
    float y[4];
    if (e + 4 <= len) {
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = x[g].get(k);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = e + k < len ? E::get(in, e + k) : -INFINITY;
    }
    if (!allow[g]) y[0] = y[1] = y[2] = y[3] = -INFINITY;
    uint4 c = make_uint4(0u, 0u, 0u, 0u), b = c;
    if (counted) c = *reinterpret_cast<const uint4*>(&s_cnt[e]);
    if (biased) b = *reinterpret_cast<const uint4*>(&s_bias[e]);
    if (c.x | c.y | c.z | c.w | b.x | b.y | b.z | b.w) {
      const uint32_t cs[4] = {c.x, c.y, c.z, c.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma clang fp contract(off)
        float v = y[k];
        if (cs[k]) v = v > 0.0f ? v / pen.repeat : v * pen.repeat;  // the reference's rule (src/sampler.cpp:63)
        const uint32_t n = cs[k] & ~kSeen;
        if (n) v = v - (pen.presence + pen.frequency * static_cast<float>(n));
        if (bs[k]) v = v + a.bias[b0 + static_cast<int>(bs[k]) - 1];
        y[k] = y[k] == -INFINITY ? y[k] : v;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[k] = allow[g] >> k & 1u ? y[k] : -INFINITY;
      left += y[k] > -INFINITY ? 1 : 0;
    }
    if (e + 4 <= len) {
      __builtin_memcpy(out + e, y, sizeof y);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k < len) out[e + k] = y[k];
    }
  }
  if (!a.acc) return;
  if (tid == 0) s_left = 0;
  __syncthreads();
  left = sum64(left);
  if ((tid & 63) == 0) atomicAdd(&s_left, left);
  __syncthreads();
  if (tid == 0) {
    // the ticket and the count in one word: the part that takes the last ticket has every part's count
    const unsigned long long old = __hip_atomic_fetch_add(&a.acc[row * (kOpPad / 2)], (1ull << 32) | static_cast<unsigned>(s_left),
                                                          __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (static_cast<int>(old >> 32) == a.P - 1) {
      a.left[row] = static_cast<int>(old & 0xFFFFFFFFu) + s_left;
      __hip_atomic_store(&a.acc[row * (kOpPad / 2)], 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// ---- k_logprobs ------------------------------------------------------------------------------------------

constexpr float kLog2e = 1.44269504088896340736f;

// exp(x - m) for x <= m: 1 at x = m, 0 at x = -inf. m finite.
__device__ __forceinline__ float exp_rel(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }

// A maximum and the sum of exp(x - maximum): the log of the sum of exponentials in one pass. The maximum of
// nothing is -inf, with a sum of 0. NaN among the x is left out of the maximum and makes the sum NaN, also where
// the maximum is -inf; so does a maximum of +inf.
struct Lse {
  float m, s;
  // The sum relative to a maximum t >= m (a sum at m = -inf is 0 or NaN, whatever it is relative to).
  __device__ float at(float t) const { return m == -INFINITY ? s : s * exp_rel(m, t); }
};
__device__ __forceinline__ unsigned long long pack_lse(const Lse& z) {
  return static_cast<unsigned long long>(__float_as_uint(z.m)) << 32 | __float_as_uint(z.s);
}
__device__ __forceinline__ Lse unpack_lse(unsigned long long w) {
  return {__uint_as_float(static_cast<uint32_t>(w >> 32)), __uint_as_float(static_cast<uint32_t>(w))};
}

__device__ __forceinline__ float lane_f32(float v, int l) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l));
}
// Reductions over a wave with the same result in every lane, all lanes taking part: within rows of 16 lanes by
// rotation, then over the four rows.
template <int N>
__device__ __forceinline__ uint32_t ror(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0u, v, 0x120 + N, 0xF, 0xF, false);
}
template <int N>
__device__ __forceinline__ float ror(float v) {
  return __uint_as_float(ror<N>(__float_as_uint(v)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, ror<8>(v));
  v = fmaxf(v, ror<4>(v));
  v = fmaxf(v, ror<2>(v));
  v = fmaxf(v, ror<1>(v));
  return fmaxf(fmaxf(lane_f32(v, 0), lane_f32(v, 16)), fmaxf(lane_f32(v, 32), lane_f32(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += ror<8>(v);
  v += ror<4>(v);
  v += ror<2>(v);
  v += ror<1>(v);
  return (lane_f32(v, 0) + lane_f32(v, 16)) + (lane_f32(v, 32) + lane_f32(v, 48));
}
__device__ __forceinline__ int wave_sum(int i) {
  uint32_t v = static_cast<uint32_t>(i);
  v += ror<8>(v);
  v += ror<4>(v);
  v += ror<2>(v);
  v += ror<1>(v);
  return static_cast<int>(__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
                          __builtin_amdgcn_readlane(v, 48));
}
__device__ __forceinline__ Lse wave_lse(const Lse& z) {
  const float m = wave_max(z.m);
  return {m, wave_sum(z.at(m))};
}

// The least float above v (finite or -inf; zeros of either sign have the same).
__device__ __forceinline__ float next_up(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return __uint_as_float((b << 1) == 0u ? 1u : (b >> 31 ? b - 1u : b + 1u));
}

// One part of a row, a step of four 16-byte groups per thread at a time, the next step's in flight while one
// is summed. Bound by the logits' read where there are many: 2,048 x 128,256 bf16 84 us without ids (6.3 TB/s), 83 to
// 96 us with one id a row (the likeliest, any); few rows by latencies and the parts' hand-off: one row of 151,936 fp32
// 4.2 us, with its 20 likeliest ids 6.8.
//
// Ranks: a wave keeps the asked ids' logits one in a lane and counts, per step, the logits before each. Only ids
// that the step's largest logit reaches can gain, and the ids that are asked for are mostly the likeliest, so
// that few steps do more than find that out. The step's few largest logits (those that reach the least of the
// four rows' maxima) are listed in LDS and compared one by one with all ids above that line at once; the ids
// below it are taken one by one, each compared with all of the step's logits. The latter takes one comparison
// and one addition per logit: where ties do not matter, v >= t before the id and v >= the next float above t
// after it. They matter in the id's own group, whose equal logits before the id the id's lane counts first. An id
// that is not among the likeliest so costs a pass over nearly every step: 21 ids anywhere in 2,048 x 128,256 517 us, the
// 20 likeliest 97.
template <class E>
__global__ __launch_bounds__(kNt) void k_logprobs(LogprobArgs a) {
  constexpr int N = 16 / E::kSize, G = 4;  // elements per group, groups per step
  constexpr int kStep = kNt * N * G, kW = kNt / 64;
  constexpr int kList = 128, kLanes = 16;  // listed logits of a step and wave, and lanes they may come from
  __shared__ float s_m[kW], s_s[kW];
  __shared__ int s_cnt[kW][kOpIds];
  __shared__ uint2 s_list[kW][kList];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.P));
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.P));
  const int lo = part * a.L, hi = min(a.V, lo + a.L);
  const char* x = static_cast<const char*>(a.x) + row * a.ld * E::kSize;

  int id = -1;
  if (lane < a.n) id = a.ids[row * a.ldj + lane];
  Raw<E, N> r[G];
  auto load_group = [&](Raw<E, N>& d, int e, int end) {
    if (e + N <= end) {
      d.load(x, e);
    } else {  // the row's end: its last elements one by one, then -inf
      float v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = e + k < end ? E::get(x, e + k) : -INFINITY;
      d.set(v);
    }
  };
  auto load = [&](int e0) {
#pragma unroll
    for (int g = 0; g < G; ++g) load_group(r[g], e0 + N * (tid + g * kNt), hi);
  };
  load(lo);
  if (id < 0 || id >= a.V) id = -1;
  Raw<E, N> d;  // the id's own group
  if (id >= 0) load_group(d, id & ~(N - 1), a.V);
  float t = NAN, tup = NAN;  // the id's logit and the next float above it; NaN where the lane has no id
  int cnt = 0;  // logits before the lane's id, as far as this wave has counted them
  int own = 0;  // equal ones before it in its own group
  auto take_ids = [&]() {
    if (id < 0) return;
    t = d.get(0);
#pragma unroll
    for (int k = 1; k < N; ++k) t = k == (id & (N - 1)) ? d.get(k) : t;
#pragma unroll
    for (int k = 0; k < N - 1; ++k) own += k < (id & (N - 1)) && d.get(k) == t ? 1 : 0;
    tup = next_up(t);
  };

  Lse z{-INFINITY, 0.0f};
  int low = 0, acc = 0;  // the id that was last taken by itself, and the lane's count of logits before it
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
    // After the first step's sums, which do not wait for the ids' logits. (Those logits' loads do wait for the first
    // step's: the row's end makes the latter conditional, and a wait for the ids cannot count past them; in fp32 the
    // compiled code waits for each of the four in its branch.)
    if (e0 == lo) take_ids();
    if (!a.rank) continue;
    float rm = mx;  // the largest of each row of 16 lanes
    rm = fmaxf(rm, ror<8>(rm));
    rm = fmaxf(rm, ror<4>(rm));
    rm = fmaxf(rm, ror<2>(rm));
    rm = fmaxf(rm, ror<1>(rm));
    const float r0 = lane_f32(rm, 0), r1 = lane_f32(rm, 16), r2 = lane_f32(rm, 32), r3 = lane_f32(rm, 48);
    unsigned long long todo = __ballot(t <= fmaxf(fmaxf(r0, r1), fmaxf(r2, r3)));
    if (!todo) continue;
    const float few = fminf(fminf(r0, r1), fminf(r2, r3));
    const unsigned long long high = __ballot(t >= few) & todo;
    if (high && __popcll(__ballot(mx >= few)) <= kLanes) {
      int n = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (!__ballot(gm[g] >= few)) continue;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const unsigned long long at = __ballot(v[g][k] >= few);
          if (!at) continue;
          const int pos = n + static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(at >> 32),
                                                                         __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(at), 0u)));
          if (v[g][k] >= few && pos < kList)
            s_list[wv][pos] = make_uint2(__float_as_uint(v[g][k]), static_cast<uint32_t>(e0 + N * (tid + g * kNt) + k));
          n += __popcll(at);
        }
      }
      if (n <= kList) {
        todo &= ~high;
        const float th = t >= few ? t : NAN;  // the other ids gain nothing here, not from a +inf either
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        for (int i = 0; i < n; i += 4) {
          uint2 c[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) c[u] = s_list[wv][min(i + u, n - 1)];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float w = i + u < n ? __uint_as_float(c[u].x) : -INFINITY;
            // its own group's equal logits are in `own`
            const int e = static_cast<int>(c[u].y);
            cnt += w > th || (w == th && e < (id & ~(N - 1)) && i + u < n) ? 1 : 0;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      }
    }
    for (; todo; todo &= todo - 1ull) {
      const int j = __ffsll(static_cast<long long>(todo)) - 1;
      if (j != low) {  // the sum over the lanes waits until another id's turn
        const int sum = wave_sum(acc);
        if (lane == low) cnt += sum;
        low = j;
        acc = 0;
      }
      const float tj = lane_f32(t, j), uj = lane_f32(tup, j);
      const int ij = __builtin_amdgcn_readlane(id, j);
      int c[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float b = e0 + N * (tid + g * kNt) + N <= ij ? tj : uj;
        c[g] = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) c[g] += v[g][k] >= b ? 1 : 0;
      }
      acc += (c[0] + c[1]) + (c[2] + c[3]);
    }
  }
  if (a.rank) {
    const int sum = wave_sum(acc);
    if (lane == low) cnt += sum;
  }
  z = wave_lse(z);
  if (lane == 0) {
    s_m[wv] = z.m;
    s_s[wv] = z.s;
  }
  s_cnt[wv][lane] = cnt;
  __syncthreads();
  if (wv != 0) return;
  z = wave_lse(lane < kW ? Lse{s_m[lane], s_s[lane]} : Lse{-INFINITY, 0.0f});
  cnt = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) cnt += s_cnt[w][lane];

  if (a.P > 1) {
    // hand over through the device's memory: agent-scope stores, completed before the ticket is taken; the
    // part with the last ticket reads them with agent-scope loads after an acquire, and clears the ticket
    const int slot = row * a.P + part;
    if (lane == 0)
      __hip_atomic_store(&a.s.part[slot], pack_lse(z), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.rank && lane < a.n) __hip_atomic_store(&a.s.count[slot * a.n + lane], cnt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    unsigned n = 0u;
    if (lane == 0) n = __hip_atomic_fetch_add(&a.s.tick[row * kOpPad], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (static_cast<int>(__builtin_amdgcn_readfirstlane(n)) != a.P - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (lane == 0) __hip_atomic_store(&a.s.tick[row * kOpPad], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    z = {-INFINITY, 0.0f};
    if (lane < a.P)
      z = unpack_lse(__hip_atomic_load(&a.s.part[row * a.P + lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    if (a.rank) {  // the parts' counts lie one after the other: every lane adds some of them up
      s_cnt[0][lane] = 0;
      const int total = a.P * a.n;
      constexpr int kAhead = 8;
      for (int i0 = lane; i0 < total; i0 += 64 * kAhead) {
        int c[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          c[u] = i0 + 64 * u < total ? __hip_atomic_load(&a.s.count[row * total + i0 + 64 * u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (c[u]) atomicAdd(&s_cnt[0][(i0 + 64 * u) % a.n], c[u]);
      }
      cnt = s_cnt[0][lane];
    }
    z = wave_lse(z);
  }
  const float ls = logf(z.s);  // of a sum in [1, V]; -inf for a row of -inf alone; NaN
  if (lane < a.n) {
    const long long o = static_cast<long long>(row) * a.n + lane;
    a.logprob[o] = id < 0 ? -INFINITY : (z.m == -INFINITY ? ls : (t - z.m) - ls);
    if (a.rank) a.rank[o] = id >= 0 ? cnt + own : -1;
  }
  if (lane == 0 && a.lse) a.lse[row] = z.m + ls;
}

}  // namespace

void launch_adjust(const AdjustArgs& a, int dtype, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.B) * static_cast<unsigned>(a.P));
  auto go = [&](auto e) {
    using E = decltype(e);
    if (a.bias_off)
      hipLaunchKernelGGL((k_adjust<E, true>), grid, dim3(kNt), 0, st, a);
    else
      hipLaunchKernelGGL((k_adjust<E, false>), grid, dim3(kNt), 0, st, a);
  };
  if (dtype == VSMP_F32)
    go(F32{});
  else if (dtype == VSMP_BF16)
    go(Bf16{});
  else
    go(F16{});
}

// Workgroups of four a CU, each of at least one step (a whole number of steps, so that every part but a row's
// last reads whole groups), at most 64 parts a row (a lane each reads their results). Measured for one and five
// ids against one, two and eight a CU: 32 x 151,936 fp32 8.9 / 9.6 us, against 10.0 / 11.0, 9.1 / 10.3, 8.7 / 9.1;
// 128 x 50,257 fp32 9.7 / 10.4 against 12.2 / 13.8, 9.8 / 10.7, 12.0 / 12.8; 1,024 x 49,152 bf16 20.6 / 22.4 against
// 20.5 / 23.0, 20.4 / 21.2, 24.7 / 27.0. Workgroups of 512 threads measured the same, of 1,024 slower from 300 rows on.
void logprob_parts(int B, int V, int dtype, int cus, int* P, int* L) {
  const int step = kNt * 4 * (dtype == VSMP_F32 ? 4 : 8);
  const int steps = (V + step - 1) / step;
  int p = (4 * cus + B - 1) / B;
  if (p > steps) p = steps;
  if (p > 64) p = 64;  // a lane each reads their results
  if (p > kOpSlots / B) p = kOpSlots / B;
  if (p < 1) p = 1;
  *L = (steps + p - 1) / p * step;
  *P = (V + *L - 1) / *L;
}

void launch_logprobs(const LogprobArgs& a, int dtype, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.B) * static_cast<unsigned>(a.P));
  if (dtype == VSMP_F32)
    hipLaunchKernelGGL(k_logprobs<F32>, grid, dim3(kNt), 0, st, a);
  else if (dtype == VSMP_BF16)
    hipLaunchKernelGGL(k_logprobs<Bf16>, grid, dim3(kNt), 0, st, a);
  else
    hipLaunchKernelGGL(k_logprobs<F16>, grid, dim3(kNt), 0, st, a);
}

}  // namespace vsmp
