// Logits adjusted before the pick (k_adjust), and log-probabilities and ranks of given tokens
// (k_logprobs). Both read a row once; rows are cut into parts so that few rows fill the chip.
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

constexpr int kNt = 256;  // threads per workgroup

// ---- loads -------------------------------------------------------------------------------------------

// Rows start where their element type allows, so that a row of a bf16 matrix with an odd number of
// columns may start at any even address: gfx950 takes global loads and stores of any size there.
template <class T>
__device__ __forceinline__ T load_any(const void* p) {
  T v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}

struct F32 {
  static constexpr int kSize = 4;
  __device__ static float get(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
};
struct Bf16 {
  static constexpr int kSize = 2;
  __device__ static float from(uint32_t h) { return __uint_as_float(h << 16); }
  __device__ static float get(const void* p, long long i) { return from(static_cast<const uint16_t*>(p)[i]); }
};
struct F16 {
  static constexpr int kSize = 2;
  __device__ static float from(uint32_t h) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h))); }
  __device__ static float get(const void* p, long long i) { return from(static_cast<const uint16_t*>(p)[i]); }
};

// N consecutive logits from element i on, N * size = 8 or 16 bytes.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <class E, int N>
struct Raw {
  static constexpr int kWords = N * E::kSize / 4;
  uint32_t w[kWords];
  __device__ void load(const void* p, long long i) {
    __builtin_memcpy(w, static_cast<const char*>(p) + i * E::kSize, sizeof w);
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
// flight while the lists are read. An element without a mark costs its LDS read alone.
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

  Raw<E, 4> x[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int e = 4 * (tid + g * kNt);
    if (e + 4 <= len) x[g].load(in, e);
  }
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

  const vsmp_penalty pen = a.pen ? a.pen[row] : a.shared;
  int h0 = 0, h1 = 0, hp = 0;  // the window, and where in the history generated ids begin
  if (a.hist && (pen.repeat != 1.0f || pen.presence != 0.0f || pen.frequency != 0.0f)) {
    const int seq = a.slot ? a.slot[row] : row;
    h0 = a.hist_off[seq];
    h1 = a.hist_len ? h0 + a.hist_len[seq] : a.hist_off[seq + 1];
    hp = h0 + (a.prompt_len ? a.prompt_len[row] : 0);
    if (pen.window > 0 && h1 - h0 > pen.window) h0 = h1 - pen.window;
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
    for (int i = h0 + tid; i < h1; i += kNt) {
      const unsigned d = static_cast<unsigned>(a.hist[i]) - static_cast<unsigned>(lo);
      if (d < static_cast<unsigned>(len)) {
        if (i < hp)
          atomicOr(&s_cnt[d], kSeen);
        else
          atomicAdd(&s_cnt[d], 1u);
      }
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
    const unsigned long long old = __hip_atomic_fetch_add(&a.acc[row], (1ull << 32) | static_cast<unsigned>(s_left),
                                                          __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (static_cast<int>(old >> 32) == a.P - 1) {
      a.left[row] = static_cast<int>(old & 0xFFFFFFFFu) + s_left;
      __hip_atomic_store(&a.acc[row], 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// ---- k_logprobs ------------------------------------------------------------------------------------------

constexpr float kLog2e = 1.44269504088896340736f;

// exp(x - m) for x <= m: 1 at x = m, 0 at x = -inf. m finite.
__device__ __forceinline__ float exp_rel(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }

// A running maximum and the sum of exp(x - maximum): log of the sum of exponentials in one pass. The
// maximum of nothing is -inf, with a sum of 0.
struct Lse {
  float m, s;
  __device__ void join(float om, float os) {
    const float t = fmaxf(m, om);
    if (t == -INFINITY) return;
    s = s * exp_rel(m, t) + os * exp_rel(om, t);
    m = t;
  }
};

// One part of a row: NV logits a step and thread in 16-byte groups. A wave keeps the asked ids' logits
// one in a lane, and compares a step with one of them only where the step's largest value reaches it:
// the ids that are asked for are mostly the likeliest, which few logits come before.
template <class E>
__global__ __launch_bounds__(kNt) void k_logprobs(LogprobArgs a) {
  constexpr int N = 16 / E::kSize, G = 4;  // elements per group, groups per step
  __shared__ float s_m[kNt / 64], s_s[kNt / 64];
  __shared__ int s_cnt[kOpIds];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.P));
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.P));
  const int lo = part * a.L, hi = min(a.V, lo + a.L);
  const char* x = static_cast<const char*>(a.x) + row * a.ld * E::kSize;

  int id = -1;
  float t = INFINITY;
  if (lane < a.n) {
    id = a.ids[row * a.ldj + lane];
    if (id < 0 || id >= a.V) id = -1;
    if (id >= 0) t = E::get(x, id);
  }
  if (tid < kOpIds) s_cnt[tid] = 0;
  __syncthreads();

  Lse z{-INFINITY, 0.0f};
  int cnt = 0;  // of the lane's id
  for (int e0 = lo; e0 < hi; e0 += kNt * N * G) {
    Raw<E, N> r[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int e = e0 + N * (tid + g * kNt);
      if (e + N <= hi) r[g].load(x, e);
    }
    float v[G][N];
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int e = e0 + N * (tid + g * kNt);
      if (e + N <= hi) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[g][k] = r[g].get(k);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[g][k] = e + k < hi ? E::get(x, e + k) : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) mx = fmaxf(mx, v[g][k]);
    }
    const float m = fmaxf(z.m, mx);
    if (m != -INFINITY) {
      float s = z.s * exp_rel(z.m, m);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < N; ++k) s += exp_rel(v[g][k], m);
      z = {m, s};
    }
    if (a.rank) {
      float wm = mx;
#pragma unroll
      for (int d = 32; d; d >>= 1) wm = fmaxf(wm, __shfl_xor(wm, d));
      for (unsigned long long todo = __ballot(id >= 0 && wm >= t); todo; todo &= todo - 1ull) {
        const int j = __ffsll(static_cast<long long>(todo)) - 1;
        const float tj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(t), j));
        const int ij = __builtin_amdgcn_readlane(id, j);
        int c = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int e = e0 + N * (tid + g * kNt);
#pragma unroll
          for (int k = 0; k < N; ++k) c += (v[g][k] > tj || (v[g][k] == tj && e + k < ij && e + k < hi)) ? 1 : 0;
        }
        c = sum64(c);
        if (lane == j) cnt += c;
      }
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) z.join(__shfl_xor(z.m, d), __shfl_xor(z.s, d));
  if (lane == 0) {
    s_m[wv] = z.m;
    s_s[wv] = z.s;
  }
  if (lane < a.n && cnt) atomicAdd(&s_cnt[lane], cnt);
  __syncthreads();
  if (wv != 0) return;
  z = {s_m[0], s_s[0]};
#pragma unroll
  for (int w = 1; w < kNt / 64; ++w) z.join(s_m[w], s_s[w]);
  cnt = s_cnt[lane];

  if (a.P > 1) {
    // hand over through the device's memory: agent-scope stores, completed before the ticket is taken;
    // the part with the last ticket reads them with agent-scope loads after an acquire
    const int slot = row * a.P + part;
    if (lane == 0) {
      __hip_atomic_store(&a.s.part[2 * slot], z.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&a.s.part[2 * slot + 1], z.s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (lane < a.n) __hip_atomic_store(&a.s.count[slot * kOpIds + lane], cnt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    unsigned n = 0u;
    if (lane == 0) n = __hip_atomic_fetch_add(&a.s.tick[row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (static_cast<int>(__builtin_amdgcn_readfirstlane(n)) != a.P - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (lane == 0) __hip_atomic_store(&a.s.tick[row], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    z = {-INFINITY, 0.0f};
    cnt = 0;
    for (int p = lane; p < a.P; p += 64) {
      const int o = row * a.P + p;
      z.join(__hip_atomic_load(&a.s.part[2 * o], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
             __hip_atomic_load(&a.s.part[2 * o + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) z.join(__shfl_xor(z.m, d), __shfl_xor(z.s, d));
    if (a.rank && lane < a.n)
      for (int p = 0; p < a.P; ++p)
        cnt += __hip_atomic_load(&a.s.count[(row * a.P + p) * kOpIds + lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // the lanes joined the parts in different orders: one of them for all, so that equal logits have equal
  // log-probabilities
  z.m = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(z.m)));
  z.s = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(z.s)));
  const float ls = logf(z.s);  // of a sum in [1, V]
  if (lane < a.n) {
    const long long o = static_cast<long long>(row) * a.n + lane;
    a.logprob[o] = id >= 0 && t != -INFINITY ? (t - z.m) - ls : -INFINITY;
    if (a.rank) a.rank[o] = id >= 0 ? cnt : -1;
  }
  if (lane == 0 && a.lse) a.lse[row] = z.m == -INFINITY ? -INFINITY : z.m + ls;
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

// Enough workgroups for four per CU, each of at least one step (a whole number of steps, so that every
// part but a row's last reads whole groups).
void logprob_parts(int B, int V, int dtype, int cus, int* P, int* L) {
  const int step = kNt * 4 * (dtype == VSMP_F32 ? 4 : 8);
  const int steps = (V + step - 1) / step;
  int p = (4 * cus + B - 1) / B;
  if (p > steps) p = steps;
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
