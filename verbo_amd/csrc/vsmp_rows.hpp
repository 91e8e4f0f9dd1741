// Rows of logits of any type, one pass over them, and reductions over a wave: device code shared by the
// operators around the pick and by beams.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vsmp {

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

}  // namespace vsmp
