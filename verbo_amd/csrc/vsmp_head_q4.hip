// The LM head's product with 4-bit weights (k_head_q4): logits = x . (s (q - z))^T.
//
// A weight enters the matrix cores unrounded. A nibble q moved to the top of a 16-bit float's mantissa
// under the exponent of 16 is the number 16 + q (bf16: bits 3-6, f16: bits 6-9), two shifts and masks
// for two weights. With o = 16 + z,
//   sum_{d in g} x_d (q_d - z) = sum_{d in g} x_d (16 + q_d) - o X_g,   X_g = sum_{d in g} x_d,
// so the group's MFMAs start from -o X_g and the group's result is scaled and added in fp32:
//   acc += s_g P_g.
// The intermediate sums are at most some 31 / 8 of those of the centred weights, which costs one to two
// bits of the fp32 accumulation.
//
// Tiles: a workgroup of four waves takes MB x 16 rows and 128 columns, each wave two strips of 16
// columns on v_mfma_f32_16x16x32. Weights go from HBM to registers, 16 bytes a lane: lane (column c,
// quarter h) holds the 32 weights [32 h, 32 h + 32) of a block of 128 of its column, each chunk of KC
// loaded while the one before is multiplied. An MFMA sums over the four quarters, so for groups of 32
// (64) the quarters' dwords are transposed between lanes 16 and 32 apart (32 apart) with the lane
// swaps, until an MFMA's four quarters lie in one group. x and the scales go through LDS, staged per
// chunk in two buffers; x in the order in which the nibbles of a dword come out: 0 4 1 5 2 6 3 7.
#include "vsmp_lds.hpp"
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kQNt = 256;  // threads per workgroup
constexpr int kQNs = 2;    // strips of 16 columns per wave
constexpr int kQBn = kQNt / 64 * 16 * kQNs;

// Eight weights of a dword as 16 + q, in the order 0 4 1 5 2 6 3 7.
template <bool H>
__device__ __forceinline__ u32x4 widen(uint32_t w) {
  constexpr uint32_t one = H ? 0x4C004C00u : 0x41804180u, mask = H ? 0x03C003C0u : 0x00780078u;
  u32x4 r;
  if constexpr (H) {
    r.x = ((w << 6) & mask) | one;
    r.y = ((w << 2) & mask) | one;
    r.z = ((w >> 2) & mask) | one;
    r.w = ((w >> 6) & mask) | one;
  } else {
    r.x = ((w << 3) & mask) | one;
    r.y = ((w >> 1) & mask) | one;
    r.z = ((w >> 5) & mask) | one;
    r.w = ((w >> 9) & mask) | one;
  }
  return r;
}

template <bool H>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool H>
__device__ __forceinline__ float half_val(uint32_t h) {
  if constexpr (H)
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
  else
    return __uint_as_float(h << 16);
}

__device__ __forceinline__ float scale_at(const void* p, int type, long long i) {
  if (type == VSMP_F32) return static_cast<const float*>(p)[i];
  const uint32_t h = static_cast<const uint16_t*>(p)[i];
  return type == VSMP_BF16 ? half_val<false>(h) : half_val<true>(h);
}

// Rows of 16 lanes r0..r3 of a and s0..s3 of b: a = (r0 r1 s0 s1), b = (r2 r3 s2 s3).
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
// a = (r0 s0 r2 s2), b = (r1 s1 r3 s3).
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

// H: f16 hidden states (else bf16). G: group. MB: blocks of 16 rows. ZP: zero points given. KC: hidden
// elements per chunk.
template <bool H, int G, int MB, bool ZP, int KC>
__global__ __launch_bounds__(kQNt) void k_head_q4(HeadQ4Args a, int rows_ld) {
  constexpr int kStr = KC + 8;        // halfwords per x row in LDS: 16 rows' reads fall on distinct banks
  constexpr int kBlk = KC / 128;      // blocks of 128 per chunk
  constexpr int kGc = KC / G;         // groups per chunk
  constexpr int kGb = 128 / G;        // groups per block
  constexpr int kPr = KC / 8;         // 16-byte pieces of an x row per chunk
  constexpr int kQx = MB * 16 * kPr / kQNt;
  constexpr int kQs = kQBn * kGc / kQNt;
  constexpr int kSteps = G / 32;      // MFMAs per group

  extern __shared__ __align__(16) unsigned char lds[];
  // two stages of: x [rows_ld][kStr], X [kGc][MB * 16], scales [kBlk][kQBn][kGb], offsets the same
  const int xbytes = rows_ld * kStr * 2;
  constexpr int kXsBytes = kGc * MB * 16 * 4, kScBytes = kQBn * kGc * 4;
  const int stage = xbytes + kXsBytes + kScBytes * (ZP ? 2 : 1);
  auto sx = [&](int b) { return reinterpret_cast<uint16_t*>(lds + b * stage); };
  auto sX = [&](int b) { return reinterpret_cast<float*>(lds + b * stage + xbytes); };
  auto sS = [&](int b) { return reinterpret_cast<float*>(lds + b * stage + xbytes + kXsBytes); };
  auto sO = [&](int b) { return reinterpret_cast<float*>(lds + b * stage + xbytes + kXsBytes + kScBytes); };

  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, c16 = lane & 15, h = lane >> 4;
  const int m0 = blockIdx.y * (MB * 16), rows = min(rows_ld, a.B - m0);
  const int n0 = blockIdx.x * kQBn;
  const uint16_t* x = a.x + m0 * a.ldx;
  const int D = a.D, nch = (D + KC - 1) / KC, groups = D / G;

  // where the lane's pieces come from
  const uint8_t* wq[kQNs];
#pragma unroll
  for (int s = 0; s < kQNs; ++s) wq[s] = a.q + min(n0 + (wv * kQNs + s) * 16 + c16, a.V - 1) * a.ldq;

  u32x4 w[kQNs][kBlk];
  auto load_w = [&](int c, int s, int b) {
    const int byte = min(c * (KC / 2) + b * 64 + h * 16, D / 2 - 16);
    w[s][b] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wq[s] + byte));
  };
  u32x4 px[kQx];
  float ps[kQs], pz[ZP ? kQs : 1];
  auto load_xs = [&](int c) {
#pragma unroll
    for (int q = 0; q < kQx; ++q) {
      const int p = tid + q * kQNt, r = p / kPr, k = c * KC + 8 * (p % kPr);
      px[q] = u32x4{0u, 0u, 0u, 0u};
      if (r < rows && k < D) px[q] = *reinterpret_cast<const u32x4*>(x + r * a.ldx + k);
    }
#pragma unroll
    for (int q = 0; q < kQs; ++q) {
      const int i = tid + q * kQNt, g = min(c * kGc + i % kGc, groups - 1);
      const long long col = min(n0 + i / kGc, a.V - 1);
      ps[q] = scale_at(a.sc, a.sc_type, col * a.lds + g);
      if (ZP) pz[q] = static_cast<float>(a.z[col * a.ldz + g]);
    }
  };
  auto store_xs = [&](int b) {
#pragma unroll
    for (int q = 0; q < kQx; ++q) {
      const int p = tid + q * kQNt, r = p / kPr, k8 = p % kPr;
      const u32x4 v = px[q];
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += half_val<H>(v[j] & 0xFFFFu) + half_val<H>(v[j] >> 16);
#pragma unroll
      for (int d = 1; d < G / 8; d <<= 1) s += __shfl_xor(s, d);
      if (r < rows) {
        u32x4 o;
        o.x = (v.x & 0xFFFFu) | (v.z << 16);
        o.y = (v.x >> 16) | (v.z & 0xFFFF0000u);
        o.z = (v.y & 0xFFFFu) | (v.w << 16);
        o.w = (v.y >> 16) | (v.w & 0xFFFF0000u);
        *reinterpret_cast<u32x4*>(&sx(b)[r * kStr + 8 * k8]) = o;
        if (k8 % (G / 8) == 0) sX(b)[k8 / (G / 8) * (MB * 16) + r] = ZP ? s : -24.0f * s;
      }
    }
#pragma unroll
    for (int q = 0; q < kQs; ++q) {
      const int i = tid + q * kQNt, g = i % kGc, col = i / kGc;
      const int at = (g / kGb * kQBn + col) * kGb + g % kGb;
      sS(b)[at] = ps[q];
      if (ZP) sO(b)[at] = -16.0f - pz[q];
    }
  };

  f32x4 acc[kQNs][MB];
#pragma unroll
  for (int s = 0; s < kQNs; ++s)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[s][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // the lane's x row and its offset in a block: k of step t is (t's) + kl
  int xa[MB];
  const int kl = G == 32 ? 8 * h : (G == 64 ? 32 * (h & 1) + 16 * (h >> 1) : 32 * h);
#pragma unroll
  for (int i = 0; i < MB; ++i) xa[i] = min(16 * i + c16, rows - 1) * kStr + kl;

  auto block = [&](int buf, int b, auto reload) {
    uint32_t t[kQNs][4];
    float sc[kQNs][kGb], of[kQNs][kGb];
#pragma unroll
    for (int s = 0; s < kQNs; ++s) {
      t[s][0] = w[s][b].x, t[s][1] = w[s][b].y, t[s][2] = w[s][b].z, t[s][3] = w[s][b].w;
      reload(s);
      if constexpr (G <= 64) {
        swap32(t[s][0], t[s][2]);
        swap32(t[s][1], t[s][3]);
      }
      if constexpr (G == 32) {
        swap16(t[s][0], t[s][1]);
        swap16(t[s][2], t[s][3]);
      }
      const int col = (wv * kQNs + s) * 16 + c16;
#pragma unroll
      for (int g = 0; g < kGb; ++g) {
        sc[s][g] = sS(buf)[(b * kQBn + col) * kGb + g];
        of[s][g] = ZP ? sO(buf)[(b * kQBn + col) * kGb + g] : 0.0f;
      }
    }
#pragma unroll
    for (int g = 0; g < kGb; ++g) {
      f32x4 X[MB], P[kQNs][MB];
#pragma unroll
      for (int i = 0; i < MB; ++i)
        X[i] = *reinterpret_cast<const f32x4*>(&sX(buf)[(b * kGb + g) * (MB * 16) + 16 * i + 4 * h]);
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int step = g * kSteps + u;
        const int k = b * 128 + (G == 32 ? 32 * step : (G == 64 ? 64 * g + 8 * u : 8 * step));
        u32x4 A[MB];
#pragma unroll
        for (int i = 0; i < MB; ++i) A[i] = *reinterpret_cast<const u32x4*>(&sx(buf)[xa[i] + k]);
#pragma unroll
        for (int s = 0; s < kQNs; ++s) {
          const u32x4 wb = widen<H>(t[s][step]);
#pragma unroll
          for (int i = 0; i < MB; ++i) {
            f32x4 c = u ? P[s][i] : X[i];
            if (ZP && u == 0) {
#pragma unroll
              for (int r = 0; r < 4; ++r) c[r] *= of[s][g];
            }
            P[s][i] = mfma<H>(A[i], wb, c);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < kQNs; ++s)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[s][i][r] = __builtin_fmaf(sc[s][g], P[s][i][r], acc[s][i][r]);
    }
  };

#pragma unroll
  for (int b = 0; b < kBlk; ++b)
#pragma unroll
    for (int s = 0; s < kQNs; ++s) load_w(0, s, b);
  load_xs(0);
  store_xs(0);
  if (nch > 1) load_xs(1);
  for (int c = 0; c < nch; ++c) {
    __syncthreads();  // chunk c's stage is written, chunk c - 1's no longer read
#pragma unroll
    for (int b = 0; b < kBlk; ++b)
      if (c * KC + b * 128 < D) block(c & 1, b, [&](int s) { if (c + 1 < nch) load_w(c + 1, s, b); });
    if (c + 1 < nch) {
      store_xs((c + 1) & 1);
      if (c + 2 < nch) load_xs(c + 2);
    }
  }
#pragma unroll
  for (int s = 0; s < kQNs; ++s) {
    const int col = n0 + (wv * kQNs + s) * 16 + c16;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * h + r;
        if (col < a.V && row < rows) a.out[(m0 + row) * a.ldo + col] = acc[s][i][r];
      }
  }
}

template <bool H, int G, int MB, bool ZP>
void launch_tile(const HeadQ4Args& a, hipStream_t st) {
  constexpr int KC = MB == 1 ? 512 : 256;
  const int rows_ld = a.B < MB * 16 ? a.B : MB * 16;
  const int stage = rows_ld * (KC + 8) * 2 + KC / G * MB * 16 * 4 + kQBn * (KC / G) * 4 * (ZP ? 2 : 1);
  const dim3 grid((a.V + kQBn - 1) / kQBn, (a.B + MB * 16 - 1) / (MB * 16));
  constexpr int kMost = 2 * (MB * 16 * (KC + 8) * 2 + KC / G * MB * 16 * 4 + kQBn * (KC / G) * 4 * (ZP ? 2 : 1));
  static DynLdsOnce configured;
  allow_dyn_lds(configured, {reinterpret_cast<const void*>(k_head_q4<H, G, MB, ZP, KC>)}, kMost);
  hipLaunchKernelGGL((k_head_q4<H, G, MB, ZP, KC>), grid, dim3(kQNt), 2 * stage, st, a, rows_ld);
}

template <bool H, int G>
void launch_group(const HeadQ4Args& a, hipStream_t st) {
  auto go = [&](auto mb) {
    constexpr int MB = decltype(mb)::value;
    if (a.z)
      launch_tile<H, G, MB, true>(a, st);
    else
      launch_tile<H, G, MB, false>(a, st);
  };
  if (a.B <= 16)
    go(std::integral_constant<int, 1>{});
  else if (a.B <= 32)
    go(std::integral_constant<int, 2>{});
  else
    go(std::integral_constant<int, 4>{});
}

}  // namespace

void launch_head_q4(const HeadQ4Args& a, int dtype, int group, int cus, hipStream_t st) {
  auto go = [&](auto h) {
    constexpr bool H = decltype(h)::value;
    if (group == 32)
      launch_group<H, 32>(a, st);
    else if (group == 64)
      launch_group<H, 64>(a, st);
    else
      launch_group<H, 128>(a, st);
  };
  if (dtype == VSMP_F16)
    go(std::true_type{});
  else
    go(std::false_type{});
}

}  // namespace vsmp
