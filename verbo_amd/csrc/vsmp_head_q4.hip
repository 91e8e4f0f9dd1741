// The LM head's product with 4-bit weights: logits = x . (s (q - z))^T.
//
// A weight enters the matrix cores unrounded. A nibble q moved to the top of a 16-bit float's mantissa
// under the exponent of 16 is the number 16 + q (bf16: bits 3-6, f16: bits 6-9), a shift and an and-or
// for two weights. With o = 16 + z,
//   sum_{d in g} x_d (q_d - z) = sum_{d in g} x_d (16 + q_d) - o X_g,   X_g = sum_{d in g} x_d,
// so the group's MFMAs start from -o X_g and the group's result is scaled and added in fp32:
//   acc += s_g P_g.
// The intermediate sums are at most some 31 / 8 of those of the centred weights, which costs one to two
// bits of the fp32 accumulation (measured against 64 bits: 1.1e-7 to 3.7e-7 of the result, where the fp32
// product of the unpacked weights has 2.1e-7 to 9.7e-7).
//
// Strips of 16 columns on v_mfma_f32_16x16x32. An operand's lane (column c, quarter h) holds the 32 weights
// [32 h, 32 h + 32) of a block of 128 of its column as four dwords. An MFMA sums over the four quarters, so for
// groups of 32 (64) the quarters' dwords are transposed between lanes 16 and 32 apart (32 apart) with the lane
// swaps, until an MFMA's four quarters lie in one group. x lies in LDS in the order in which the nibbles of a
// dword come out: 0 4 1 5 2 6 3 7.
//
// What bounds it: few rows read their weights and scales once from HBM (1 x 128,256 x 4,096 in groups of 32: 57 us,
// 5.2 TB/s; 4 x 151,936 x 2,048: 33 us, 5.0 TB/s); small hidden sizes the launch, the staging of x and the few units a
// wave has (1 x 151,936 x 896: 25 us, 3.3 TB/s); more rows the staging of x too, a round trip for each 16-byte piece
// of a thread (16 x 128,256 x 4,096: 64 us, 4.4 TB/s), and many rows the conversions, the scaling and the LDS reads
// beside the MFMAs (64 x 151,936 x 2,048: 93 us, 428 TFLOP/s).
//
// k_head_q4 takes hidden sizes from 256 on, k_head_q4_tile the smaller ones.
#include <algorithm>

#include "vsmp_lds.hpp"
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kQNt = 256;  // threads per workgroup
constexpr int kQNs = 2;    // strips of 16 columns per wave
constexpr int kQBn = kQNt / 64 * 16 * kQNs;

// Eight weights of a dword as 16 + q, in the order 0 4 1 5 2 6 3 7. The constants are held in registers, one scalar
// and one vector: an and-or takes no literal, and with literals it would be two instructions.
template <bool H>
struct Widen {
  uint32_t mask = H ? 0x03C003C0u : 0x00780078u, one = H ? 0x4C004C00u : 0x41804180u;
  __device__ Widen() {
    asm("" : "+s"(mask));
    asm("" : "+v"(one));
  }
  __device__ u32x4 operator()(uint32_t w) const {
    if constexpr (H)
      return u32x4{((w << 6) & mask) | one, ((w << 2) & mask) | one, ((w >> 2) & mask) | one, ((w >> 6) & mask) | one};
    else
      return u32x4{((w << 3) & mask) | one, ((w >> 1) & mask) | one, ((w >> 5) & mask) | one, ((w >> 9) & mask) | one};
  }
};

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

// The small hidden sizes (D < 256): a workgroup of four waves takes 16 rows and 128 columns, x and the scales staged
// in LDS once while the weights are on their way to registers.
//
// H: f16 hidden states (else bf16). G: group. ZP: zero points given.
constexpr int kTileD = 256;              // hidden elements that the stage holds
constexpr int kTileStr = kTileD + 8;     // halfwords per x row in LDS: 16 rows' reads fall on distinct banks
constexpr int tile_groups(int g) { return kTileD / g; }
constexpr int tile_lds(int rows, int g, bool zp) {
  return rows * kTileStr * 2 + tile_groups(g) * 16 * 4 + kQBn * tile_groups(g) * 4 * (zp ? 2 : 1);
}
template <bool H, int G, bool ZP>
__global__ __launch_bounds__(kQNt) void k_head_q4_tile(HeadQ4Args a, int rows_ld) {
  constexpr int kBlk = kTileD / 128;       // blocks of 128
  constexpr int kGc = tile_groups(G);
  constexpr int kGb = 128 / G;             // groups per block
  constexpr int kPr = kTileD / 8;          // 16-byte pieces of an x row
  constexpr int kQx = 16 * kPr / kQNt;
  constexpr int kQs = kQBn * kGc / kQNt;
  constexpr int kSteps = G / 32;           // MFMAs per group

  // x [rows_ld][kTileStr], X [kGc][16], scales [kBlk][kQBn][kGb], offsets the same
  extern __shared__ __align__(16) unsigned char lds[];
  uint16_t* sx = reinterpret_cast<uint16_t*>(lds);
  float* sX = reinterpret_cast<float*>(lds + rows_ld * kTileStr * 2);
  float* sS = sX + kGc * 16;
  float* sO = sS + kQBn * kGc;

  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, c16 = lane & 15, h = lane >> 4;
  const int m0 = blockIdx.y * 16, rows = min(rows_ld, a.B - m0);
  const int n0 = blockIdx.x * kQBn;
  const uint16_t* x = a.x + m0 * a.ldx;
  const int D = a.D, groups = D / G;

  u32x4 w[kQNs][kBlk];
#pragma unroll
  for (int s = 0; s < kQNs; ++s) {
    const uint8_t* q = a.q + min(n0 + (wv * kQNs + s) * 16 + c16, a.V - 1) * a.ldq;
#pragma unroll
    for (int b = 0; b < kBlk; ++b)  // past D: some weights or others, x is zero there
      w[s][b] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(q + min(b * 64 + h * 16, D / 2 - 16)));
  }

  u32x4 px[kQx];
  float ps[kQs], pz[ZP ? kQs : 1];
#pragma unroll
  for (int q = 0; q < kQx; ++q) {
    const int p = tid + q * kQNt, r = p / kPr, k = 8 * (p % kPr);
    px[q] = u32x4{0u, 0u, 0u, 0u};
    if (r < rows && k < D) px[q] = *reinterpret_cast<const u32x4*>(x + r * a.ldx + k);
  }
#pragma unroll
  for (int q = 0; q < kQs; ++q) {
    const int i = tid + q * kQNt, g = min(i % kGc, groups - 1);
    const long long col = min(n0 + i / kGc, a.V - 1);
    ps[q] = scale_at(a.sc, a.sc_type, col * a.lds + g);
    if (ZP) pz[q] = static_cast<float>(a.z[col * a.ldz + g]);
  }
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
      *reinterpret_cast<u32x4*>(&sx[r * kTileStr + 8 * k8]) = o;
      if (k8 % (G / 8) == 0) sX[k8 / (G / 8) * 16 + r] = ZP ? s : -24.0f * s;
    }
  }
#pragma unroll
  for (int q = 0; q < kQs; ++q) {
    const int i = tid + q * kQNt, g = i % kGc, col = i / kGc;
    const int at = (g / kGb * kQBn + col) * kGb + g % kGb;
    sS[at] = ps[q];
    if (ZP) sO[at] = -16.0f - pz[q];
  }
  __syncthreads();

  const Widen<H> widen;
  f32x4 acc[kQNs];
#pragma unroll
  for (int s = 0; s < kQNs; ++s) acc[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // the lane's x row and its offset in a block: k of step t is (t's) + kl
  const int kl = G == 32 ? 8 * h : (G == 64 ? 32 * (h & 1) + 16 * (h >> 1) : 32 * h);
  const int xa = min(c16, rows - 1) * kTileStr + kl;
#pragma unroll
  for (int b = 0; b < kBlk; ++b) {
    if (b * 128 >= D) break;
    uint32_t t[kQNs][4];
    float sc[kQNs][kGb], of[kQNs][kGb];
#pragma unroll
    for (int s = 0; s < kQNs; ++s) {
      t[s][0] = w[s][b].x, t[s][1] = w[s][b].y, t[s][2] = w[s][b].z, t[s][3] = w[s][b].w;
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
        sc[s][g] = sS[(b * kQBn + col) * kGb + g];
        of[s][g] = ZP ? sO[(b * kQBn + col) * kGb + g] : 0.0f;
      }
    }
#pragma unroll
    for (int g = 0; g < kGb; ++g) {
      const f32x4 X = *reinterpret_cast<const f32x4*>(&sX[(b * kGb + g) * 16 + 4 * h]);
      f32x4 P[kQNs];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int step = g * kSteps + u;
        const int k = b * 128 + (G == 32 ? 32 * step : (G == 64 ? 64 * g + 8 * u : 8 * step));
        const u32x4 A = *reinterpret_cast<const u32x4*>(&sx[xa + k]);
#pragma unroll
        for (int s = 0; s < kQNs; ++s) {
          f32x4 c = u ? P[s] : X;
          if (ZP && u == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) c[r] *= of[s][g];
          }
          P[s] = mfma<H>(A, widen(t[s][step]), c);
        }
      }
#pragma unroll
      for (int s = 0; s < kQNs; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(sc[s][g], P[s][r], acc[s][r]);
    }
  }
#pragma unroll
  for (int s = 0; s < kQNs; ++s) {
    const int col = n0 + (wv * kQNs + s) * 16 + c16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * h + r;
      if (col < a.V && row < rows) a.out[(m0 + row) * a.ldo + col] = acc[s][r];
    }
  }
}

// ---- hidden sizes from 256 on: x stays in LDS ------------------------------------------------------------

constexpr int kQAhead = 2;    // units of 256 in flight per wave and strip
constexpr int kQTurn = 2048;  // bytes of LDS in which a strip's unit is turned
// The most waves of a workgroup whose registers then suffice.
constexpr int few_waves(int rt, int group, bool zp, int st) {
  return rt > 16 ? 8 : (st == VSMP_F32 || (zp && group < 128) ? 12 : 16);
}

// One workgroup per CU, RT rows (4, 16, 32 or 64). x (rows_ld rows) and its group sums are staged once; each wave
// then takes pairs of strips by itself, without a barrier, in units of 256 weights a column, kQAhead units always in
// flight, across the end of a pair too (the last units are loaded again there and their products dropped). The
// last unit ends at D: it overlaps the one before where D is no multiple of 256, and x is zero there.
//
// A unit of a column is 128 bytes, which eight neighbouring lanes load: one line where ldq is a multiple of 128, so
// that a load touches 8 lines (up to 16 where it is not, as for hidden sizes of 896 and 576). Loaded as the products
// need them, 16 bytes of a column in lanes 16 apart, every 16 lanes touch 16 lines, and the
// weights' stream alone was 1.2 to 1.3 times as long (1 x 128,256 x 4,096 70.6 against 56.8 us, 4 x 151,936 x 2,048
// 42.1 / 33.0, timing only). The lanes exchange them through LDS of the wave's own; piece p of column c lies at
// p ^ c, so that neither side meets a bank twice. Scales and zero points of a unit are loaded with it, a column's
// side by side, and go through LDS likewise. (No load depends on a condition: the compiler's waits then count only
// the loads that are behind.) With RT = 4 row r is the matrix cores' row 4 r, so that one accumulator register of
// four holds results and the others are left alone.
//
// CH: x does not fit. It is staged chu units at a time (an even number), between two barriers, and each wave takes
// one pair.
template <bool H, int G, int RT, bool ZP, int ST, bool CH>
__global__ __launch_bounds__(64 * few_waves(RT, G, ZP, ST)) void k_head_q4(HeadQ4Args a, int rows_ld, int pairs, int chu) {
  constexpr int kGb = 128 / G, kSteps = G / 32;
  constexpr int MB = RT <= 16 ? 1 : RT / 16, RR = RT == 4 ? 1 : 4;
  constexpr int kSize = ST == VSMP_F32 ? 4 : 2, kSg = 2 * kGb;  // groups of a unit
  extern __shared__ __align__(16) unsigned char lds[];
  const int D = a.D, nun = (D + 255) / 256, held = CH ? chu : nun, str = held * 256 + 8;
  uint16_t* sx = reinterpret_cast<uint16_t*>(lds);
  float* sX = reinterpret_cast<float*>(lds + ((rows_ld * str * 2 + 15) & ~15));  // [held * kSg][RT]
  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, h = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int m0 = blockIdx.y * RT, rows = min(rows_ld, a.B - m0);

  unsigned char* sT = reinterpret_cast<unsigned char*>(sX + held * kSg * RT) + wv * (kQTurn + kQNs * 16 * kSg * 4 * (ZP ? 2 : 1));
  float* sS = reinterpret_cast<float*>(sT + kQTurn);  // the wave's [kQNs * 16][kSg]
  float* sO = sS + kQNs * 16 * kSg;

  const int first = blockIdx.x * nw + wv, pstep = gridDim.x * nw;
  u32x4 w[kQAhead][2][kQNs];
  int lp = first, lu = 0;  // the next unit to load
  uint32_t ls[kQAhead][kGb], lz[kQAhead][ZP ? kGb : 1];
  const char *qb, *sb, *zb = nullptr;     // the pair's first column
  uint32_t qo[kQNs][2], so[kGb], zo[kGb];  // the lane's columns and piece from there, and the columns of its scales
  auto at_pair = [&]() {
    const int col = lp * (16 * kQNs);
    qb = reinterpret_cast<const char*>(a.q) + col * a.ldq;
    sb = static_cast<const char*>(a.sc) + col * a.lds * kSize;
    if (ZP) zb = reinterpret_cast<const char*>(a.z) + col * a.ldz;
#pragma unroll
    for (int s = 0; s < kQNs; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        qo[s][b] = static_cast<uint32_t>(min(16 * s + 8 * b + (lane >> 3), a.V - 1 - col)) * static_cast<uint32_t>(a.ldq) +
                   16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int i = 0; i < kGb; ++i) {
      const uint32_t c = min(i * (64 / kSg) + lane / kSg, a.V - 1 - col);
      so[i] = c * static_cast<uint32_t>(a.lds) * kSize;
      if (ZP) zo[i] = c * static_cast<uint32_t>(a.ldz);
    }
  };
  auto load = [&](int u) {
    const int k = min(lu * 256, D - 256);
    const uint32_t g = k / G + lane % kSg;
#pragma unroll
    for (int i = 0; i < kGb; ++i) {
      if constexpr (ST == VSMP_F32)
        ls[u][i] = *reinterpret_cast<const uint32_t*>(sb + (so[i] + 4u * g));
      else
        ls[u][i] = *reinterpret_cast<const uint16_t*>(sb + (so[i] + 2u * g));
      if (ZP) lz[u][i] = *reinterpret_cast<const uint8_t*>(zb + (zo[i] + g));
    }
#pragma unroll
    for (int s = 0; s < kQNs; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        w[u][b][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(qb + k / 2 + qo[s][b]));
    if (++lu == nun) {
      lu = 0;
      lp = min(lp + pstep, pairs - 1);
      at_pair();
    }
  };
  const int mine = first < pairs ? (pairs - 1 - first) / pstep + 1 : 0;
  if (mine) {
    at_pair();
#pragma unroll
    for (int u = 0; u < kQAhead; ++u) load(u);
  }

  auto stage = [&](int u0, int n) {  // units [u0, u0 + n) of x
    const uint16_t* x = a.x + m0 * a.ldx;
    const int ppr = n * 32;  // 16-byte pieces per row
    for (int p = tid; p < rows * ppr; p += blockDim.x) {
      const int r = p / ppr, k8 = p - r * ppr, u = u0 + (k8 >> 5);
      const int k = u == nun - 1 ? D - 256 + 8 * (k8 & 31) : u * 256 + 8 * (k8 & 31);  // the last unit ends at D
      u32x4 v{0u, 0u, 0u, 0u};
      if (k >= u * 256) v = *reinterpret_cast<const u32x4*>(x + r * a.ldx + k);
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += half_val<H>(v[j] & 0xFFFFu) + half_val<H>(v[j] >> 16);
#pragma unroll
      for (int d = 1; d < G / 8; d <<= 1) s += __shfl_xor(s, d);
      u32x4 o;
      o.x = (v.x & 0xFFFFu) | (v.z << 16);
      o.y = (v.x >> 16) | (v.z & 0xFFFF0000u);
      o.z = (v.y & 0xFFFFu) | (v.w << 16);
      o.w = (v.y >> 16) | (v.w & 0xFFFF0000u);
      *reinterpret_cast<u32x4*>(&sx[r * str + 8 * k8]) = o;
      if (k8 % (G / 8) == 0) sX[k8 / (G / 8) * RT + r] = ZP ? s : -24.0f * s;
    }
  };
  if constexpr (!CH) {
    stage(0, nun);
    __syncthreads();
    if (!mine) return;
  }

  const Widen<H> widen;
  float acc[kQNs][MB][RR];
#pragma unroll
  for (int s = 0; s < kQNs; ++s)
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int r = 0; r < RR; ++r) acc[s][i][r] = 0.0f;
  int xa[MB];
  const int kl = G == 32 ? 8 * h : (G == 64 ? 32 * (h & 1) + 16 * (h >> 1) : 32 * h);
#pragma unroll
  for (int i = 0; i < MB; ++i) xa[i] = min(RT == 4 ? c16 >> 2 : 16 * i + c16, rows - 1) * str + kl;

  int cp = first, cu = 0;  // the unit that is multiplied
  const bool half = D - (nun - 1) * 256 <= 128;  // the first block of the last unit lies before it
  int c0 = 0;  // the first unit of x that is staged
  auto unit = [&](int u) {  // unit cu, which lies in slot u
#pragma unroll
    for (int i = 0; i < kGb; ++i) {
      sS[lane + 64 * i] = ST == VSMP_F32 ? __uint_as_float(ls[u][i]) : half_val<ST == VSMP_F16>(ls[u][i]);
      if (ZP) sO[lane + 64 * i] = -16.0f - static_cast<float>(lz[u][i]);
    }
    u32x4 turned[2][kQNs];
#pragma unroll
    for (int s = 0; s < kQNs; ++s) {
      *reinterpret_cast<u32x4*>(sT + 16 * lane) = w[u][0][s];
      *reinterpret_cast<u32x4*>(sT + 1024 + 16 * lane) = w[u][1][s];
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int b = 0; b < 2; ++b)
        turned[b][s] = *reinterpret_cast<const u32x4*>(sT + 128 * c16 + 16 * ((4 * b + h) ^ (c16 & 7)));
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
    __builtin_amdgcn_sched_barrier(0);
    load(u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b == 0 && half && cu == nun - 1) continue;
      uint32_t t[kQNs][4];
      float sc[kQNs][kGb], of[kQNs][kGb];
#pragma unroll
      for (int s = 0; s < kQNs; ++s) {
        t[s][0] = turned[b][s].x, t[s][1] = turned[b][s].y, t[s][2] = turned[b][s].z, t[s][3] = turned[b][s].w;
        if constexpr (G <= 64) {
          swap32(t[s][0], t[s][2]);
          swap32(t[s][1], t[s][3]);
        }
        if constexpr (G == 32) {
          swap16(t[s][0], t[s][1]);
          swap16(t[s][2], t[s][3]);
        }
#pragma unroll
        for (int g = 0; g < kGb; ++g) {
          const int at = (16 * s + c16) * kSg + b * kGb + g;
          sc[s][g] = sS[at];
          of[s][g] = ZP ? sO[at] : 0.0f;
        }
      }
      const uint16_t* xb = sx + (2 * (cu - c0) + b) * 128;
      const float* Xb = sX + (2 * (cu - c0) + b) * kGb * RT;
#pragma unroll
      for (int g = 0; g < kGb; ++g) {
        f32x4 X[MB], P[kQNs][MB];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (RT == 4)
            X[i] = f32x4{Xb[g * RT + h], 0.0f, 0.0f, 0.0f};
          else
            X[i] = *reinterpret_cast<const f32x4*>(&Xb[g * RT + 16 * i + 4 * h]);
        }
#pragma unroll
        for (int v = 0; v < kSteps; ++v) {
          const int step = g * kSteps + v;
          const int k = G == 32 ? 32 * step : (G == 64 ? 64 * g + 8 * v : 8 * step);
          u32x4 A[MB];
#pragma unroll
          for (int i = 0; i < MB; ++i) A[i] = *reinterpret_cast<const u32x4*>(&xb[xa[i] + k]);
#pragma unroll
          for (int s = 0; s < kQNs; ++s) {
            const u32x4 wb = widen(t[s][step]);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
              f32x4 c = v ? P[s][i] : X[i];
              if (ZP && v == 0) {
#pragma unroll
                for (int r = 0; r < RR; ++r) c[r] *= of[s][g];
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
            for (int r = 0; r < RR; ++r) acc[s][i][r] = __builtin_fmaf(sc[s][g], P[s][i][r], acc[s][i][r]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  };
  auto finish = [&](int pair) {
#pragma unroll
    for (int s = 0; s < kQNs; ++s) {
      const int col = (pair * kQNs + s) * 16 + c16;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const int row = 16 * i + RR * h + r;
          if (col < a.V && row < rows) a.out[(m0 + row) * a.ldo + col] = acc[s][i][r];
          acc[s][i][r] = 0.0f;
        }
    }
  };
  if constexpr (CH) {
    for (; c0 < nun; c0 += chu) {
      if (c0) __syncthreads();
      const int end = min(c0 + chu, nun);
      stage(c0, end - c0);
      __syncthreads();
      if (!mine) continue;
      for (cu = c0; cu < end;) {
#pragma unroll
        for (int u = 0; u < kQAhead; ++u) {  // chu is even: a chunk begins in slot 0
          if (cu < end) unit(u);
          ++cu;
        }
      }
    }
    if (mine) finish(first);
  } else {
    const int total = mine * nun;
    for (int it = 0; it < total; it += kQAhead) {
#pragma unroll
      for (int u = 0; u < kQAhead; ++u) {
        unit(u);
        if (++cu == nun) {
          if (it + u < total) finish(cp);
          cu = 0;
          cp += pstep;
        }
      }
    }
  }
}

// LDS: `units` units of x with their group sums, and what a wave has of its own.
size_t x_lds(int rows, int rt, int units, int group) {
  return ((static_cast<size_t>(rows) * (units * 256 + 8) * 2 + 15) & ~size_t{15}) +
         static_cast<size_t>(units) * (256 / group) * rt * sizeof(float);
}
size_t wave_lds(int group, bool zp) { return kQTurn + 16 * kQNs * 2 * (128 / group) * sizeof(float) * (zp ? 2 : 1); }
constexpr size_t kMostLds = 160 * 1024;

struct Shape {
  bool chunks;
  int units, waves;  // units of x in LDS; waves of a workgroup at most
};
// What fits: x whole with at least kFewWaves waves, or as many units of it as do with the most waves.
Shape shape_of(int rows, int rt, int D, int group, bool zp, int most) {
  constexpr int kFewWaves = 4;
  const int nun = (D + 255) / 256;
  const size_t whole = x_lds(rows, rt, nun, group), own = wave_lds(group, zp);
  if (whole + kFewWaves * own <= kMostLds) return {false, nun, std::min(most, static_cast<int>((kMostLds - whole) / own))};
  int u = 2;
  while (u + 2 < nun && x_lds(rows, rt, u + 2, group) + most * own <= kMostLds) u += 2;
  return {true, u, most};
}

template <bool H, int G, int RT, bool ZP, int ST, bool CH>
void launch_kernel(const HeadQ4Args& a, dim3 grid, int nw, size_t lds, int rows_ld, int pairs, int units, hipStream_t st) {
  static DynLdsOnce configured;
  allow_dyn_lds(configured, {reinterpret_cast<const void*>(k_head_q4<H, G, RT, ZP, ST, CH>)}, static_cast<int>(kMostLds));
  hipLaunchKernelGGL((k_head_q4<H, G, RT, ZP, ST, CH>), grid, dim3(64 * nw), lds, st, a, rows_ld, pairs, units);
}

template <bool H, int G, int RT, bool ZP, int ST>
void launch_as(const HeadQ4Args& a, int cus, hipStream_t st) {
  const int rows_ld = std::min(a.B, RT), groups = (a.B + RT - 1) / RT;
  const int pairs = (a.V + 16 * kQNs - 1) / (16 * kQNs);
  const Shape sh = shape_of(rows_ld, RT, a.D, G, ZP, few_waves(RT, G, ZP, ST));
  int nw = sh.waves;
  // as many rounds of pairs as the most waves would need, and no more waves than those fill
  const int wgs = cus > 0 ? cus : 256, per = (pairs + wgs - 1) / wgs, rounds = (per + nw - 1) / nw;
  nw = (per + rounds - 1) / rounds;
  // With many rows the products bound it, and the SIMDs share them evenly (64 x 151,936 x 2,048: 8 waves 91 us, 7 101)
  if (RT >= 32) nw = std::min(sh.waves, (nw + 3) / 4 * 4);
  const int need = (pairs + nw - 1) / nw;
  const size_t lds = x_lds(rows_ld, RT, sh.units, G) + nw * wave_lds(G, ZP);
  if (!sh.chunks)
    launch_kernel<H, G, RT, ZP, ST, false>(a, dim3(std::min(need, wgs), groups), nw, lds, rows_ld, pairs, sh.units, st);
  else if constexpr (RT > 4)  // four rows always fit
    launch_kernel<H, G, RT, ZP, ST, true>(a, dim3(need, groups), nw, lds, rows_ld, pairs, sh.units, st);
}
template <bool H, int G, int RT>
void launch_rows(const HeadQ4Args& a, int cus, hipStream_t st) {
  auto go = [&](auto zp) {
    constexpr bool ZP = decltype(zp)::value;
    if (a.sc_type == VSMP_F32)
      launch_as<H, G, RT, ZP, VSMP_F32>(a, cus, st);
    else if (a.sc_type == VSMP_BF16)
      launch_as<H, G, RT, ZP, VSMP_BF16>(a, cus, st);
    else
      launch_as<H, G, RT, ZP, VSMP_F16>(a, cus, st);
  };
  if (a.z)
    go(std::true_type{});
  else
    go(std::false_type{});
}

template <bool H, int G, bool ZP>
void launch_tile(const HeadQ4Args& a, hipStream_t st) {
  const int rows_ld = std::min(a.B, 16);
  const dim3 grid((a.V + kQBn - 1) / kQBn, (a.B + 15) / 16);
  static_assert(tile_lds(16, 32, true) <= 64 * 1024, "the stage fits the default limit of dynamic LDS");
  hipLaunchKernelGGL((k_head_q4_tile<H, G, ZP>), grid, dim3(kQNt), tile_lds(rows_ld, G, ZP), st, a, rows_ld);
}

// The rows of a workgroup: the fewest of 4, 16 and 32 that hold the batch; for larger ones 64, or 32 where the x of
// 32 rows fits whole and that of 64 does not (64 x 151,936 x 2,048 93 us in two groups of 32 against 125 in chunks of
// 64; where neither fits, 40 x 128,256 x 4,096 170 / 131 and 64 rows 200 / 164; where both do, 64 x 151,936 x 1,024 53 /
// 45; 24 rows of 4,096 in chunks of 32 91 us against 123 in two groups of 16).
template <bool H, int G>
void launch_group(const HeadQ4Args& a, int cus, hipStream_t st) {
  if (a.D < 256) {
    if (a.z)
      launch_tile<H, G, true>(a, st);
    else
      launch_tile<H, G, false>(a, st);
  } else if (a.B <= 4) {
    launch_rows<H, G, 4>(a, cus, st);
  } else if (a.B <= 16) {
    launch_rows<H, G, 16>(a, cus, st);
  } else {
    const bool zp = a.z != nullptr;
    const bool whole32 = !shape_of(32, 32, a.D, G, zp, 8).chunks, whole64 = !shape_of(std::min(a.B, 64), 64, a.D, G, zp, 8).chunks;
    if (a.B <= 32 || (whole32 && !whole64))
      launch_rows<H, G, 32>(a, cus, st);
    else
      launch_rows<H, G, 64>(a, cus, st);
  }
}

}  // namespace

void launch_head_q4(const HeadQ4Args& a, int dtype, int group, int cus, hipStream_t st) {
  auto go = [&](auto h) {
    constexpr bool H = decltype(h)::value;
    if (group == 32)
      launch_group<H, 32>(a, cus, st);
    else if (group == 64)
      launch_group<H, 64>(a, cus, st);
    else
      launch_group<H, 128>(a, cus, st);
  };
  if (dtype == VSMP_F16)
    go(std::true_type{});
  else
    go(std::false_type{});
}

}  // namespace vsmp
