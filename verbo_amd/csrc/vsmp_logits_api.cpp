// C ABI of the operators around the pick (include/vsmp_logits.h): argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

#include "vsmp_error.hpp"
#include "vsmp_internal.hpp"
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

size_t elem_size(int dtype) { return dtype == VSMP_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// -1 with the message set unless a batch of rows of logits is one that the operators take.
int check_rows(const void* x, int dtype, long long ld, int B, int V) {
  if (!x) return set_error("vsmp: logits are required");
  if (dtype < VSMP_F32 || dtype > VSMP_F16) return set_error("vsmp: unknown dtype");
  if (B < 1 || V < 1) return set_error("vsmp: need B >= 1 and V >= 1");
  if (V > kOpVocab) return set_error("vsmp: vocabulary larger than " + std::to_string(kOpVocab));
  if (ld < V || ld > (LLONG_MAX >> 4) / B) return set_error("vsmp: the rows' stride must be >= V and the batch addressable");
  if (!aligned(x, elem_size(dtype))) return set_error("vsmp: logits must be aligned to their elements");
  return 0;
}

}  // namespace

int check_adjust(const AdjustArgs& a, int dtype, bool pen_per_row, const vsmp_penalty* pen) {
  if (check_rows(a.in, dtype, a.ldi, a.B, a.V) != 0) return -1;
  if (!a.out || !aligned(a.out, 4)) return set_error("vsmp: out is required, aligned to 4 bytes");
  if (a.ldo < a.V || a.ldo > (LLONG_MAX >> 4) / a.B) return set_error("vsmp: ldo must be >= V and the batch addressable");
  if ((a.hist == nullptr) != (a.hist_off == nullptr)) return set_error("vsmp: hist and hist_off go together");
  if ((a.bias_ids == nullptr) != (a.bias_off == nullptr) || (a.bias == nullptr) != (a.bias_off == nullptr))
    return set_error("vsmp: bias_ids, bias and bias_off go together");
  if (a.prompt_len && !a.hist) return set_error("vsmp: prompt_len needs histories");
  if (!a.mask && (a.mask_row || a.n_masks != 0)) return set_error("vsmp: mask_row and n_masks need masks");
  if (a.mask) {
    if (a.n_masks < 1 || a.ldm < (a.V + 31) / 32 || a.ldm > (LLONG_MAX >> 4) / a.n_masks)
      return set_error("vsmp: need n_masks >= 1 masks of ldm >= ceil(V / 32) words");
    if (!a.mask_row && a.n_masks < a.B) return set_error("vsmp: without mask_row every row needs a mask of its own");
  }
  if (pen && !pen_per_row) {
    if (!(pen->repeat > 0.0f) || !std::isfinite(pen->repeat) || !std::isfinite(pen->presence) || !std::isfinite(pen->frequency))
      return set_error("vsmp: penalties must be finite, repeat above 0");
  }
  // a row's struct is read with scalar loads, which take an address's low two bits for zero
  if (pen_per_row && !aligned(pen, 4)) return set_error("vsmp: per-row penalties must be aligned to 4 bytes");
  // the rows in memory: the same ones, or none of the others' bytes (apart as wholes, or row by row in turn)
  const long long size = static_cast<long long>(elem_size(dtype)), il = a.V * size, ol = a.V * 4LL, is = a.ldi * size, os = a.ldo * 4;
  const uintptr_t i0 = reinterpret_cast<uintptr_t>(a.in), o0 = reinterpret_cast<uintptr_t>(a.out);
  const uintptr_t i1 = i0 + (a.B - 1) * is + il, o1 = o0 + (a.B - 1) * os + ol;
  const bool in_place = i0 == o0 && dtype == VSMP_F32 && a.ldi == a.ldo;
  if (!in_place && i0 < o1 && o0 < i1) {
    const long long at = (static_cast<long long>(o0 - i0) % is + is) % is;  // an output row's place in the logits' stride
    if (is != os || at < il || at + ol > is) return set_error("vsmp: out must be the fp32 logits themselves or not overlap them");
  }
  return 0;
}

int adjust_logits(vsmp_ctx* ctx, AdjustArgs a, int dtype, bool pen_per_row, const vsmp_penalty* pen, hipStream_t st) {
  const vsmp_penalty none = {1.0f, 0.0f, 0.0f, 0};
  a.shared = pen && !pen_per_row ? *pen : none;
  a.pen = pen_per_row ? pen : nullptr;
  a.P = (a.V + kAdjustParts - 1) / kAdjustParts;
  if (a.left) {
    OpScratch s{};
    if (!ops_scratch(ctx, st, &s)) return -1;
    a.acc = s.left;
  }
  const int rows = std::min(a.left ? kOpRows : 1 << 20, (1 << 23) / a.P);  // a launch takes fewer than 2^32 threads
  for (int r = 0, n; r < a.B; r += n) {  // the counting words of one launch serve the next one too
    n = std::min(rows, a.B - r);
    AdjustArgs p = a;
    p.B = n;
    p.in = static_cast<const char*>(a.in) + static_cast<size_t>(r) * a.ldi * elem_size(dtype);
    p.out = a.out + static_cast<size_t>(r) * a.ldo;
    if (a.pen) p.pen = a.pen + r;
    if (a.slot) p.slot = a.slot + r;
    else if (a.hist_off) {
      p.hist_off = a.hist_off + r;
      if (a.hist_len) {
        p.hist_len = a.hist_len + r;
        p.gone = a.gone + r;
        p.seq_params = a.seq_params + r;
      }
    }
    if (a.prompt_len) p.prompt_len = a.prompt_len + r;
    if (a.bias_off) p.bias_off = a.bias_off + r;
    if (a.mask_row) p.mask_row = a.mask_row + r;
    else if (a.mask) {
      p.mask = a.mask + static_cast<size_t>(r) * a.ldm;
      p.n_masks = a.n_masks - r;
    }
    if (a.left) p.left = a.left + r;
    launch_adjust(p, dtype, st);
    if (!hip_ok(hipGetLastError(), "adjust launch")) return -1;
  }
  return 0;
}

}  // namespace vsmp

extern "C" {

int vsmp_adjust_logits(vsmp_ctx* ctx, const void* in, int dtype, long long ldi, int B, int V, const vsmp_penalty* pen,
                       int pen_per_row, const int* hist, const int* hist_off, const int* prompt_len, const int* bias_ids,
                       const float* bias, const int* bias_off, const unsigned int* mask, long long ldm, int n_masks,
                       const int* mask_row, float* out, long long ldo, int* left, void* stream) {
  vsmp::clear_error();
  if (!ctx) return vsmp::set_error("vsmp: null context");
  vsmp::AdjustArgs a{};
  a.in = in;
  a.ldi = ldi;
  a.B = B;
  a.V = V;
  a.hist = hist;
  a.hist_off = hist_off;
  a.prompt_len = prompt_len;
  a.bias_ids = bias_ids;
  a.bias = bias;
  a.bias_off = bias_off;
  a.mask = mask;
  a.ldm = ldm;
  a.n_masks = n_masks;
  a.mask_row = mask_row;
  a.out = out;
  a.ldo = ldo;
  a.left = left;
  const bool per_row = pen && pen_per_row != 0;
  if (vsmp::check_adjust(a, dtype, per_row, pen) != 0) return -1;
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  if (!scope.ok() || !vsmp::stream_on_device(ctx, static_cast<hipStream_t>(stream))) return -1;
  return vsmp::adjust_logits(ctx, a, dtype, per_row, pen, static_cast<hipStream_t>(stream));
}

int vsmp_logprobs(vsmp_ctx* ctx, const void* logits, int dtype, long long ld, int B, int V, const int* ids, long long ldj,
                  int n, float* logprob, int* rank, float* lse, void* stream) {
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (vsmp::check_rows(logits, dtype, ld, B, V) != 0) return -1;
  if (n < 0 || n > vsmp::kOpIds) return set_error("vsmp: need 0 <= n <= " + std::to_string(vsmp::kOpIds));
  if (n > 0 && (!ids || !logprob || ldj < n || ldj > (LLONG_MAX >> 4) / B))
    return set_error("vsmp: ids (ldj >= n) and logprob are required with n > 0");
  if (n == 0 && !lse) return set_error("vsmp: lse is required with n = 0");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::LogprobArgs a{};
  a.x = logits;
  a.ld = ld;
  a.V = V;
  a.ids = ids;
  a.ldj = ldj;
  a.n = n;
  const int rows = 1 << 20;  // of one launch
  for (int r = 0, m; r < B; r += m) {
    m = std::min(rows, B - r);
    vsmp::LogprobArgs p = a;
    p.B = m;
    p.x = static_cast<const char*>(logits) + static_cast<size_t>(r) * ld * vsmp::elem_size(dtype);
    p.ids = n ? ids + static_cast<size_t>(r) * ldj : nullptr;
    p.logprob = n ? logprob + static_cast<size_t>(r) * n : nullptr;
    p.rank = n && rank ? rank + static_cast<size_t>(r) * n : nullptr;
    p.lse = lse ? lse + r : nullptr;
    vsmp::logprob_parts(p.B, V, dtype, vsmp::ctx_cus(ctx), &p.P, &p.L);
    if (!(p.P > 1 ? vsmp::ops_scratch(ctx, st, &p.s) : vsmp::ops_warm(ctx, st))) return -1;
    vsmp::launch_logprobs(p, dtype, st);
    if (!vsmp::hip_ok(hipGetLastError(), "logprobs launch")) return -1;
  }
  return 0;
}

int vsmp_head_logits_q4(vsmp_ctx* ctx, const void* hidden, int dtype, long long ldh, const void* q, long long ldq,
                        const void* scales, int scale_dtype, long long lds, const unsigned char* zeros, long long ldz,
                        int group, int B, int V, int D, float* logits, long long ldl, void* stream) {
  using vsmp::aligned;
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (!hidden || !q || !scales || !logits) return set_error("vsmp: hidden, q, scales and logits are required");
  if (dtype != VSMP_BF16 && dtype != VSMP_F16) return set_error("vsmp: hidden must be bf16 or f16");
  if (scale_dtype < VSMP_F32 || scale_dtype > VSMP_F16) return set_error("vsmp: unknown scale dtype");
  if (group != 32 && group != 64 && group != 128) return set_error("vsmp: group must be 32, 64 or 128");
  if (B < 1 || V < 1) return set_error("vsmp: need B >= 1 and V >= 1");
  if (V > vsmp::kOpVocab) return set_error("vsmp: vocabulary larger than " + std::to_string(vsmp::kOpVocab));
  if (D < 32 || D > 16384 || D % group != 0) return set_error("vsmp: D must be a multiple of group in [32, 16384]");
  if (ldh < D || ldh % 8 != 0 || ldh > (LLONG_MAX >> 4) / B || !aligned(hidden, 16))
    return set_error("vsmp: hidden must be 16-byte aligned with ldh >= D a multiple of 8");
  if (ldq < D / 2 || ldq % 16 != 0 || ldq > (LLONG_MAX >> 4) / V || !aligned(q, 16))
    return set_error("vsmp: q must be 16-byte aligned with ldq >= D / 2 a multiple of 16");
  if (lds < D / group || lds > (LLONG_MAX >> 4) / V || !aligned(scales, vsmp::elem_size(scale_dtype)))
    return set_error("vsmp: scales must be aligned to their elements with lds >= D / group");
  if (ldq >= 1 << 26 || lds >= 1 << 24 || (zeros && ldz >= 1 << 26))  // a tile's columns are addressed with 32 bits
    return set_error("vsmp: ldq and ldz must be below 2^26, lds below 2^24");
  if (zeros && (ldz < D / group || ldz > (LLONG_MAX >> 4) / V)) return set_error("vsmp: ldz must be >= D / group");
  if (ldl < V || ldl > (LLONG_MAX >> 4) / B || !aligned(logits, 4)) return set_error("vsmp: ldl must be >= V, logits aligned to 4 bytes");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::HeadQ4Args a{};
  a.x = static_cast<const uint16_t*>(hidden);
  a.ldx = ldh;
  a.q = static_cast<const uint8_t*>(q);
  a.ldq = ldq;
  a.sc = scales;
  a.lds = lds;
  a.sc_type = scale_dtype;
  a.z = zeros;
  a.ldz = ldz;
  a.V = V;
  a.D = D;
  a.ldo = ldl;
  const int rows = 1 << 16;  // of one launch
  for (int r = 0; r < B; r += a.B) {
    a.B = std::min(rows, B - r);
    a.x = static_cast<const uint16_t*>(hidden) + static_cast<size_t>(r) * ldh;
    a.out = logits + static_cast<size_t>(r) * ldl;
    vsmp::launch_head_q4(a, dtype, group, vsmp::ctx_cus(ctx), st);
    if (!vsmp::hip_ok(hipGetLastError(), "head launch")) return -1;
  }
  return 0;
}

}  // extern "C"
