// The entry points of vsmp_logits_api.cpp over doubles of the kernels' launchers, on the CPU: which rows each launch
// is given. Every row of a batch has to be given once, in order, with the addresses that are its own.
//
//   logits_launches <call> <B>: prints "ok <launches>", or what went wrong
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <string>

#include "vsmp_error.hpp"
#include "vsmp_internal.hpp"
#include "vsmp_logits.hpp"

namespace {

const uintptr_t kIn = 1ull << 44, kOut = 1ull << 48, kIds = 1ull << 52, kOff = 1ull << 53, kMask = 1ull << 54, kLp = 1ull << 55,
                kLse = 1ull << 56, kLeft = 1ull << 57, kPen = 1ull << 58;
long long B, next_row = 0, launches = 0;
std::string error;

[[noreturn]] void wrong(const char* what) {
  std::printf("%s: launch %lld, row %lld of %lld\n", what, launches, next_row, B);
  std::exit(1);
}
template <class T>
void at(const T* p, uintptr_t base, long long per_row) {
  if (reinterpret_cast<uintptr_t>(p) != base + static_cast<uintptr_t>(next_row) * static_cast<uintptr_t>(per_row)) wrong("address");
}
void rows(int n, int most) {
  ++launches;
  if (n < 1 || n > most || next_row + n > B) wrong("rows");
  next_row += n;
}

}  // namespace

extern "C" hipError_t hipGetDevice(int* d) {
  *d = 0;
  return hipSuccess;
}
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }
extern "C" hipError_t hipGetLastError() { return hipSuccess; }

namespace vsmp {

int set_error(const std::string& m) {
  error = m;
  return -1;
}
void clear_error() { error.clear(); }
bool hip_ok(hipError_t e, const char*) { return e == hipSuccess; }
int ctx_device(const vsmp_ctx*) { return 0; }
int ctx_cus(const vsmp_ctx*) { return 256; }
bool stream_on_device(const vsmp_ctx*, hipStream_t) { return true; }
bool ops_scratch(vsmp_ctx*, hipStream_t, OpScratch* out) {
  *out = OpScratch{};
  return true;
}
bool ops_warm(vsmp_ctx*, hipStream_t) { return true; }

void launch_adjust(const AdjustArgs& a, int, hipStream_t) {
  at(static_cast<const char*>(a.in), kIn, 2);
  at(a.out, kOut, 4);
  if (a.pen) at(a.pen, kPen, sizeof(vsmp_penalty));
  at(a.hist_off, kOff, 4);
  at(a.mask, kMask, 4);
  if (a.n_masks != B - next_row) wrong("masks");
  rows(a.B, 1 << 20);
}
void logprob_parts(int, int V, int, int, int* P, int* L) {
  *P = 1;
  *L = V;
}
void launch_logprobs(const LogprobArgs& a, int, hipStream_t) {
  at(static_cast<const char*>(a.x), kIn, 2);
  at(a.ids, kIds, 4);
  at(a.logprob, kLp, 4);
  at(a.lse, kLse, 4);
  rows(a.B, 1 << 20);
}
void launch_head_q4(const HeadQ4Args& a, int, int, int, hipStream_t) {
  at(a.x, kIn, 64);
  at(a.out, kOut, 4);
  rows(a.B, 1 << 16);
}

}  // namespace vsmp

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  const std::string call = argv[1];
  B = std::atoll(argv[2]);
  const int n = static_cast<int>(B);
  auto* ctx = reinterpret_cast<vsmp_ctx*>(uintptr_t{64});
  auto i = [](uintptr_t p) { return reinterpret_cast<int*>(p); };
  auto f = [](uintptr_t p) { return reinterpret_cast<float*>(p); };
  const void* in = reinterpret_cast<const void*>(kIn);
  int rc = -1;
  if (call == "adjust" || call == "adjust_left")
    rc = vsmp_adjust_logits(ctx, in, VSMP_BF16, 1, n, 1, reinterpret_cast<const vsmp_penalty*>(kPen), 1, i(kIds), i(kOff), nullptr, nullptr,
                            nullptr, nullptr, reinterpret_cast<const unsigned*>(kMask), 1, n, nullptr, f(kOut), 1,
                            call == "adjust" ? nullptr : i(kLeft), nullptr);
  else if (call == "logprobs")
    rc = vsmp_logprobs(ctx, in, VSMP_BF16, 1, n, 1, i(kIds), 1, 1, f(kLp), nullptr, f(kLse), nullptr);
  else if (call == "head")
    rc = vsmp_head_logits_q4(ctx, in, VSMP_BF16, 32, reinterpret_cast<const void*>(kIds), 16, reinterpret_cast<const void*>(kPen), VSMP_F32,
                             1, nullptr, 0, 32, n, 1, 32, f(kOut), 1, nullptr);
  if (rc != 0 || next_row != B) wrong(error.empty() ? "rows left out" : error.c_str());
  std::printf("ok %lld\n", launches);
  return 0;
}
