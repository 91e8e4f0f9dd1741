// Host-side pieces shared by the library's C-ABI sources (not part of the ABI).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "vsmp_logits.h"

namespace vsmp {

// false, with the calling thread's error set to "vsmp: <what>: <HIP message>", unless e is success.
bool hip_ok(hipError_t e, const char* what);

// The device a context was created on, and its compute units.
int ctx_device(const vsmp_ctx* c);
int ctx_cus(const vsmp_ctx* c);
// true when `st` (null: the device's null stream) belongs to the context's device; else false, with
// the error set.
bool stream_on_device(const vsmp_ctx* c, hipStream_t st);

// An entry point's device: makes `dev` the calling thread's current HIP device for the scope, and
// gives the caller's current device back on leaving it, so that a call leaves the thread's device
// as it found it. ok() is false (error set) when the device could not be made current.
class DeviceScope {
 public:
  explicit DeviceScope(int dev) : dev_(dev) {
    if (dev < 0) {  // no device named (a null handle, which the entry point then rejects)
      ok_ = true;
      return;
    }
    if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
    ok_ = prev_ == dev || hip_ok(hipSetDevice(dev), "hipSetDevice");
  }
  ~DeviceScope() {
    if (prev_ >= 0 && prev_ != dev_) (void)hipSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  bool ok() const { return ok_; }

 private:
  int dev_;
  int prev_ = -1;
  bool ok_ = false;
};

// One batched pick: the work of vsmp_pick_batch. hist_len (device-resident decode loops): row r's
// history is hist[hist_off[r], hist_off[r] + hist_len[r]) instead of ending at hist_off[r + 1], so
// that each row may own a region larger than its history. slot (device, B distinct entries): row r
// (logits row r, out[r]) samples for sequence slot[r], whose parameters (per row), history entries
// and draw stream it uses. Returns 0 or -1 (error set).
int pick_batch(vsmp_ctx* ctx, const float* logits, int B, int V, long long ld, const vsmp_params* params,
               int params_per_row, const int* hist, const int* hist_off, int u_mode, const double* u,
               unsigned long long* rng_state, unsigned long long counter, int* out, const vsmp_debug* dbg,
               hipStream_t st, const int* hist_len = nullptr, const int* slot = nullptr);

// The scratch of the operators around the pick (vsmp_logits.hpp): allocated and zeroed on `st` by the
// context's first call that needs it, the same memory from then on. false (error set) when it could not
// be, or when `st` is capturing and it is not there yet.
struct OpScratch;
bool ops_scratch(vsmp_ctx* c, hipStream_t st, OpScratch* out);
// true when the context has that scratch, or got it here; a capturing `st` leaves things as they are. For calls that
// need none themselves but are promised to bring it. false (error set) when it could not be allocated.
bool ops_warm(vsmp_ctx* c, hipStream_t st);

// The scratch of vsmp_beam_select, and that of vsmp_pages_step and vsmp_pages_compact (vsmp_beam.hpp), as ops_scratch's.
struct BeamScratch;
struct PageScratch;
bool beam_scratch(vsmp_ctx* c, hipStream_t st, BeamScratch* out);
bool page_scratch(vsmp_ctx* c, hipStream_t st, PageScratch* out);

// vsmp_adjust_logits's argument checks, and its work for arguments that pass them: rows with histories of
// their own (hist_off with B + 1 entries) or, with hist_len, with sequences' regions (see pick_batch).
// pen_per_row: pen is a device array of B. Both return 0 or -1 (error set).
struct AdjustArgs;
int check_adjust(const AdjustArgs& a, int dtype, bool pen_per_row, const vsmp_penalty* pen);
int adjust_logits(vsmp_ctx* ctx, AdjustArgs a, int dtype, bool pen_per_row, const vsmp_penalty* pen, hipStream_t st);

// verbo::Sampler's seeding (reference src/sampler.cpp:11-16,26-31): two successive SplitMix64
// outputs of the seed; seed 0 stands for the steady clock in microseconds.
std::uint64_t splitmix(std::uint64_t& s);
void seed_stream(std::uint64_t seed, std::uint64_t out[2]);

}  // namespace vsmp
