// Shared between the kernels of the operators around the pick (include/vsmp_logits.h) and their host
// launch code: constants, kernel arguments, launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "vsmp_logits.h"

namespace vsmp {

constexpr int kOpVocab = 1 << 20;     // logits per row
constexpr int kOpIds = 64;            // tokens a row of vsmp_logprobs may ask for: one lane each
constexpr int kOpRows = 1 << 13;      // rows of one launch of k_adjust that counts `left`
constexpr int kOpSlots = 4096;        // parts of one launch of split rows, two a row at least
// 32-bit words between two rows' tickets: 128 bytes, so that rows do not share a line. Every part of every row
// adds to its row's, and a line takes them one after the other (32 rows of 151,936 logits in 38 parts: 16.1 us
// with the tickets side by side).
constexpr int kOpPad = 32;
constexpr int kAdjustParts = 4096;    // logits per 256-thread workgroup of k_adjust, 16 per thread

// Device scratch of these operators: allocated at its full size by a context's first call that needs
// it, never replaced. The words are zero between calls, which the last part of a row sees to.
struct OpScratch {
  unsigned long long* left;  // [kOpRows][kOpPad / 2], the first of each: tickets << 32 | logits counted
  unsigned int* tick;        // [kOpSlots / 2][kOpPad], the first of each
  unsigned long long* part;  // [kOpSlots]: a part's maximum << 32 | its sum relative to it (any value between calls)
  int* count;                // [kOpSlots][kOpIds]: per part, ids before each asked id (any value between calls)
};

struct AdjustArgs {
  const void* in;
  long long ldi;
  int B, V, P;               // P parts of kAdjustParts logits per row
  const vsmp_penalty* pen;   // device array (per row) or null
  vsmp_penalty shared;       // every row's when pen is null
  const int* hist;           // null: no history
  const int* hist_off;
  const int* hist_len;       // null: row r's history ends at hist_off[r + 1]; else after hist_len[r] ids
  const int* gone;           // with hist_len: ids that a sequence's history has lost at its front
  const vsmp_params* seq_params;  // with hist_len: a sequence's parameters (repeat_last above 0 bounds its window)
  const int* slot;           // null, or the sequence whose history row r has
  const int* prompt_len;
  const int* bias_ids;
  const float* bias;
  const int* bias_off;       // null: no biases
  const uint32_t* mask;      // null: no masks
  long long ldm;
  int n_masks;
  const int* mask_row;
  float* out;
  long long ldo;
  int* left;
  unsigned long long* acc;   // OpScratch::left, or null without `left`
};

struct LogprobArgs {
  const void* x;
  long long ld;
  int B, V;
  int P, L;                  // P parts of L logits per row
  const int* ids;
  long long ldj;
  int n;
  float* logprob;
  int* rank;
  float* lse;
  OpScratch s;               // used when P > 1
};

struct HeadQ4Args {
  const uint16_t* x;
  long long ldx;
  const uint8_t* q;
  long long ldq;
  const void* sc;
  long long lds;
  int sc_type;               // vsmp_dtype
  const uint8_t* z;          // null: 8 everywhere
  long long ldz;
  int B, V, D;
  float* out;
  long long ldo;
};

void launch_adjust(const AdjustArgs& a, int dtype, hipStream_t st);
// Parts and part length of vsmp_logprobs's rows.
void logprob_parts(int B, int V, int dtype, int cus, int* P, int* L);
void launch_logprobs(const LogprobArgs& a, int dtype, hipStream_t st);
void launch_head_q4(const HeadQ4Args& a, int dtype, int group, int cus, hipStream_t st);

}  // namespace vsmp
