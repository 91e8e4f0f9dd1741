// Shared between the kernels of beams and the states behind them (include/vsmp_beam.h) and their host launch
// code: constants, kernel arguments, launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "vsmp_beam.h"

namespace vsmp {

constexpr int kBeamMax = 64;          // beams of a group, now and next: one lane each
constexpr int kBeamStops = 16;        // stop tokens
constexpr int kBeamSlots = 4096;      // parts of one launch
constexpr int kBeamPad = 32;          // 32-bit words between two groups' tickets (kOpPad's reason)
constexpr int kPagesMax = 1 << 20;    // pages of a pool
constexpr int kPageRows = 8192;       // rows of a paged cache
constexpr int kPageRoom = 1 << 30;    // tokens of a row
constexpr int kPageChunk = 256;       // 16-byte columns of a plane that a wave copies at a time

// Device scratch of vsmp_beam_select: allocated by a context's first call, never replaced. The tickets are zero
// between calls, which the last part of a group sees to.
struct BeamScratch {
  unsigned int* tick;        // [kBeamSlots][kBeamPad], the first of each: a group's
  unsigned long long* key;   // [kBeamSlots][kBeamMax]: a part's largest logits, in order (any value between calls)
  double* sum;               // [kBeamSlots]: a part's sum of exponentials relative to its maximum
  float* max;                // [kBeamSlots]
};

// idx / n, with m = (2^32 - 1) / n: m n >= 2^32 - n, so that idx m / 2^32 is less than one below idx / n.
__device__ __forceinline__ uint32_t divide(uint32_t idx, uint32_t n, uint32_t m) {
  const uint32_t q = __umulhi(idx, m);
  return idx - q * n >= n ? q + 1 : q;
}

struct BeamArgs {
  const void* x;
  long long ld;
  int G, W, V, N;
  int P, L;                  // P parts of L logits per row
  int row0;                  // number of the first row, added to parents
  const float* scores;
  int stops[kBeamStops];
  int n_stop;
  uint32_t m_parts, m_n, m_stop;  // (2^32 - 1) / P, N, n_stop (launch_beam)
  int log_s;                      // lanes of a row's parts in the last part: 2^log_s
  int log_j;                      // entries of each list that make its bound: 2^log_j
  bool alone;                     // a wave ends a part and a group by itself
  int* token;
  int* parent;
  float* score;
  int* end_token;            // null: no ends
  int* end_parent;
  float* end_score;
  int* n_end;
  BeamScratch s;
};

// What the kernels need of vsmp_planes.
struct PlaneArgs {
  void* const* planes;
  int n_planes;
  long long row_stride;
  int pieces;
  long long piece_stride;
  int tokens, token_bytes;
};

struct ReorderArgs {
  PlaneArgs p;
  int plane0;                // the launch's first plane
  int row0;                  // its first row
  const int* parent;         // of the whole batch
  const int* len;            // null: all tokens
  int width;
  bool streams;              // the planes hold more than the caches do (launch_reorder)
  int unit;                  // 0: tokens are whole columns; else bytes that divide a token (launch_reorder)
};

struct PageCopy {
  int src, row, at, tokens;  // a page's first tokens, to the page that the row has at this table entry
};

// Device scratch of vsmp_pages_step and vsmp_pages_compact: allocated by a context's first call of either, never
// replaced. delta, writers, order, n_moves and tick are zero between calls.
struct PageScratch {
  int* delta;                   // [kPagesMax]: holders that a page gains
  int* writers;                 // [kPagesMax]: rows that grow in a begun page
  unsigned long long* order;    // [kPagesMax]: the largest of their tokens << 32 | ~row
  unsigned long long* bits;     // [kPagesMax / 64]: pages that are free (step) or in use (compact)
  int* before;                  // [kPagesMax / 64 + 1]: compact: pages in use before each word
  int* moves;                   // [kPagesMax]: compact: the pages in use at n and beyond; step: pages whose holders change
  int* n_moves;                 // step: how many, with repetitions
  int* room;                    // [kPagesMax]: compact: the free pages below n
  PageCopy* copies;             // [kPageRows]
  int* n_copies;
  unsigned int* tick;
};

struct PageArgs {
  vsmp_pages from, to;
  const int* parent;
  const int* add;
  int add_all;
  int* ok;
  int* moved;
  int* live;
  PlaneArgs cache;              // n_planes 0: none
  uint32_t m_cap;               // (2^32 - 1) / to.row_pages, and workgroups for the tables (launch_pages_step)
  int table_wgs;
  uint32_t m_chunks, m_planes;  // (2^32 - 1) / a page's chunks, and cache.n_planes (copy_wgs)
  PageScratch s;
};

// Parts and part length of vsmp_beam_select's rows: B of them, W a group.
void beam_parts(int B, int W, int V, int dtype, int cus, int* P, int* L);
void launch_beam(BeamArgs a, int dtype, hipStream_t st);
void launch_reorder(ReorderArgs a, int groups, int cus, hipStream_t st);
void launch_pages_step(PageArgs a, int cus, hipStream_t st);
void launch_pages_compact(PageArgs a, int cus, hipStream_t st);

}  // namespace vsmp
