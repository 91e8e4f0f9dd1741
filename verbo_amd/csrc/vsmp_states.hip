// States that follow their beams: rows of planes moved in place (k_reorder), and a cache in pages: a step's forks,
// cuts and growth (k_pages_fork, k_pages_take, k_page_copy) and compaction (k_pages_scan, k_pages_pair, k_pages_move).
#include <algorithm>

#include "vsmp_beam.hpp"

namespace vsmp {
namespace {

constexpr int kNt = 256;

template <class T>
__device__ __forceinline__ T agent_load(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ void agent_store(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T agent_add(T* p, T v) {
  return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What this thread has stored and added so far is in memory.
__device__ __forceinline__ void drain() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// ---- k_reorder -------------------------------------------------------------------------------------------

template <int B>
using Column = uint32_t __attribute__((ext_vector_type(B / 4), aligned(1)));
// A plane's bytes are device memory: the compiler cannot know from an address that is loaded, and would take instructions
// that serve LDS and the stack as well.
typedef __attribute__((address_space(1))) char Bytes;
__device__ __forceinline__ Bytes* plane_at(const PlaneArgs& p, uint32_t i) { return (Bytes*)p.planes[i]; }
template <class T>
__device__ __forceinline__ T get(const Bytes* p) {
  return *(const __attribute__((address_space(1))) T*)p;
}
template <class T>
__device__ __forceinline__ void set(Bytes* p, T v) {
  *(__attribute__((address_space(1))) T*)p = v;
}
template <class T>
__device__ __forceinline__ void stream(Bytes* p, T v) {  // of more than the caches hold
  __builtin_nontemporal_store(v, (__attribute__((address_space(1))) T*)p);
}

template <class T>
using Loose __attribute__((aligned(1))) = T;

// A column in which tokens may end, unit by unit: whole units, since a token is.
template <int MAXW, int B, class T>
__device__ __forceinline__ void ends(Bytes* base, uint32_t at, int n, const long long* from, const long long* to, const int* bytes) {
#pragma unroll 1
  for (uint32_t k = 0; k < B; k += sizeof(T)) {
    asm volatile("" ::: "memory");
    T v[MAXW];
#pragma unroll
    for (int i = 0; i < MAXW; ++i)
      if (i < n && at + k < static_cast<uint32_t>(bytes[i])) v[i] = get<Loose<T>>(base + k + from[i]);
#pragma unroll
    for (int i = 0; i < MAXW; ++i)
      if (i < n && at + k < static_cast<uint32_t>(bytes[i])) set<Loose<T>>(base + k + to[i], v[i]);
  }
}

// A column of B bytes over a group's rows belongs to one thread, which loads it from every parent before it stores it in
// any row: in place without a wait. Where tokens are no whole columns (a.unit: 4, 2 or 1 bytes, which they are in whole), the
// columns beyond the least of the rows' ends go unit by unit. Rows that stay are neither read nor written for themselves; a
// parent with several children is read by each of their loads, from memory once.
//
// Bound by reads and writes together: 16 groups of 4 rows, 48 planes of 2 x 2,048 x 128 bf16, 1.74 GB moved 364 us (4.8
// TB/s; a large copy reaches 4.75), with stores that are not streamed 372; 32 groups of 6 rows of 20,012 bytes in 24
// planes, 104 MB, 21.4 us. Where a row's end is no whole column, moving it byte by byte took 30.6 us.
template <int MAXW, int B>
__global__ __launch_bounds__(kNt, MAXW == 8 ? 4 : 1) void k_reorder(ReorderArgs a) {
  typedef Column<B> vec;
  __shared__ long long s_from[MAXW], s_to[MAXW];  // of the rows that move: where their parents and they lie in a plane
  __shared__ int s_bytes[MAXW];                   // and what they take of each piece
  __shared__ int s_n, s_most, s_least;
  const int tid = threadIdx.x, first = a.row0 + static_cast<int>(blockIdx.y) * a.width;
  if (tid < 64) {
    int p = tid, bytes = 0;
    if (tid < a.width) {
      p = a.parent[first + tid] - first;
      if (p != tid && static_cast<unsigned>(p) < static_cast<unsigned>(a.width))
        bytes = (a.len ? min(max(a.len[first + p], 0), a.p.tokens) : a.p.tokens) * a.p.token_bytes;
    }
    const unsigned long long moves = __ballot(bytes > 0);
    int most = bytes, least = bytes > 0 ? bytes : 0x7FFFFFFF;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      most = max(most, __shfl_xor(most, d));
      least = min(least, __shfl_xor(least, d));
    }
    if (bytes > 0) {
      const int k = __popcll(moves & ((1ull << tid) - 1ull));
      s_from[k] = (first + p) * a.p.row_stride;
      s_to[k] = (first + tid) * a.p.row_stride;
      s_bytes[k] = bytes;
    }
    if (tid == 0) {
      s_n = __popcll(moves);
      s_most = most;
      s_least = least;
    }
  }
  __syncthreads();
  const int n = s_n;
  if (n == 0) return;
  const uint32_t cols = (static_cast<uint32_t>(s_most) + B - 1) / B, m = 0xFFFFFFFFu / cols, least = static_cast<uint32_t>(s_least);
  const uint32_t pieces = static_cast<uint32_t>(a.p.pieces), mp = 0xFFFFFFFFu / pieces;
  const uint32_t total = static_cast<uint32_t>(a.p.n_planes) * pieces * cols;
  for (uint32_t idx = blockIdx.x * kNt + tid; idx < total; idx += gridDim.x * kNt) {
    asm volatile("" ::: "memory");  // the rows' places are read from LDS when they are used: all of them in registers leave no waves
    const uint32_t run = divide(idx, cols, m), at = (idx - run * cols) * B;
    const uint32_t plane = divide(run, pieces, mp), piece = run - plane * pieces;
    Bytes* base = plane_at(a.p, a.plane0 + plane) + piece * a.p.piece_stride + at;
    if (at + B <= least) {
      vec v[MAXW];
#pragma unroll
      for (int i = 0; i < MAXW; ++i)
        if (i < n) v[i] = get<vec>(base + s_from[i]);
      if (a.streams) {
#pragma unroll
        for (int i = 0; i < MAXW; ++i)
          if (i < n) stream<vec>(base + s_to[i], v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < MAXW; ++i)
          if (i < n) set<vec>(base + s_to[i], v[i]);
      }
    } else if (a.unit) {  // beyond some row's tokens
      if (a.unit == 4) ends<MAXW, B, uint32_t>(base, at, n, s_from, s_to, s_bytes);
      else if (a.unit == 2) ends<MAXW, B, uint16_t>(base, at, n, s_from, s_to, s_bytes);
      else ends<MAXW, B, uint8_t>(base, at, n, s_from, s_to, s_bytes);
    } else {
      vec v[MAXW];
#pragma unroll
      for (int i = 0; i < MAXW; ++i)
        if (i < n && at < static_cast<uint32_t>(s_bytes[i])) v[i] = get<vec>(base + s_from[i]);
#pragma unroll
      for (int i = 0; i < MAXW; ++i)
        if (i < n && at < static_cast<uint32_t>(s_bytes[i])) set<vec>(base + s_to[i], v[i]);
    }
  }
}

// ---- a cache in pages ------------------------------------------------------------------------------------

struct RowPlan {
  int src;         // the parent's row in `from`, or -1
  int len, want;   // tokens taken over, and wanted (len where they do not fit the table)
  bool fits;
};
__device__ __forceinline__ int held(const vsmp_pages& p, int row) {
  return min(max(p.lens[row], 0), p.row_pages * p.page_tokens);
}
__device__ __forceinline__ RowPlan row_plan(const PageArgs& a, int i) {
  RowPlan r;
  r.src = a.parent ? a.parent[i] : i;
  if (r.src < 0 || r.src >= a.from.rows) r.src = -1;
  r.len = r.src >= 0 ? held(a.from, r.src) : 0;
  const long long want = max(static_cast<long long>(r.len) + (a.add ? a.add[i] : a.add_all), 0ll);
  r.fits = want <= static_cast<long long>(a.to.row_pages) * a.to.page_tokens;
  r.want = r.fits ? static_cast<int>(want) : r.len;
  return r;
}
__device__ __forceinline__ int pages_of(int tokens, int page_tokens) { return (tokens + page_tokens - 1) / page_tokens; }
__device__ __forceinline__ bool is_page(int p, int n) { return static_cast<unsigned>(p) < static_cast<unsigned>(n); }

// The next tables, as far as pages are taken over; what each page gains in holders; for begun pages the rows that grow in
// them. Integer atomics, whose order does not matter, where a row's old page and its new one differ: the pages that a
// row shares with its parent cost none.
__global__ __launch_bounds__(kNt) void k_pages_fork(PageArgs a) {
  const int i = blockIdx.x, T = a.to.page_tokens, P = a.to.n_pages;
  RowPlan r{-1, 0, 0, true};
  if (i < a.to.rows) r = row_plan(a, i);
  const int keep = pages_of(min(r.len, r.want), T), had = i < a.from.rows ? pages_of(held(a.from, i), T) : 0;
  const int* take = a.from.table + max(r.src, 0) * a.from.ldt;
  const int* old = a.from.table + i * a.from.ldt;
  int* out = a.to.table + i * a.to.ldt;
  const int n = i < a.to.rows ? a.to.row_pages : had;
  for (int j = threadIdx.x; j < n; j += kNt) {
    const int was = j < had ? old[j] : -1, now = j < keep ? take[j] : -1;
    if (was != now) {
      if (is_page(was, P)) agent_add(&a.s.delta[was], -1);
      if (is_page(now, P)) agent_add(&a.s.delta[now], 1);
    }
    if (i < a.to.rows) out[j] = now;
    if (j == r.len / T && r.want > r.len && r.len % T && is_page(now, P)) {
      agent_add(&a.s.writers[now], 1);
      __hip_atomic_fetch_max(&a.s.order[now], static_cast<unsigned long long>(r.len) << 32 | static_cast<uint32_t>(~i), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

constexpr int kTakeNt = 1024;
constexpr int kTakePages = 4 * kTakeNt;  // pages of a workgroup

// Sums over the lanes up to this one (row shifts by 1, 2, 4 and 8, then the rows' sums handed on).
__device__ __forceinline__ int scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
// Of K numbers a thread: their sums over the workgroup's threads before this one; total: over all.
template <int K>
__device__ __forceinline__ void scan_before(int (&v)[K], int (&total)[K]) {
  __shared__ int s_sum[K][kTakeNt / 64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int at[K];
#pragma unroll
  for (int k = 0; k < K; ++k) at[k] = scan64(v[k]);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (lane == 63) s_sum[k][wv] = at[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int sums = scan64(lane < kTakeNt / 64 ? s_sum[k][lane] : 0);
    total[k] = __builtin_amdgcn_readlane(sums, kTakeNt / 64 - 1);
    v[k] = at[k] - v[k] + (wv ? __builtin_amdgcn_readlane(sums, wv - 1) : 0);
  }
}
__device__ __forceinline__ int scan_before(int v, int* total) {
  int a[1] = {v}, t[1];
  scan_before<1>(a, t);
  *total = t[0];
  return a[0];
}

// The free page of rank k goes to the row that asks for the k-th page: a wave takes a word, a lane a page. start: pages
// that the rows before a row ask for; first: where in the table its new pages begin; before: free pages before each word.
template <int NT, class Bits>
__device__ __forceinline__ void give_pages(const PageArgs& a, int words, int asked, int n_free, const int* start, const int* first,
                                           const int* before, Bits bits) {
  const int lane = threadIdx.x & 63, R = a.to.rows;
  for (int w = threadIdx.x >> 6; w < words && before[w] < asked; w += NT / 64) {
    const unsigned long long b = bits(w);
    const int k = before[w] + __popcll(b & ((1ull << lane) - 1ull));
    if (!(b >> lane & 1ull) || k >= asked) continue;
    // the last row that starts at or before it: rows that ask for nothing start where the next one does
    int lo = 0, hi = R - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    if ((lo + 1 < R ? start[lo + 1] : asked) > n_free) continue;  // the row does not get all of its pages, and so none
    agent_store(&a.to.table[lo * a.to.ldt + first[lo] + (k - start[lo])], w * 64 + lane);
    agent_store(&a.to.ref[w * 64 + lane], 1);
  }
}

// The next ref, and the free pages as bits; then, in the last workgroup, what each row needs, the pages it gets, lens,
// ok and the list of copies.
__global__ __launch_bounds__(kTakeNt) void k_pages_take(PageArgs a) {
  __shared__ int s_start[kPageRows];         // pages that the rows before this one ask for
  __shared__ int s_first[kPageRows];         // where in the table a row's new pages begin
  __shared__ int s_before[kPagesMax / 64];   // free pages before each word
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, P = a.to.n_pages, T = a.to.page_tokens, R = a.to.rows;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = blockIdx.x * kTakePages + k * kTakeNt + tid;
    int ref = 1;
    if (p < P) {
      const int d = a.s.delta[p];
      ref = a.from.ref[p] + d;
      if (d) a.s.delta[p] = 0;
      agent_store(&a.to.ref[p], ref);
    }
    const unsigned long long is_free = __ballot(ref <= 0);
    if (lane == 0 && p < P) agent_store(&a.s.bits[p >> 6], is_free);
  }
  drain();
  __syncthreads();
  if (tid == 0) s_last = agent_add(a.s.tick, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  if (tid == 0) agent_store(a.s.tick, 0u);

  // the rows' needs
  long long wanted = 0;  // so far: rows may ask for more than any pool has, together for more than 32 bits hold
  int copies = 0;
  constexpr long long kNever = 1 << 30;
  int need_[kPageRows / kTakeNt];
  bool away_[kPageRows / kTakeNt];
#pragma unroll
  for (int k = 0; k < kPageRows / kTakeNt; ++k) {
    need_[k] = 0;
    away_[k] = false;
    if (k * kTakeNt >= R) continue;
    const int i = k * kTakeNt + tid;
    if (i < R) {
      const RowPlan r = row_plan(a, i);
      if (r.want > r.len) {
        const int q = r.len % T ? a.to.table[i * a.to.ldt + r.len / T] : -1;
        if (is_page(q, P))
          away_[k] = agent_load(&a.to.ref[q]) != a.s.writers[q] ||
                     a.s.order[q] != (static_cast<unsigned long long>(r.len) << 32 | static_cast<uint32_t>(~i));
        s_first[i] = pages_of(r.len, T) - away_[k];
        need_[k] = pages_of(r.want, T) - s_first[i];
      }
    }
    // (a need of more than a pool is as good as any that no pool meets: 1,024 of them fit 31 bits)
    int total;
    need_[k] = min(need_[k], kPagesMax + 1);
    const int at = scan_before(need_[k], &total);
    if (i < R) s_start[i] = static_cast<int>(min(wanted + at, kNever));
    wanted += total;
  }
  const int asked = static_cast<int>(min(wanted, kNever));
  // how many pages are free, and before each thread's words
  const int words = (P + 63) / 64, mine = (words + kTakeNt - 1) / kTakeNt;
  int count = 0;
  for (int w = tid * mine; w < min(words, (tid + 1) * mine); ++w) count += __popcll(agent_load(&a.s.bits[w]));
  int n_free;
  int rank = scan_before(count, &n_free);
  for (int w = tid * mine; w < min(words, (tid + 1) * mine); ++w) {
    s_before[w] = rank;
    rank += __popcll(agent_load(&a.s.bits[w]));
  }
#pragma unroll
  for (int k = 0; k < kPageRows / kTakeNt; ++k) {
    if (k * kTakeNt >= R) continue;
    const int i = k * kTakeNt + tid;
    bool copied = false;
    RowPlan r{};
    if (i < R) {
      r = row_plan(a, i);
      const bool given = need_[k] == 0 || (s_start[i] <= n_free && need_[k] <= n_free - s_start[i]);
      a.to.lens[i] = given ? r.want : r.len;
      if (a.ok) a.ok[i] = r.fits && given;
      copied = given && away_[k];
      if (r.want > r.len && r.len % T) {
        const int q = a.to.table[i * a.to.ldt + r.len / T];
        if (is_page(q, P)) {
          a.s.writers[q] = 0;
          a.s.order[q] = 0;
        }
      }
    }
    int total;
    const int at = scan_before(copied ? 1 : 0, &total);
    if (copied) {
      const int q = a.to.table[i * a.to.ldt + r.len / T];
      agent_add(&a.to.ref[q], -1);
      a.s.copies[copies + at] = {q, i, r.len / T, r.len % T};
    }
    copies += total;
  }
  if (tid == 0) *a.s.n_copies = copies;
  __syncthreads();
  give_pages<kTakeNt>(a, words, asked, n_free, s_start, s_first, s_before, [&](int w) { return agent_load(&a.s.bits[w]); });
}

// A step of at most kTakeNt rows over a pool of at most kSmallPages pages: workgroups that take over ref and gather the free
// pages as bits, and a last one that does the rest, a thread for each row and each word of bits. With WHOLE the tables are
// among the workgroups' work (the first a.table_wgs of them), in one launch: ref is taken over as it is, the pages whose holders
// change are listed, and the last workgroup makes them good. Without it k_pages_fork has been there, and delta is whole.
// What one workgroup writes after another has is written through to memory by both: they may not share an L2.
//
// Bound by loads that follow one another (parent, length, table entry; ticket; bits and lists; ref; the pages' stores): 4 rows
// over 256 pages 7.9 us in one workgroup, 64 rows over 2,048 pages 10.8 us, the copies a launch more. Pages that many rows
// change at once cost the last workgroup scattered loads and stores (256 rows of which 16 end, 1,300 pages: 19 us); there,
// beyond kSmallEntries table entries, the tables have a launch of their own (3.2 us and 10.4). Tables alone, calls through Python,
// which take 9.7 us at the least, in one launch and in two: 1,024 entries 9.7 and 9.7, 4,096 10.5 and 9.9, 8,192 11.7 and 10.1,
// 16,384 14.7 and 10.4, 65,536 28.6 and 11.1. So two are level or better from some 4,096 on; the limit is above that.
constexpr int kSmallPages = 64 * kTakeNt, kSmallEntries = 1 << 13;
template <bool WHOLE>
__global__ __launch_bounds__(kTakeNt) void k_pages_small(PageArgs a) {
  __shared__ unsigned long long s_bits[kTakeNt];
  __shared__ int s_before[kTakeNt], s_start[kTakeNt], s_first[kTakeNt];
  __shared__ int s_list[WHOLE ? 2 * kTakeNt : 1];  // alone: the pages whose holders change, at most two an entry
  __shared__ int s_last, s_copies, s_changes;
  const int tid = threadIdx.x, lane = tid & 63, P = a.to.n_pages, T = a.to.page_tokens, R = a.to.rows, words = (P + 63) / 64;
  const bool alone = WHOLE && gridDim.x == 1;  // nothing to hand over
  if (alone) {
    if (tid == 0) s_changes = 0;
    __syncthreads();
  }
  // The pages of this workgroup, all of them if it is alone: what does not wait for other loads is loaded first.
  const int wg = static_cast<int>(blockIdx.x) - a.table_wgs, pages = (alone ? 1 : gridDim.x - a.table_wgs) * kTakeNt;
  int p0 = alone ? tid & ~63 : wg >= 0 ? (wg * kTakeNt + tid) & ~63 : P;
  auto load_ref = [&](int p) { return p < P ? a.from.ref[p] : 1; };
  auto load_delta = [&](int p) { return !WHOLE && p < P ? a.s.delta[p] : 0; };
  int ref = load_ref(p0 + lane), gain = load_delta(p0 + lane);
  // its table entries: those of `to`, and the rows beyond it that `from` has
  const uint32_t cap = static_cast<uint32_t>(a.to.row_pages);
  const uint32_t entries = WHOLE ? static_cast<uint32_t>(max(a.from.rows, R)) * cap : 0u, step = (alone ? 1 : a.table_wgs) * kTakeNt;
  for (uint32_t e0 = wg < 0 || alone ? (blockIdx.x * kTakeNt + tid) & ~63u : entries; e0 < entries; e0 += step) {
    const uint32_t e = min(e0 + lane, entries - 1);
    const int i = static_cast<int>(divide(e, cap, a.m_cap)), j = static_cast<int>(e - static_cast<uint32_t>(i) * cap);
    const bool mine = e0 + lane < entries;
    RowPlan o{-1, 0, 0, true};
    if (i < R) o = row_plan(a, i);
    const int keep = pages_of(min(o.len, o.want), T), had = i < a.from.rows ? pages_of(held(a.from, i), T) : 0;
    const int was = mine && j < had ? a.from.table[i * a.from.ldt + j] : -1;
    const int now = mine && j < keep ? a.from.table[o.src * a.from.ldt + j] : -1;
    if (mine && i < R) agent_store(&a.to.table[i * a.to.ldt + j], now);
    const bool gone = was != now && is_page(was, P), come = was != now && is_page(now, P);
    const unsigned long long at_gone = __ballot(gone), at_come = __ballot(come), lower = (1ull << lane) - 1ull;
    const int n_gone = __popcll(at_gone), n_both = n_gone + __popcll(at_come);
    if (n_both) {
      int to = 0;
      if (lane == 0) to = alone ? atomicAdd(&s_changes, n_both) : agent_add(a.s.n_moves, n_both);
      to = __builtin_amdgcn_readfirstlane(to);
      auto change = [&](int page, int at, int by) {
        agent_add(&a.s.delta[page], by);
        if (alone) s_list[at] = page;
        else agent_store(&a.s.moves[at], page);
      };
      if (gone) change(was, to + __popcll(at_gone & lower), -1);
      if (come) change(now, to + n_gone + __popcll(at_come & lower), 1);
    }
    if (mine && j == o.len / T && o.want > o.len && o.len % T && is_page(now, P)) {
      agent_add(&a.s.writers[now], 1);
      __hip_atomic_fetch_max(&a.s.order[now], static_cast<unsigned long long>(o.len) << 32 | static_cast<uint32_t>(~i), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // this thread's row in the last workgroup, and the begun page that it grows in
  RowPlan r{-1, 0, 0, true};
  int begun = -1;
  if (tid < R) {
    r = row_plan(a, tid);
    if (r.want > r.len && r.len % T) begun = a.from.table[r.src * a.from.ldt + r.len / T];
    if (!is_page(begun, P)) begun = -1;
  }
  for (; p0 < P; p0 += pages) {
    ref += gain;
    const unsigned long long is_free = __ballot(ref <= 0);
    if (p0 + lane < P) agent_store(&a.to.ref[p0 + lane], ref);
    if (gain) a.s.delta[p0 + lane] = 0;
    if (lane == 0) {
      if (alone) s_bits[p0 >> 6] = is_free;
      else agent_store(&a.s.bits[p0 >> 6], is_free);
    }
    ref = load_ref(p0 + pages + lane);
    gain = load_delta(p0 + pages + lane);
  }
  drain();
  __syncthreads();
  if (!alone) {
    if (tid == 0) s_last = agent_add(a.s.tick, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!s_last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (tid == 0) agent_store(a.s.tick, 0u);
  }

  int writers = 0;
  unsigned long long order = 0;
  if (begun >= 0) {
    writers = agent_load(&a.s.writers[begun]);
    order = agent_load(&a.s.order[begun]);
  }
  const int changes = alone ? s_changes : WHOLE ? agent_load(a.s.n_moves) : 0;
  if (!alone && tid < words) s_bits[tid] = agent_load(&a.s.bits[tid]);
  if (tid == 0) s_copies = 0;
  __syncthreads();
  if (WHOLE && !alone && tid == 0) agent_store(a.s.n_moves, 0);
  for (int t0 = 0; t0 < changes; t0 += 4 * kTakeNt) {
    int p[4], d[4], was[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + k * kTakeNt + tid;
      p[k] = t >= changes ? -1 : alone ? s_list[min(t, 2 * kTakeNt - 1)] : agent_load(&a.s.moves[t]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      d[k] = p[k] >= 0 ? agent_load(&a.s.delta[p[k]]) : 0;
      was[k] = a.from.ref[max(p[k], 0)];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!d[k]) continue;  // a page listed before, or one that as many give up as take
      // (where a page is listed again, another thread may do the same beside this one)
      const int ref = was[k] + d[k];
      agent_store(&a.s.delta[p[k]], 0);
      agent_store(&a.to.ref[p[k]], ref);
      if (was[k] > 0 && ref <= 0) atomicOr(&s_bits[p[k] >> 6], 1ull << (p[k] & 63));
      if (was[k] <= 0 && ref > 0) atomicAnd(&s_bits[p[k] >> 6], ~(1ull << (p[k] & 63)));
    }
  }
  drain();
  __syncthreads();
  const bool away = begun >= 0 && (agent_load(&a.to.ref[begun]) != writers ||
                                   order != (static_cast<unsigned long long>(r.len) << 32 | static_cast<uint32_t>(~tid)));
  // (a need of more than the pool has is as good as any that it does not meet: 1,024 of them fit 31 bits)
  const int first = pages_of(r.len, T) - away, need = r.want > r.len ? min(pages_of(r.want, T) - first, kSmallPages + 1) : 0;
  int sum[2] = {need, tid < words ? static_cast<int>(__popcll(s_bits[tid])) : 0}, all[2];
  scan_before<2>(sum, all);
  const int asked = all[0], n_free = all[1], start = sum[0], before = sum[1];
  if (tid < words) s_before[tid] = before;
  if (tid < R) {
    s_start[tid] = start;
    s_first[tid] = first;
    const bool given = need == 0 || start + need <= n_free;
    a.to.lens[tid] = given ? r.want : r.len;
    if (a.ok) a.ok[tid] = r.fits && given;
    if (begun >= 0) {
      a.s.writers[begun] = 0;
      a.s.order[begun] = 0;
    }
    if (given && away) {
      agent_add(&a.to.ref[begun], -1);
      a.s.copies[atomicAdd(&s_copies, 1)] = {begun, tid, r.len / T, r.len % T};
    }
  }
  __syncthreads();
  if (tid == 0) *a.s.n_copies = s_copies;
  give_pages<kTakeNt>(a, words, asked, n_free, s_start, s_first, s_before, [&](int w) { return s_bits[w]; });
}

// Tokens of a page into another page of a plane: a wave's chunk, four 16-byte columns a lane. The columns of all pieces
// follow one another. Bound by reads and writes together: of 10,007 pages of 8 KB in 56 planes some 2,480 move, 2.26 GB, 477
// us (4.7 TB/s); by workgroups of one plane's 16 KB 474, of several planes' (each lane loads its plane's address first) 512.
constexpr int kChunk = kPageChunk;
__device__ __forceinline__ uint32_t chunks_of(const PlaneArgs& c, int tokens) {
  const uint32_t cols = (static_cast<uint32_t>(tokens) * static_cast<uint32_t>(c.token_bytes) + 15) / 16;
  return (cols * static_cast<uint32_t>(c.pieces) + kChunk - 1) / kChunk;
}
template <bool STREAM>
__device__ __forceinline__ void copy_tokens(const PlaneArgs& c, uint32_t plane, int src, int dst, int tokens, uint32_t chunk) {
  typedef Column<16> vec;
  const uint32_t run = static_cast<uint32_t>(tokens) * static_cast<uint32_t>(c.token_bytes);
  const uint32_t cols = (run + 15) / 16, m = 0xFFFFFFFFu / cols, total = cols * static_cast<uint32_t>(c.pieces);
  const long long there = dst * c.row_stride - src * c.row_stride;
  const Bytes* base = plane_at(c, plane) + src * c.row_stride;
  vec v[4];
  const Bytes* from[4];
  int n[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t idx = chunk * kChunk + k * 64 + (threadIdx.x & 63);
    n[k] = 0;
    if (idx < total) {
      const uint32_t piece = c.pieces == 1 ? 0u : divide(idx, cols, m), byte = (idx - piece * cols) * 16;
      from[k] = base + piece * c.piece_stride + byte;
      n[k] = static_cast<int>(min(run - byte, 16u));
      if (n[k] == 16) v[k] = get<vec>(from[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (n[k] == 16) STREAM ? stream<vec>((Bytes*)from[k] + there, v[k]) : set<vec>((Bytes*)from[k] + there, v[k]);
  // the runs' ends
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (n[k] == 0 || n[k] == 16) continue;
    Bytes* to = (Bytes*)from[k] + there;
    int b = 0;
    for (; b + 4 <= n[k]; b += 4) set<Loose<uint32_t>>(to + b, get<Loose<uint32_t>>(from[k] + b));
    for (; b < n[k]; ++b) set(to + b, get<uint8_t>(from[k] + b));
  }
}

// What wave `unit` of a copy does: unit = (page * planes + plane) * chunks + chunk.
struct CopyUnit {
  uint32_t page, plane, chunk;
};
__device__ __forceinline__ CopyUnit copy_unit(const PageArgs& a, uint32_t unit, uint32_t chunks) {
  const uint32_t at = divide(unit, chunks, a.m_chunks), planes = static_cast<uint32_t>(a.cache.n_planes), page = divide(at, planes, a.m_planes);
  return {page, at - page * planes, unit - at * chunks};
}
__device__ __forceinline__ uint32_t wave_of_grid() { return __builtin_amdgcn_readfirstlane(blockIdx.x * (kNt / 64) + (threadIdx.x >> 6)); }

__global__ __launch_bounds__(kNt) void k_page_copy(PageArgs a) {
  const uint32_t chunks = chunks_of(a.cache, a.cache.tokens);
  const uint32_t total = static_cast<uint32_t>(*a.s.n_copies) * static_cast<uint32_t>(a.cache.n_planes) * chunks;
  for (uint32_t u = wave_of_grid(); u < total; u += gridDim.x * (kNt / 64)) {
    const CopyUnit w = copy_unit(a, u, chunks);
    const PageCopy c = a.s.copies[w.page];
    if (w.chunk < chunks_of(a.cache, c.tokens)) copy_tokens<false>(a.cache, w.plane, c.src, a.to.table[c.row * a.to.ldt + c.at], c.tokens, w.chunk);
  }
}

// ---- compaction ------------------------------------------------------------------------------------------

// The pages in use as bits; in the last workgroup, how many are in use before each word; of a small pool also the lists of
// k_pages_pair.
__global__ __launch_bounds__(kTakeNt) void k_pages_scan(PageArgs a) {
  __shared__ unsigned long long s_bits[kTakeNt];
  __shared__ int s_before[kTakeNt + 1];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, P = a.to.n_pages;
  const bool alone = gridDim.x == 1, small = P <= kSmallPages;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = blockIdx.x * kTakePages + k * kTakeNt + tid;
    const unsigned long long used = __ballot(p < P && a.from.ref[min(p, P - 1)] > 0);
    if (lane == 0 && p < P) {
      agent_store(&a.s.bits[p >> 6], used);
      if (alone) s_bits[p >> 6] = used;
    }
  }
  if (!alone) {
    drain();
    __syncthreads();
    if (tid == 0) s_last = agent_add(a.s.tick, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!s_last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    if (tid == 0) agent_store(a.s.tick, 0u);
  } else {
    __syncthreads();
  }
  const int words = (P + 63) / 64;
  if (small) {
    unsigned long long b = 0;
    if (tid < words) b = alone ? s_bits[tid] : agent_load(&a.s.bits[tid]);
    int n;
    const int at = scan_before(__popcll(b), &n);
    if (tid < words) {
      s_bits[tid] = b;
      s_before[tid] = at;
      a.s.before[tid] = at;
    }
    if (tid == 0) {
      a.s.before[words] = n;
      if (a.live) *a.live = n;
    }
    __syncthreads();
    // a wave takes a word, a lane a page
    const int kept = n < P ? s_before[n >> 6] + __popcll(s_bits[n >> 6] & ((1ull << (n & 63)) - 1ull)) : n;
    for (int w = tid >> 6; w < words; w += kTakeNt / 64) {
      const unsigned long long bits = s_bits[w];
      const int p = w * 64 + lane, below = s_before[w] + __popcll(bits & ((1ull << lane) - 1ull));
      const bool used = bits >> lane & 1ull;
      if (p < n && !used) a.s.room[p - below] = p;
      if (p >= n && used) a.s.moves[below - kept] = p;
    }
    return;
  }
  const int mine = (words + kTakeNt - 1) / kTakeNt;
  int count = 0;
  for (int w = tid * mine; w < min(words, (tid + 1) * mine); ++w) count += __popcll(agent_load(&a.s.bits[w]));
  int total;
  int at = scan_before(count, &total);
  for (int w = tid * mine; w < min(words, (tid + 1) * mine); ++w) {
    a.s.before[w] = at;
    at += __popcll(agent_load(&a.s.bits[w]));
  }
  if (tid == 0) {
    a.s.before[words] = total;
    if (a.live) *a.live = total;
  }
}

// Pages in use below page p.
__device__ __forceinline__ int used_before(const PageArgs& a, int p) {
  return a.s.before[p >> 6] + __popcll(a.s.bits[p >> 6] & ((1ull << (p & 63)) - 1ull));
}
__device__ __forceinline__ bool is_used(const PageArgs& a, int p) { return a.s.bits[p >> 6] >> (p & 63) & 1ull; }

// The pages in use at n and beyond, and the free ones below n, in order.
__global__ __launch_bounds__(kNt) void k_pages_pair(PageArgs a) {
  const int p = blockIdx.x * kNt + threadIdx.x, P = a.to.n_pages;
  if (p >= P) return;
  const int n = a.s.before[(P + 63) / 64], below = used_before(a, p);
  if (p < n && !is_used(a, p)) a.s.room[p - below] = p;
  if (p >= n && is_used(a, p)) a.s.moves[below - used_before(a, n)] = p;
}

__device__ __forceinline__ int moved_to(const PageArgs& a, int p, int n, int kept) {
  return p < n ? p : a.s.room[used_before(a, p) - kept];
}

// Tables, ref and moved; the pages' tokens.
__global__ __launch_bounds__(kNt) void k_pages_move(PageArgs a) {
  const int P = a.to.n_pages, T = a.to.page_tokens, n = a.s.before[(P + 63) / 64];
  const int kept = n < P ? used_before(a, n) : n;  // pages in use below n
  const int moves = n - kept;
  // small work first: tables by rows, then the pool
  for (int i = blockIdx.x; i < a.to.rows; i += gridDim.x) {
    const int len = held(a.from, i), used = pages_of(len, T);
    for (int j = threadIdx.x; j < a.to.row_pages; j += kNt) {
      int p = -1;
      if (j < used) {
        p = a.from.table[i * a.from.ldt + j];
        if (is_page(p, P)) p = is_used(a, p) ? moved_to(a, p, n, kept) : -1;
      }
      a.to.table[i * a.to.ldt + j] = p;
    }
    if (threadIdx.x == 0) a.to.lens[i] = len;
  }
  for (int p = blockIdx.x * kNt + threadIdx.x; p < P; p += gridDim.x * kNt) {
    const bool used = is_used(a, p);
    const int to = used ? moved_to(a, p, n, kept) : -1;
    if (a.moved) a.moved[p] = to;
    if (used) a.to.ref[to] = a.from.ref[p];
    if (p >= n) a.to.ref[p] = 0;
  }
  if (!a.cache.n_planes) return;
  const uint32_t chunks = chunks_of(a.cache, a.cache.tokens);
  const uint32_t total = static_cast<uint32_t>(moves) * static_cast<uint32_t>(a.cache.n_planes) * chunks;
  for (uint32_t u = wave_of_grid(); u < total; u += gridDim.x * (kNt / 64)) {
    const CopyUnit w = copy_unit(a, u, chunks);
    copy_tokens<true>(a.cache, w.plane, a.s.moves[w.page], a.s.room[w.page], a.cache.tokens, w.chunk);
  }
}

template <int MAXW, int B>
void go_reorder(const ReorderArgs& a, int groups, int blocks, hipStream_t st) {
  hipLaunchKernelGGL((k_reorder<MAXW, B>), dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(groups)), dim3(kNt), 0, st, a);
}

}  // namespace

void launch_reorder(ReorderArgs a, int groups, int cus, hipStream_t st) {
  const int bytes = a.width <= 32 ? 16 : 8;
  a.unit = a.p.token_bytes % bytes == 0 ? 0 : a.p.token_bytes % 4 == 0 ? 4 : a.p.token_bytes % 2 == 0 ? 2 : 1;
  const long long cols = (static_cast<long long>(a.p.tokens) * a.p.token_bytes + bytes - 1) / bytes * a.p.n_planes * a.p.pieces;
  const long long most = (cols + kNt - 1) / kNt;
  a.streams = cols * bytes * a.width * groups > 512ll << 20;
  const int blocks = static_cast<int>(std::max<long long>(1, std::min<long long>(most, (64ll * cus + groups - 1) / groups)));
  if (a.width <= 4) go_reorder<4, 16>(a, groups, blocks, st);
  else if (a.width <= 8) go_reorder<8, 16>(a, groups, blocks, st);
  else if (a.width <= 16) go_reorder<16, 16>(a, groups, blocks, st);
  else if (a.width <= 32) go_reorder<32, 16>(a, groups, blocks, st);
  else go_reorder<64, 8>(a, groups, blocks, st);
}

// Workgroups for the copies of up to n pages, at most `most`, and what the waves divide by.
static unsigned copy_wgs(PageArgs& a, int n, int most) {
  const long long cols = (static_cast<long long>(a.cache.tokens) * a.cache.token_bytes + 15) / 16 * a.cache.pieces;
  const long long chunks = (cols + kChunk - 1) / kChunk;
  a.m_chunks = 0xFFFFFFFFu / static_cast<uint32_t>(chunks);
  a.m_planes = 0xFFFFFFFFu / static_cast<uint32_t>(a.cache.n_planes);
  return static_cast<unsigned>(std::min<long long>(most, (chunks * a.cache.n_planes * n + kNt / 64 - 1) / (kNt / 64)));
}

void launch_pages_step(PageArgs a, int cus, hipStream_t st) {
  const int rows = std::max(a.from.rows, a.to.rows);
  const long long entries = static_cast<long long>(rows) * a.to.row_pages;
  const bool small = rows <= kTakeNt && a.to.n_pages <= kSmallPages;
  const int wgs = (a.to.n_pages + kTakeNt - 1) / kTakeNt;  // 64 at most of a small pool
  if (small && entries <= kSmallEntries) {
    a.m_cap = 0xFFFFFFFFu / static_cast<uint32_t>(a.to.row_pages);
    a.table_wgs = static_cast<int>((entries + kTakeNt - 1) / kTakeNt);
    const bool alone = a.table_wgs == 1 && wgs == 1;
    hipLaunchKernelGGL(k_pages_small<true>, dim3(static_cast<unsigned>(alone ? 1 : a.table_wgs + wgs)), dim3(kTakeNt), 0, st, a);
  } else {
    hipLaunchKernelGGL(k_pages_fork, dim3(static_cast<unsigned>(rows)), dim3(kNt), 0, st, a);
    if (small)
      hipLaunchKernelGGL(k_pages_small<false>, dim3(static_cast<unsigned>(wgs)), dim3(kTakeNt), 0, st, a);
    else
      hipLaunchKernelGGL(k_pages_take, dim3(static_cast<unsigned>((a.to.n_pages + kTakePages - 1) / kTakePages)), dim3(kTakeNt), 0, st, a);
  }
  if (a.cache.n_planes && (a.add || a.add_all > 0)) {
    const unsigned wgs = copy_wgs(a, a.to.rows, 16 * cus);
    hipLaunchKernelGGL(k_page_copy, dim3(wgs), dim3(kNt), 0, st, a);
  }
}

void launch_pages_compact(PageArgs a, int cus, hipStream_t st) {
  const int P = a.to.n_pages;
  hipLaunchKernelGGL(k_pages_scan, dim3(static_cast<unsigned>((P + kTakePages - 1) / kTakePages)), dim3(kTakeNt), 0, st, a);
  if (P > kSmallPages) hipLaunchKernelGGL(k_pages_pair, dim3(static_cast<unsigned>((P + kNt - 1) / kNt)), dim3(kNt), 0, st, a);
  unsigned wgs = std::min(static_cast<unsigned>(std::max(a.to.rows, (P + kNt - 1) / kNt)), 4u * cus);  // tables and pool
  if (a.cache.n_planes) wgs = std::max(wgs, copy_wgs(a, P / 2 + 1, 16 * cus));
  hipLaunchKernelGGL(k_pages_move, dim3(wgs), dim3(kNt), 0, st, a);
}

}  // namespace vsmp
