/*
 * vsmp_beam — beams and the states behind them, on AMD Instinct MI355X (gfx950): one step of beam search over
 * rows of logits, and what lets a sequence go on from another's state: rows of states that follow their
 * beams, and a cache in pages that rows share, fork, grow, copy on write, give back and compact.
 * A step of a search is
 *
 *   vsmp_beam_select -> vsmp_reorder_rows (states held row by row) or vsmp_pages_step (states held in pages)
 *
 * None has a counterpart in the reference, which decodes one sequence at a time (reference
 * src/sampler.cpp:111-181).
 *
 * Conventions are vsmp.h's: 0 on success and -1 on error with a per-thread message; device pointers;
 * stream-ordered, without host synchronisation; calls that share a context (replays of graphs that
 * captured them included) are issued in order. What a call writes does not overlap what it reads unless it
 * says so.
 */
#ifndef VSMP_BEAM_H
#define VSMP_BEAM_H

#include "vsmp_logits.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One step of beam search for G groups (searches) of W rows (beams) each, row g * W + b being beam b of group
 * g. A row is live if its score is finite and so is lse, the log of the sum of the exponentials of its logits (a
 * row of -inf alone is not live, nor is one with a NaN or a +inf). The continuations of a group are its live
 * rows' tokens with a logit x above -inf, each with
 *   s = score + (x - lse)
 * in 64 bits (the exponentials are added up in 32 bits within a wave, in 64 beyond), in the order of s descending, beam
 * ascending, x descending, token ascending.
 *   logits, dtype, ld: device logits (vsmp_dtype), row r at element r * ld (ld >= V), aligned to their elements.
 *       V <= 1048576 (2^20).
 *   scores: device float[G * W].
 *   N: beams of the next step, 1 <= N <= 64 (1 <= W <= 64; N is not W where one row becomes several).
 *   stop_ids, n_stop: HOST array of at most 16 tokens that end a sequence (those outside [0, V) end nothing).
 *   token, parent, score: device [G][N], the first N continuations that no stop token makes: their tokens, their
 *       rows (g * W + b) and s rounded to fp32. An entry i beyond the last continuation gets token -1, parent
 *       g * W + i mod W and score -inf: a row that is not live in the next step.
 *   end_token, end_parent, end_score, n_end: device [G][N] and [G], or all NULL: the stop tokens among the group's
 *       first N continuations of all, and how many they are; entries beyond as above.
 * The context holds about 3 MB of scratch from the first call on; a call that is captured into a graph needs one
 * before it. Returns 0 or -1. */
VSMP_API int vsmp_beam_select(vsmp_ctx* ctx, const void* logits, int dtype, long long ld, int G, int W, int V,
                              const float* scores, int N, const int* stop_ids, int n_stop, int* token, int* parent,
                              float* score, int* end_token, int* end_parent, float* end_score, int* n_end, void* stream);

/* Tensors ("planes": the keys of a layer, its values, ...) of the same shape whose rows hold tokens: token t of
 * piece k of row r lies at planes[p] + r * row_stride + k * piece_stride + t * token_bytes, all in bytes. Planes do not
 * overlap, nor do rows and pieces: pieces lie within their rows, or rows within pieces. */
typedef struct {
  void* const* planes;    /* DEVICE array of n_planes addresses */
  int n_planes;
  int rows;               /* rows of a plane */
  long long row_stride;
  int pieces;             /* runs of tokens a row has (heads that lie apart, or 1) */
  long long piece_stride; /* unused with one piece */
  int tokens;             /* room of a piece */
  int token_bytes;        /* tokens * token_bytes < 2^31 */
} vsmp_planes;

/* Rows follow their beams, in place, in every plane: in each group of `width` rows (1 <= width <= 64; planes->rows a
 * multiple of it) row i takes what row parent[i] held before the call.
 *   parent: device int[rows], row numbers of the planes. A row whose parent is itself or lies outside its group
 *       stays as it is.
 *   len: device int[rows], the tokens that each row held before the call, or NULL for all: the first
 *       len[parent[i]] tokens of each piece are taken, what lies behind them in row i is left as it is.
 * Rows are moved whole, whatever their type; any alignment. Returns 0 or -1. */
VSMP_API int vsmp_reorder_rows(vsmp_ctx* ctx, const vsmp_planes* planes, const int* parent, int width, const int* len,
                               void* stream);

/* A cache in pages as its rows use it: row r holds lens[r] tokens in its first ceil(lens[r] / page_tokens) table
 * entries. All arrays are the caller's, in device memory. */
typedef struct {
  int rows;          /* 1 .. 8192 */
  int row_pages;     /* room of a row; row_pages * page_tokens <= 2^30 */
  int n_pages;       /* pages of the pool, 1 .. 1048576 (2^20) */
  int page_tokens;   /* tokens of a page */
  int* table;        /* [rows][ldt] page numbers; one outside [0, n_pages) stands for no page */
  long long ldt;     /* >= row_pages */
  int* lens;         /* [rows]; below 0 or above the row's room: taken for 0 or that room */
  int* ref;          /* [n_pages]: how many hold the page: rows, and the caller, who may add to it. <= 0: free */
} vsmp_pages;

/* One step of a cache in pages, from the state *from, which stays as it is, to the state *to. Row i of `to` takes the
 * L = lens[parent[i]] tokens of its parent, sharing its pages, and then
 *   add[i] < 0: is cut by as many (to 0 at the least) and gives up the pages behind them;
 *   add[i] > 0: gets room for as many. Pages are the pool's free ones, lowest first, to the rows in ascending order. A
 *       page that the row has begun (L no multiple of page_tokens) is written next, so that it must be the row's own:
 *       if all that hold it are rows that grow in it in this step, the one with the most tokens (the lowest row among
 *       those) keeps it; every other row, and all of them if anyone else holds it, gets a page of its own, into
 *       which the begun page's tokens are copied in every plane of `cache`.
 * A row for which there are not enough free pages left after what the rows before it ask for, or not enough room in the
 * table, holds its parent's L tokens and shares its pages (ok 0). What a row asks for in vain counts for the rows behind
 * it: from the first one on that the pool has too few pages for, all that need a page get none in this step (rows that
 * need none go on; a row without room in the table asks for none). So a prompt that may not fit goes into the last
 * rows, or into a step of its own.
 *   from, to: HOST pointers; the same n_pages and page_tokens, to->row_pages >= from->row_pages, no array of one
 *       overlapping the other's. to->table is written whole (-1 behind a row's pages), as are to->lens and to->ref.
 *       A page that only rows given up in this step held is free in it, and may be given out and written again.
 *   parent: device int[to->rows], rows of `from`; outside [0, from->rows): the row starts empty. NULL: row i's
 *       parent is row i.
 *   add: device int[to->rows], or NULL for add_all everywhere.
 *   cache: HOST pointer to the planes whose rows are the pages (rows = n_pages, tokens = page_tokens), or NULL where
 *       the caller copies by itself or has nothing to copy. Half of the pool's pages, and a page of each row, hold fewer
 *       than 2^31 pieces of 4 KB (or less) in all planes.
 *   ok: device int[to->rows], or NULL.
 * Rows that no row of `to` has for its parent give up their pages; so do all those of `from` beyond to->rows. The
 * context holds about 26 MB of scratch from the first call of vsmp_pages_step or vsmp_pages_compact on; a call that is
 * captured into a graph needs one before it. Returns 0 or -1. */
VSMP_API int vsmp_pages_step(vsmp_ctx* ctx, const vsmp_pages* from, const vsmp_pages* to, const int* parent,
                             const int* add, int add_all, const vsmp_planes* cache, int* ok, void* stream);

/* A cache in pages moved together: of its n pages in use (ref > 0) those at n and beyond, in ascending order, move to the
 * free ones below n, in ascending order, in every plane of `cache`; tables and ref follow.
 *   from, to: as vsmp_pages_step's, to->rows = from->rows. `from` stays as it is, and so do its pages' tokens. A table
 *       entry whose page is not in use becomes -1.
 *   moved: device int[n_pages], or NULL: each page's new number, -1 for a page that was free (for pages that the
 *       caller holds).
 *   live: device int[1], or NULL: n.
 * The scratch is vsmp_pages_step's. Returns 0 or -1. */
VSMP_API int vsmp_pages_compact(vsmp_ctx* ctx, const vsmp_pages* from, const vsmp_pages* to, const vsmp_planes* cache,
                                int* moved, int* live, void* stream);

#ifdef __cplusplus
}
#endif

#endif
