/*
 * vsmp_logits — the operators around the pick, on AMD Instinct MI355X (gfx950): the LM head's product
 * with 4-bit weights, logits adjusted before the pick (penalties, biases, grammar masks), and the
 * log-probabilities of what was picked. Together with vsmp_pick_batch they make one serving step:
 *
 *   vsmp_head_logits_q4 -> vsmp_adjust_logits -> vsmp_pick_batch -> vsmp_logprobs
 *
 * None has a counterpart in the reference's sampler, whose one adjustment is the multiplicative
 * penalty (reference src/sampler.cpp:53-65); vsmp_adjust_logits applies that rule to the bit, so a
 * caller sets it there or in vsmp_params, not in both.
 *
 * Conventions are vsmp.h's: 0 on success and -1 on error with a per-thread message; device pointers;
 * stream-ordered, without host synchronisation; calls that share a context (replays of graphs that
 * captured them included) are issued in order. Logits of the dtype codes below are converted to fp32
 * exactly; rows need no alignment beyond that of their elements unless a call says otherwise.
 */
#ifndef VSMP_LOGITS_H
#define VSMP_LOGITS_H

#include "vsmp.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of logits, hidden states and scales. */
typedef enum { VSMP_F32 = 0, VSMP_BF16 = 1, VSMP_F16 = 2 } vsmp_dtype;

/* One row's penalties (16 bytes). `window`: how many of the history's last ids count (<= 0: all). */
typedef struct {
  float repeat;    /* seen logits: x / repeat where x > 0, else x * repeat; 1: off; > 0 */
  float presence;  /* subtracted once from a logit whose id was generated */
  float frequency; /* subtracted for each time that its id was generated */
  int window;
} vsmp_penalty;

/* Logits made ready for the pick. For every row r and id i, with x the row's logit in fp32:
 *   y = x
 *   i in the row's window:                  y = x > 0 ? x / repeat : x * repeat
 *   i in it c > 0 times after the prompt:   y = y - (presence + frequency * c)
 *   i among the row's biased ids:           y = y + bias (of the last entry that names i)
 *   x = -inf stays -inf; an id that the row's mask forbids gets -inf whatever its logit (NaN included)
 * each step rounded to fp32. Ids outside [0, V) in histories and biases are ignored.
 *   in, dtype, ldi: device logits, row r at element r * ldi (ldi >= V).
 *   pen, pen_per_row: NULL for no penalties; 0 -> a HOST pointer to one struct used by every row;
 *       1 -> a DEVICE array of B structs (aligned to 4 bytes).
 *   hist, hist_off: device CSR of histories, oldest first, as vsmp_pick_batch's; both NULL for none.
 *   prompt_len: device int[B], the number of ids at the start of row r's history that are its prompt
 *       (they count for `repeat` alone), or NULL for 0.
 *   bias_ids, bias, bias_off: device CSR of (id, bias) entries, bias_off with B + 1 offsets; all NULL
 *       for none.
 *   mask, ldm, n_masks, mask_row: a device table of n_masks masks, mask m at word m * ldm
 *       (ldm >= ceil(V / 32) words of 32 bits; bit i % 32 of word i / 32 set: id i is allowed), and
 *       device int[B] with each row's mask in it (negative: the row is not masked; n_masks or more:
 *       nothing is allowed), or NULL where row r's mask is mask r (n_masks >= B). mask NULL for none.
 *   out, ldo: device fp32 [B][ldo], ldo >= V: `in` itself with ldi = ldo (fp32), or memory that does
 *       not overlap it (apart as a whole, or rows between its rows at the same stride in bytes). Columns V .. ldo - 1 are left as they are. (vsmp_pick_batch reads it where it
 *       is 16-byte aligned with ldo a multiple of 4.)
 *   left: NULL, or device int[B]: how many of the row's ids have y > -inf. A row with 0 has nothing to
 *       pick from (vsmp_pick_batch is not defined on it).
 * V <= 1048576 (2^20). With `left`, the context holds about 2 MB of scratch from the first such call on;
 * a call that is captured into a graph needs one before it. Returns 0 or -1. */
VSMP_API int vsmp_adjust_logits(vsmp_ctx* ctx, const void* in, int dtype, long long ldi, int B, int V,
                                const vsmp_penalty* pen, int pen_per_row, const int* hist, const int* hist_off,
                                const int* prompt_len, const int* bias_ids, const float* bias, const int* bias_off,
                                const unsigned int* mask, long long ldm, int n_masks, const int* mask_row, float* out,
                                long long ldo, int* left, void* stream);

/* Log-probabilities under the softmax of a row of logits, and ranks in the sampler's order (value
 * descending, id ascending). For every row r, with lse[r] = log(sum_i exp(x_i)):
 *   logprob[r * n + j] = x_i - lse[r]  and  rank[r * n + j] = how many ids come before i,
 * for i = ids[r * ldj + j], j < n. An id outside [0, V) (a position that is not scored) gets -inf and
 * rank -1. Sums are taken relative to the row's largest logit in fp32. A logit of -inf has probability
 * 0; a row of nothing else has lse -inf and log-probabilities -inf. A row with a NaN or a +inf has no
 * probabilities: its lse and the log-probabilities of ids in [0, V) are NaN. Ranks count +inf as the largest
 * value; a NaN comes before no id, and an id whose logit is NaN has rank 0.
 *   logits, dtype, ld: device logits, row r at element r * ld (ld >= V). V <= 1048576 (2^20).
 *   ids, ldj, n: device int ids, 0 <= n <= 64 (0: lse alone; ids, logprob and rank unused), ldj >= n.
 *   logprob, rank: device [B][n]; rank may be NULL. lse: device float[B], may be NULL (n > 0).
 * The context holds about 2 MB of scratch from the first call on, of whatever shape; a call that is
 * captured into a graph needs one before it. Returns 0 or -1. */
VSMP_API int vsmp_logprobs(vsmp_ctx* ctx, const void* logits, int dtype, long long ld, int B, int V, const int* ids,
                           long long ldj, int n, float* logprob, int* rank, float* lse, void* stream);

/* The LM head's product with 4-bit weights:
 *   logits[r][c] = sum_d hidden[r][d] * scale[c][d / group] * (q[c][d] - zero[c][d / group])
 * for r < B, c < V, accumulated in fp32 on the matrix cores: the weights enter them as small integers,
 * unrounded, and each group's sum is scaled in fp32. Every logit is computed in the same order
 * whatever the batch.
 *   hidden, dtype, ldh: device bf16 or f16 [B][ldh], 16-byte aligned, ldh a multiple of 8 and >= D;
 *       finite values.
 *   q, ldq: device bytes [V][ldq], two weights a byte, the even d in the low half; 16-byte aligned, ldq
 *       a multiple of 16 and >= D / 2.
 *   scales, scale_dtype, lds: device [V][lds] of fp32, bf16 or f16, lds >= D / group.
 *   zeros, ldz: device bytes [V][ldz], one zero point per group (0 .. 255), ldz >= D / group; NULL: 8
 *       everywhere.
 *   ldq and ldz below 2^26, lds below 2^24.
 *   group: 32, 64 or 128. D: a multiple of group in [32, 16384]. V <= 1048576 (2^20).
 *   logits, ldl: device fp32 [B][ldl], ldl >= V.
 * Returns 0 or -1. */
VSMP_API int vsmp_head_logits_q4(vsmp_ctx* ctx, const void* hidden, int dtype, long long ldh, const void* q,
                                 long long ldq, const void* scales, int scale_dtype, long long lds,
                                 const unsigned char* zeros, long long ldz, int group, int B, int V, int D,
                                 float* logits, long long ldl, void* stream);

/* vsmp_adjust_logits for the live slots of a batch of sequences, between vsmp_head_logits* and
 * vsmp_bsampler_pick_rows: row i of the call belongs to slot rows[i] (device array of n_rows distinct
 * slots; NULL: row i is slot i, n_rows = the sampler's slots) and is penalised by that slot's history
 * on the device. The rest is vsmp_adjust_logits's with B = n_rows, per-row arrays by row of the call.
 * Where the slot's repeat_last is above 0 its window is at most that: a pen.window of 0 or less, or of
 * more, counts repeat_last ids, whatever the slot happens to keep beyond them. prompt_len counts from the
 * first id that the sequence accepted (its prompt's, with vsmp_bsampler_admit), also after the slot has
 * dropped it. n_rows = 0 does nothing. Returns 0 or -1. */
VSMP_API int vsmp_bsampler_adjust_rows(vsmp_bsampler* s, const void* in, int dtype, long long ldi, int V,
                                       const int* rows, int n_rows, const vsmp_penalty* pen, int pen_per_row,
                                       const int* prompt_len, const int* bias_ids, const float* bias,
                                       const int* bias_off, const unsigned int* mask, long long ldm, int n_masks,
                                       const int* mask_row, float* out, long long ldo, int* left, void* stream);

#ifdef __cplusplus
}
#endif

#endif
