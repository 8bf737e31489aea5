/* What a served model runs between its pinned linears, MI355X (gfx950), in
 * libglint_serve.so: queries and keys normed and turned to their positions, a paged key/value
 * cache held in 4 bits, attention over that cache for single tokens and for chunks, causal
 * attention over packed prompts, both also bounded to a window, and log probabilities of given tokens.
 * The reference keeps attention and scoring in its model harness (tests/arm0_forward.h);
 * these entry points have no counterpart in its ABI.
 *
 * The cache holds a key or value row in the codec's parent-only form: per 64 dimensions an
 * f32 absmax s and 4-bit codes h, an element standing for PARENT[h] * s, h the first
 * minimum of |w / s - PARENT[k]| (w / s in f32, 0 where s is 0; NaN is left out of the
 * absmax and takes code 0), as glint_encode.h encodes a hole. Pages hold 64 tokens of
 * every head; with NB = D / 64:
 *   k_hole   [pages][H][64][D/2] bytes: the row of a token is [4][NB][8] bytes, byte (c, b, e)
 *            holding dimension 64 b + 16 c + 2 e in its low nibble and the next one in its high;
 *   k_absmax [pages][H][NB][64] f32;
 *   v_hole   [pages][H][D/2][64] bytes: row 16 p + d, column t holds dimension 32 p + d (low
 *            nibble) and 32 p + 16 + d (high nibble) of token t;
 *   v_absmax [pages][H][NB][64] f32.
 * The place of a token is its slot, page * 64 + t.
 *
 * Return codes: 0 success, -1 null pointer, -2 shape, stride or alignment not supported,
 * -3 launch failure. All calls are asynchronous on `stream` and allocate nothing (but
 * a workspace, once per stream: see glint_serve_workspace_reserve). D is 64 or
 * 128; strides count elements, a row's D elements are adjacent. */
#ifndef GLINT_SERVE_H
#define GLINT_SERVE_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif
struct ihipStream_t;

#define GLINT_KV_PAGE 64
#define GLINT_KV_BF16 0
#define GLINT_KV_F32 1

/* Encodes T keys and values of H heads into the cache. k, v: elements of type elt
 * (GLINT_KV_BF16 or GLINT_KV_F32) at t * stride_t + h * stride_h; addresses and strides are
 * multiples of 4 elements. slots [T]: a slot outside [0, pages * 64) is skipped. Two tokens
 * with the same slot leave one of them there, or a mix of both. */
int glint_kv4_append(const void *k, const void *v, int elt, int64_t k_stride_t, int64_t k_stride_h,
                     int64_t v_stride_t, int64_t v_stride_h, const int64_t *slots, int64_t T, int H, int D,
                     uint8_t *k_hole, float *k_absmax, uint8_t *v_hole, float *v_absmax, int64_t pages,
                     struct ihipStream_t *stream);

/* The tokens of slots [T] as BF16 (round to nearest even) k, v [T][H][D]; zeros for a slot
 * outside [0, pages * 64). k, v 4-B aligned. */
int glint_kv4_gather(const int64_t *slots, int64_t T, int H, int D, const uint8_t *k_hole, const float *k_absmax,
                     const uint8_t *v_hole, const float *v_absmax, int64_t pages, uint16_t *k, uint16_t *v,
                     struct ihipStream_t *stream);

/* Attention of B sequences' newest tokens over the cache. Sequence b has lens[b] tokens in
 * the cache, token t in page table[b * table_stride + t / 64] (at most max_pages of them; a
 * page outside [0, pages) is not seen), and nq query rows: rows cu_q[b] .. cu_q[b + 1] of
 * q [Tq], at most max_q, or max_q rows each where cu_q is NULL (then Tq = B max_q). Row i of
 * its nq stands at position lens[b] - nq + i and sees the positions up to its own:
 *   out[row][hq][:] = sum_j softmax_j(scale q . k_j) v_j,   k, v of head hq / (Hq / H),
 * BF16 out [Tq][Hq][D]; a row that sees nothing is zero. Rows past max_q, or outside every
 * sequence, are left as they are. q: BF16 bits, strides multiples of 8, 16-B aligned. Scores,
 * softmax and sums are f32; PARENT and the softmax weights times the value scales enter the
 * matrix products in f16, under a power of two that follows the largest value scale met: a weight times its
 * value scale loses bits below 2^-24 of that scale, and below 2^-35, or a weight below 2^-25, adds nothing but to the
 * weights' sum. A batch whose list of work passes 2^30 goes in several launches, and
 * a sequence for which H max_q (Hq / H) max_pages / 16 does is -2.
 * Long sequences are split over workgroups that meet in a workspace of the
 * stream's (glint_serve_workspace_reserve): it is allocated by the first such call outside a
 * capture and never grows. A capture on a stream that has none runs unsplit. */
int glint_kv4_attend(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq, const uint8_t *k_hole,
                     const float *k_absmax, const uint8_t *v_hole, const float *v_absmax, int64_t pages,
                     const int32_t *table, int64_t table_stride, int max_pages, const int32_t *lens,
                     const int32_t *cu_q, int B, int max_q, int Hq, int H, int D, float scale, uint16_t *out,
                     struct ihipStream_t *stream);

/* The same, bounded: the row at position p sees the positions j up to p with j > p - window or
 * j < sinks. window 1 .. GLINT_WINDOW_MAX, or 0: no bound (sinks mean nothing then); sinks >= 0. What
 * no row of a sequence sees is not read, nor are its pages' numbers in the table, so that a caller may
 * give such pages back. */
#define GLINT_WINDOW_MAX (1 << 30)
int glint_kv4_attend_window(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq, const uint8_t *k_hole,
                            const float *k_absmax, const uint8_t *v_hole, const float *v_absmax, int64_t pages,
                            const int32_t *table, int64_t table_stride, int max_pages, const int32_t *lens,
                            const int32_t *cu_q, int B, int max_q, int Hq, int H, int D, float scale, int window,
                            int sinks, uint16_t *out, struct ihipStream_t *stream);

/* Attention of B sequences' newest tokens over the cache, for many of them a sequence: arguments and result as
 * glint_kv4_attend_window, out 16-B aligned and apart from every input. Where k and v are given [Tq], BF16, rows as
 * q's, strides multiples of 8, stride_t from D to 2^24, 16-B aligned, they are the new tokens' keys and values, and
 * what the cache holds of these tokens is not read (it need not hold them; its max_pages bound the tokens before
 * them alone; a length past 2^31 - 65 counts as that).
 * Scores, softmax and sums are f32; keys, values and softmax weights enter the matrix products in f16, 64 tokens'
 * keys under one power of two and their values under another: a held element is rounded by 2^-11 of itself, and of
 * elements below 2^-14 of the largest of the token's 64 dimensions 2^-20 of that largest may be lost. 64 tokens
 * whose values span more (2^12 and more from one token's largest to another's, or sizes past 2^+-32), or whose scores
 * might pass 2^21, enter as pairs of BF16, at some ten times the cost and a second pass over what their workgroup has:
 * what a row gives no weight, or does not see, costs it no bits. A weight below 2^-32 of its row's largest adds
 * nothing but to the weights' sum. A value that is not finite leaves itself or NaN in its dimension of the rows that
 * see it.
 * max_q (Hq / H) is at most 2^18. Few rows without own keys go as glint_kv4_attend_window does, its limits, refusals
 * and workspace included, and _scratch gives 0. scratch: 16-B aligned, at least as many bytes as _scratch gives (-2: a
 * shape that is refused) for the current device; the call's alone until it has run. */
int64_t glint_kv4_attend_chunk_scratch(int B, int max_q, int Hq, int H, int D, int max_pages, int own);
int glint_kv4_attend_chunk(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, int64_t Tq, const uint8_t *k_hole,
                           const float *k_absmax, const uint8_t *v_hole, const float *v_absmax, int64_t pages,
                           const int32_t *table, int64_t table_stride, int max_pages, const int32_t *lens,
                           const int32_t *cu_q, int B, int max_q, int Hq, int H, int D, const uint16_t *k,
                           int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v, int64_t v_stride_t,
                           int64_t v_stride_h, float scale, int window, int sinks, uint16_t *out, void *scratch,
                           int64_t scratch_bytes, struct ihipStream_t *stream);

/* The stream's workspace, 4.1 MiB on 256 CUs: one for eager calls and, once the stream was
 * captured, one for the graphs captured on it, whose replays must not overlap one another.
 * reserve allocates the eager one ahead of time (0; -1: no memory, or the stream is being
 * captured). release waits for the stream and frees both (0, or -1); graphs captured before
 * must not be replayed after it. */
int glint_serve_workspace_reserve(struct ihipStream_t *stream);
int glint_serve_workspace_release(struct ihipStream_t *stream);

/* Causal attention of B packed sequences. Sequence b has queries cu_q[b] .. cu_q[b + 1] of
 * q [Tq] (at most max_q) and keys cu_k[b] .. cu_k[b + 1] of k, v [Tk]; the last query sees
 * the last key, each earlier query one key less, and a query before the first key gives
 * zeros. Queries past max_q, or outside every sequence, are left as they are. Hq % H == 0;
 * BF16 in and out, out [Tq][Hq][D]; strides multiples of 8, k's and v's stride_t from D to 2^24,
 * addresses 16-B aligned. f32 scores, softmax and sums; the softmax weights enter the second
 * product in BF16. */
int glint_attend_prompt(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t *k,
                        int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v, int64_t v_stride_t,
                        int64_t v_stride_h, const int32_t *cu_q, const int32_t *cu_k, int64_t Tq, int64_t Tk, int B,
                        int max_q, int Hq, int H, int D, float scale, uint16_t *out, struct ihipStream_t *stream);

/* The same, bounded as glint_kv4_attend_window; positions are a sequence's keys. */
int glint_attend_prompt_window(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t *k,
                               int64_t k_stride_t, int64_t k_stride_h, const uint16_t *v, int64_t v_stride_t,
                               int64_t v_stride_h, const int32_t *cu_q, const int32_t *cu_k, int64_t Tq, int64_t Tk,
                               int B, int max_q, int Hq, int H, int D, float scale, int window, int sinks, uint16_t *out,
                               struct ihipStream_t *stream);

/* Rows of T tokens, q of Hq heads and k of H, normed (where a norm is given) and turned to the tokens'
 * positions pos [T]:
 *   x_d = row_d (1 / sqrt(mean_d row_d^2 + eps)) norm_d;
 *   pair i of the first `rot` dimensions turns by a = pos[t] freqs[i], freqs [rot / 2] in radians a position:
 *   (x, y) -> magnitude (x cos a - y sin a, y cos a + x sin a), pairs being dimensions (i, i + rot / 2), or
 *   (2 i, 2 i + 1) where interleaved is not 0; the others stay.
 * f32 arithmetic, rounded once at the end; a is formed in f64, so that its error is 2^-52 of its size (past
 * 2^51 it means nothing). D a multiple of 16, 16 .. 256, rot one too, 16 .. D. q, k and the outputs
 * q_out [T][Hq][D], k_out [T][H][D] are of type elt (GLINT_KV_BF16 or GLINT_KV_F32); an output may be its
 * own input where that is as contiguous. q_norm and k_norm [D], each or NULL, are of type norm_elt. Addresses
 * are 16-B aligned, strides multiples of 16 B. A launch holds 2^23 - 1 workgroups (from 2048 tokens on one a token, and
 * into the cache one for 32 tokens' values of a head): more is -2. */
int glint_rotate_qk(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
                    int64_t k_stride_h, int elt, const int64_t *pos, const double *freqs, int64_t T, int Hq, int H, int D,
                    int rot, int interleaved, double magnitude, const void *q_norm, const void *k_norm, int norm_elt,
                    float eps, void *q_out, void *k_out, struct ihipStream_t *stream);

/* The same on the way into the cache: the keys that glint_rotate_qk gives, and v, are encoded as
 * glint_kv4_append does. D is 64 or 128; k_out may be NULL. */
int glint_kv4_append_rotated(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
                             int64_t k_stride_h, const void *v, int64_t v_stride_t, int64_t v_stride_h, int elt,
                             const int64_t *pos, const double *freqs, const int64_t *slots, int64_t T, int Hq, int H,
                             int D, int rot, int interleaved, double magnitude, const void *q_norm, const void *k_norm,
                             int norm_elt, float eps, void *q_out, void *k_out, uint8_t *k_hole, float *k_absmax,
                             uint8_t *v_hole, float *v_absmax, int64_t pages, struct ihipStream_t *stream);

/* Scores of T rows of V logits (BF16 bits or f32, row t at t * stride), with
 * lse = log sum_j exp x_j:
 *   logprob[t] = x[tok] - lse;  entropy[t] = lse - sum_j p_j x_j (0 where p_j is 0);
 *   rank[t] = how many entries come before tok: larger, or equal at a lower index;
 *   top_logprob, top_index [T][top]: the largest entries, equal ones by index.
 * A token below 0 (a place without one) gives logprob 0 and rank -1, one of V or above NaN
 * and -1. A row with a NaN or +inf, or with -inf alone, gives NaN log probabilities and
 * entropy; in the top list NaN takes the place of -inf, and rank counts no NaN. T < 4194304,
 * 0 <= top <= min(20, V), and V <= 262144 where top > 0. A few long rows are split
 * over workgroups as glint_kv4_attend's sequences are. entropy, rank and, for top == 0, the top_ pointers may be NULL. */
int glint_token_logprobs(const void *logits, int elt, int64_t stride, const int64_t *tokens, int64_t T, int64_t V,
                         int top, float *logprob, float *entropy, int32_t *rank, float *top_logprob,
                         int32_t *top_index, struct ihipStream_t *stream);

#ifdef __cplusplus
}
#endif
#endif
