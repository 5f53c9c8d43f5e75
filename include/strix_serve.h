/*
 * strix_serve.h -- C ABI of the serving operators: a paged KV cache shared by many sequences (append, attention) and
 * drawing a token from logits. No counterpart in the reference, which decodes one sequence over a contiguous cache
 * (decode.rs:5262-5388) and picks tokens greedily (kernels.rs:2088-2110); the arithmetic in common (per-head RMS
 * norm, position rotation, grouped-query softmax) is that of the reference's forwards.
 *
 * Conventions of strix_cuda.h apply: 1 = done, 0 = declined (a shape the kernels do not take), <0 = error with text in
 * strix_cuda_last_error(). All pointers named d_* and all pointers inside strix_kv_pages are DEVICE pointers of the
 * handle's device. The `_dev` calls enqueue on `stream`, do not copy, allocate or synchronise, may be captured into a
 * CUDA graph, and leave the calling thread's current device as it was. Lengths, page ids and sampling parameters are
 * read from device memory by the kernels, so a captured graph serves every step.
 *
 * What the device data says wrong cannot be answered by a return code: it sets bit 1 of the handle's status
 * (strix_cuda_device_status; no other call reports or clears what these set) and the part concerned is skipped as described below. No value of row0, ctx or pages makes a
 * kernel read or write outside the buffers described to it.
 */
#ifndef STRIX_SERVE_H
#define STRIX_SERVE_H

#include "strix_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of a paged cache. E4M3: 8-bit floats (4 exponent, 3 mantissa bits; largest value 448) and one f32 scale
 * for each page and KV head, a cached value being code * scale. Scales are positive; strix_cuda_kv_append_dev writes powers of two
 * (with others in k, attention scores of 2^20 and more are not kept to f32 accuracy). */
enum { STRIX_KV_F16 = 0, STRIX_KV_E4M3 = 1 };
/* Which elements of a head a rotation pairs: none, (j, j + head_dim/2), or (2j, 2j + 1). */
enum { STRIX_ROPE_NONE = 0, STRIX_ROPE_HALVES = 1, STRIX_ROPE_ADJACENT = 2 };

/* The paged cache of one layer; the caller owns the memory. Page p, KV head h, slot t, element i of k lies at element
 * p * page_stride + (h * page_tokens + t) * head_dim + i, the same in v; scales at [p * n_kv + h].
 * page_tokens: 16, 32, 64 or 128. head_dim: 64, 96, 128, 192 or 256. page_stride: elements between pages, 0 =
 * n_kv * page_tokens * head_dim; a larger one interleaves the pages of several layers. Other sizes are declined.
 * k, v and page_stride must be 16-byte aligned. Values of cached tokens must be finite; slots behind a sequence's last
 * token may hold anything. */
typedef struct strix_kv_pages {
    void *k, *v;
    float *d_k_scale, *d_v_scale; /* E4M3: [n_pages][n_kv]; unused (may be NULL) for F16 */
    size_t page_stride;
    uint32_t n_pages, n_kv, page_tokens, head_dim;
    int type; /* STRIX_KV_* */
    int reserved;
} strix_kv_pages;

/* The sequences of a step. Sequence s owns rows d_row0[s] .. d_row0[s + 1] - 1 of q, k, v and out: its new tokens, at
 * positions d_ctx[s], d_ctx[s] + 1, ... behind the d_ctx[s] tokens that are cached already. Position t lives in slot
 * t % page_tokens of page d_pages[s * pages_ld + t / page_tokens]. d_ctx[s] < 0 marks an idle slot of a padded batch: its
 * rows enter no cache and get zeros from the attention. Rows from d_row0[n_seq] on belong to nobody and are left alone.
 * Both operators choose one form of their kernel for a call, by n_rows / n_seq. Where prompts and single tokens come together, put the
 * single tokens first and make two calls, one with the n sequences and rows of these, one with d_row0 + n, d_ctx + n,
 * d_pages + n * pages_ld, the other sequences and all n_rows: that is several times as fast.
 * Bad device data: offsets are clamped into [0, n_rows], and a sequence whose end lies before its start has no rows (where
 * offsets go down, two sequences may own a row: which of them the operators take it for, one, both or none, is unspecified);
 * positions at or beyond pages_ld * page_tokens and pages with an id outside [0, n_pages) are neither written nor attended to.
 * Each sets the status bit. */
typedef struct strix_kv_batch {
    const int32_t *d_row0;  /* [n_seq + 1] */
    const int32_t *d_ctx;   /* [n_seq] */
    const int32_t *d_pages; /* [n_seq][pages_ld] */
    uint32_t n_seq, n_rows, pages_ld;
    int reserved;
} strix_kv_batch;

/* What happens to q, k and v on their way: an RMS norm of each head of q and k with a weight (NULL = none), of v without
 * one (norm_v), then the rotation of q and k by angle position * theta^(-2j/head_dim) / d_freq[j] for pair j (d_freq NULL =
 * ones; ops.rs:159-176), taken exactly (not in f32) so that far positions stay right. */
typedef struct strix_kv_prep {
    const float *d_q_norm, *d_k_norm; /* [head_dim] */
    const float *d_freq;              /* [head_dim / 2] */
    float theta, eps;
    int rope, norm_v; /* rope: STRIX_ROPE_* */
} strix_kv_prep;

/* The checks of the calls below on a cache and a batch (may be NULL), without a handle or a device: 1 = taken, 0 = declined
 * (page_tokens, head_dim, n_kv, or n_heads not a multiple of n_kv; n_heads 0 = not looked at), -1 = an error in the arguments.
 * Pointers are looked at, not followed. */
STRIX_API int strix_cuda_kv_check(const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads);

/* Puts the batch's rows of k and v into the cache and prepares q, in one launch. d_k, d_v: [n_rows][n_kv * head_dim] f32
 * with ld_k / ld_v floats between rows (0 = packed; the rows of a fused q|k|v projection are slices with a larger ld).
 * A layer whose V is its raw K (k_eq_v) passes d_v = d_k. d_q / d_q_out (both NULL: no q): [n_rows][n_heads * head_dim],
 * d_q_out may be d_q with the same ld; rows of idle slots and rows of nobody are left as they were in d_q_out.
 * F16: values rounded to nearest, beyond +-65504 to that. E4M3: the scale of a page and head is the least power of two s with
 * |value| <= 448 s for every row that entered the page (at least 2^-120). It starts anew when slot 0 is written and only
 * grows afterwards; when it does, all other codes of the page and head move down by that power of two (exact until they
 * become subnormal). NaN is stored as 0, an infinity as the largest finite value.
 * Two rows of one call must not have the same page and slot, and a page that one call appends to must belong to one
 * sequence of the batch: the stored values are otherwise unspecified. */
STRIX_API int strix_cuda_kv_append_dev(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, const strix_kv_prep *prep,
                             uint32_t n_heads, const float *d_k, size_t ld_k, const float *d_v, size_t ld_v, const float *d_q,
                             size_t ld_q, float *d_q_out, size_t ld_q_out, void *stream);

/* Bytes of workspace for strix_cuda_attn_pages_dev, 0 = declined (device data is not looked at): enough for every batch of up to
 * n_rows rows, into whatever number of sequences they divide, over any cache of this head_dim with at most as many query heads to a
 * KV head. */
STRIX_API size_t strix_cuda_attn_pages_workspace(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads);
/* out[row][head] = softmax(scale * q k^T) v over the cached tokens the row sees: positions 0 .. its own (its own k and v
 * are in the cache by then), with window > 0 only the last `window` of them. scale is finite. n_heads is a multiple of n_kv; head h reads KV
 * head h / (n_heads / n_kv). q and out: [n_rows][n_heads * head_dim] f32, ld_q / ld_out floats between rows (0 = packed), which
 * must not overlap. With a window, pages that end before all rows' windows are not looked at: they may be given away.
 * A row that sees no token gets zeros. Offsets that give away more rows than n_rows (possible where they go down) set the status
 * bit and leave out as it was. At most 8192 sequences in one call, and 2^31 tiles of 16 tokens in all blocks of rows when
 * every sequence fills its row of d_pages (-1 beyond). Products and sums keep f32 accuracy (f16 tensor-core products of q and
 * of the probabilities in two halves of 11 bits each: an element of q is off by 2^-22 of itself or 2^-38 of the largest of its head, a
 * probability times its page's scale by 2^-22 of itself or 2^-39 of the row's largest among 16 to 64 neighbouring tokens).
 * d_work: work_bytes >= strix_cuda_attn_pages_workspace, 256-byte aligned, zeroed once before its first use; every
 * call leaves it ready for the next (of any sizes that the workspace serves), but for one whose bounded wait ran out (bit 0 of the status): out is
 * unspecified then and d_work has to be zeroed again. Calls that share a workspace must not run at the same time; graphs
 * replayed on different streams therefore need one each. The result does not depend on what else runs: partial sums
 * are joined in a fixed order. */
STRIX_API int strix_cuda_attn_pages_dev(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads,
                              const float *d_q, size_t ld_q, float scale, uint32_t window, float *d_out, size_t ld_out, void *d_work,
                              size_t work_bytes, void *stream);

/* Sampling parameters, one entry per row; a NULL array means the neutral value in brackets. */
typedef struct strix_sample_params {
    const float *d_temperature; /* [1] <= 0: greedy */
    const int32_t *d_top_k;     /* [0] 0 or less: off */
    const float *d_top_p;       /* [1] 1 or more: off */
    const float *d_min_p;       /* [0] */
} strix_sample_params;

/* Draws one token per row of d_x[rows][stride] (n <= STRIX_SAMPLE_MAX_N logits each):
 *   w_i = exp((x_i - max x) / temperature)
 *   top-k: the k largest logits; top-p: of those, in descending order, the tokens before which the weights sum to less
 *   than top_p of the whole (the first always stays); min-p: of those, the ones with w_i >= min_p (w = 1 at the maximum)
 *   d_ids[row] = the least i whose kept weights up to and including i exceed d_u[row] * (sum of kept weights), d_u in [0, 1)
 * Equal logits rank by index, lower first; NaN counts as -inf; with +inf among the logits only those have weight.
 * A row without any logit above -inf gives id 0 and probability 0. d_probs (may be NULL): the drawn token's weight over the kept
 * sum. A weight is off by about 2^-22 (1 + |x_i - max x| / temperature) of itself (f32 exponent); min_p and top_p
 * cut to that accuracy. Weights are summed as 64-bit integers (in steps of 2^-40; the sum of a whole row in f32 over stretches of fixed
 * order), so the same logits and the same u draw the same token every time.
 * The greedy choice is that of strix_cuda_argmax_dev except below its floor of -3.0e38. */
#define STRIX_SAMPLE_MAX_N 393216
STRIX_API int strix_cuda_sample_dev(strix_cuda *h, const float *d_x, size_t n, size_t stride, size_t rows, const strix_sample_params *params,
                          const float *d_u, uint32_t *d_ids, float *d_probs, void *stream);
/* strix_cuda_decode_step_argmax with a draw in place of the argmax: one decode step, the logits (soft-capped where the
 * model is) stay on the device, the token id and its probability (prob may be NULL) come back. 0 = not configured, a
 * row-sharded handle, or a vocabulary above STRIX_SAMPLE_MAX_N. */
STRIX_API int strix_cuda_decode_step_sample(strix_cuda *h, const float *hvec, size_t pos, float temperature, int32_t top_k, float top_p,
                                  float min_p, float u, uint32_t *id, float *prob);

#ifdef __cplusplus
}
#endif
#endif /* STRIX_SERVE_H */
