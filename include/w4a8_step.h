/*
 * w4a8_step.h -- the rest of a decode step around the engine's matrices
 * (libkv260gemv.so): rope and the key/value cache between q|k|v and o
 * (board/tp/tp_llama.cpp:835-856), the residual adds and norms behind o and
 * down, and the sampler's draw behind the LM head.
 *
 * Conventions of w4a8.h: every array is a device address, `stream` is a
 * hipStream_t of the current device, calls enqueue work and return, nothing is
 * allocated, a failed check returns a negative status and enqueues nothing. What
 * a call writes (the workspace too) may be no part of its other arrays, but x_out.
 * What the device holds (positions, page numbers, a row's settings) cannot be
 * checked by the host; each call below says what its kernels do with values
 * out of range, and none of them reads or writes outside the arrays given.
 */
#ifndef W4A8_STEP_H
#define W4A8_STEP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum w4a8_kv_dtype {
    W4A8_KV_F16 = 0,
    W4A8_KV_BF16 = 1,
};

/* A paged cache of one layer. k and v are [pages, kv_heads, page_size,
 * head_dim] each, 16-byte aligned. head_dim 64, 96, 128 or 256; page_size 16,
 * 32, 64, 128 or 256 tokens; kv_heads 1..4096. pages may be any number that
 * memory holds: offsets are 64-bit. */
typedef struct w4a8_kv_cache {
    void *k;
    void *v;
    int pages;
    int page_size;
    int kv_heads;
    int head_dim;
    int dtype;              /* enum w4a8_kv_dtype */
} w4a8_kv_cache;

/* Where each of m rows (one new token each) stands. pos[i]: the row's position
 * in its sequence, or negative: an empty row (padding). Row i's pages are
 * table[i * table_stride + 0 .. table_pages - 1]: entry j holds the number of
 * the page with positions j * page_size onwards. With table_stride 0 all rows
 * share one table row: the tokens of a prompt, or drafted ones, whose attention
 * then reads the cache once for several of them. An entry outside [0, pages) is
 * an absent page: nothing is stored for its positions, and attention takes them
 * as masked; so it does positions from table_pages * page_size on. How rows are
 * split over the GPU goes by table_pages: a table no wider than its longest row
 * needs is the fastest. */
typedef struct w4a8_kv_rows {
    const int32_t *table;
    int64_t table_stride;   /* entries; 0 or table_pages .. 2^30 */
    int table_pages;        /* >= 1, at most 2^30 positions */
    const int32_t *pos;     /* [m] */
    int m;                  /* 1..65536 */
} w4a8_kv_rows;

/* The q|k|v rows a layer's first GEMV leaves (float32 [m][(heads + 2 kv_heads)
 * * head_dim], 16-byte aligned) into the cache: q and k rotated by the row's
 * position, k and v rounded to the cache's type (to nearest even) and stored at
 * it. q_out: float32 [m][heads * head_dim], 16-byte aligned, may be no part of
 * qkv; zeros for an empty row, whose cache entries are left as they are.
 * inv_freq: float32 [rope_dim / 2], the angle of pair i being pos * inv_freq[i]
 * radians (sine and cosine within 2^-23, up to 2^40 of them); rope_dim even, 2 ..
 * head_dim, dimensions past it pass unrotated. Pairs are (i, i + rope_dim / 2), or
 * (2i, 2i + 1) with interleaved (GGUF's Llama order, board/tp/tp_llama.cpp:528-705).
 * Two rows of one call must not share a page and position: either's values may
 * stand.
 * heads a multiple of kv_heads, m * heads at most 2^22. */
int w4a8_rope_append(const float *qkv, int heads, const w4a8_kv_cache *cache, const w4a8_kv_rows *rows,
                     const float *inv_freq, int rope_dim, int interleaved, float *q_out, void *stream);

/* Attention of each row's token over its cached positions 0 .. pos (so the
 * row's own token has been appended): out[i][h] = sum_j p_j v_j, p the softmax
 * over j of scale * (q[i][h] . k_j), query head h reading KV head
 * h / (heads / kv_heads). q, out: float32 [m][heads * head_dim], 16-byte
 * aligned, out no part of q. Scores, softmax and sums are float32. q and p meet
 * the cache's 16-bit values in 16-bit parts: q holds 22 bits, or steps of 2^-38
 * of its head's largest |q| where those are coarser (fp16); p holds 22 bits at
 * any size (bf16: down to 2^-64 of the row's largest, and none under 2^-88). A
 * row without a position left (empty, or all its pages absent) gives zeros.
 * Finite K and V give finite outputs, V up to the type's largest included, where
 * the scores are within float32's range. An infinite or NaN K (or a score past
 * that range) at a position attended makes the outputs of its row's query heads
 * of that KV head NaN, an infinite or NaN V the outputs of its dimension there
 * non-finite.
 * workspace: w4a8_paged_attention_workspace_bytes of device memory, 16-byte
 * aligned, its contents without meaning between calls; calls that may overlap
 * need one each. */
size_t w4a8_paged_attention_workspace_bytes(int heads, const w4a8_kv_cache *cache, const w4a8_kv_rows *rows);
int w4a8_paged_attention(const float *q, int heads, const w4a8_kv_cache *cache, const w4a8_kv_rows *rows, float scale,
                         float *out, void *workspace, size_t workspace_bytes, void *stream);

/* The residual add behind a block, with the norms on both sides of it:
 *   t = post_w ? rmsnorm(y) * post_w : y
 *   x_out = x + scale * (gate * t)       (gate NULL: t)
 *   h = rmsnorm(x_out) * norm_w          (norm_w NULL: no h)
 * for m <= 2^23 rows of float32[k] (k as in w4a8.h), rmsnorm as w4a8_rmsnorm_q8_0's, bit
 * for bit. gate: float32 [k] (gate_stride 0) or rows gate_stride apart
 * (gate_stride >= k, a multiple of 4). h: float32 [m][k], or, with q8, engine
 * layout rows (w4a8_engine_x_bytes(k) each, what w4a8_rmsnorm_q8_0 makes of
 * x_out). x_out may be x; nothing else may overlap. All 16-byte aligned. */
int w4a8_residual_rmsnorm(const float *x, const float *y, const float *post_w, const float *gate, int64_t gate_stride,
                          float scale, const float *norm_w, float eps, float *x_out, void *h, int q8, int k, int m,
                          void *stream);

/* One token for each of m rows of n logits (rows logits_stride >= n floats
 * apart), from the row's random number u[i] in [0, 1). The order is by logit,
 * descending, the smaller index first among equals; w_j = exp((l_j - max) /
 * temperature). Kept are the first top_k; of those the shortest prefix whose
 * mass reaches top_p of theirs; of those the tokens with w >= min_p (the first
 * always). The token drawn is the first whose running mass over the kept ones
 * exceeds u * their mass. Masses are sums of w to 2^-44, exact in 64-bit
 * integers, so the token does not depend on any order of summation.
 *   temperature <= 0 (or NaN): the first token (greedy); top_k <= 0: all;
 *   top_p >= 1 (or NaN): all; min_p <= 0 (or NaN): all; u < 0 or NaN as 0, u >= 1
 *   as the last kept token. A logit that is NaN or -inf is never drawn; -1 for a
 *   row without any other. Where the largest is +inf, those that are share w = 1.
 * Each setting is an array of m values, or, where its pointer is NULL, the one
 * value beside it. 1 <= n <= W4A8_SAMPLE_MAX_N, 1 <= m <= 65536.
 * workspace: w4a8_sample_workspace_bytes(m, n) of device memory, 16-byte
 * aligned, its contents without meaning between calls; calls that may overlap
 * need one each. */
typedef struct w4a8_sampling {
    const float *temperature_rows;
    const int32_t *top_k_rows;
    const float *top_p_rows;
    const float *min_p_rows;
    float temperature;
    int32_t top_k;
    float top_p;
    float min_p;
} w4a8_sampling;
#define W4A8_SAMPLE_MAX_N 524288
size_t w4a8_sample_workspace_bytes(int m, int n);
int w4a8_sample(const float *logits, int64_t logits_stride, int m, int n, const float *u,
                const w4a8_sampling *settings, int32_t *tokens, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A8_STEP_H */
