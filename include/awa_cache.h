/*
 * awa_cache.h -- a paged key/value cache for attention over rows that arrive
 * step by step: appending rows with the position rotation applied on the way,
 * and attention over the cache with a sliding window and a prefix that stays
 * visible.
 *
 * The AWA layers (awa_b200.h) attend within the windows of a clip that is
 * there as a whole. A caller that restores a video as its frames arrive, or
 * generates token by token, keeps the keys and values of earlier rows instead:
 * awa_cache_append does for new rows what awa_pack and awa_mmrope do for a
 * clip's (lay out, rotate), awa_cache_attention what awa_window_attention
 * does. The reference has no counterpart (its layers see one clip).
 *
 * Conventions are awa_b200.h's: the same status codes and awa_last_error(),
 * device pointers, strides in elements, work enqueued on the given stream,
 * nothing synchronises or allocates device memory. The lengths of a batch live
 * in device memory, so a captured graph serves later steps when only their
 * contents change. What the device finds wrong in them (a page number or a
 * coordinate out of range, a sequence longer than its page table) it reports
 * through awa_device_status(): AWA_CACHE_BAD_PAGE or AWA_CACHE_BAD_COORD; it
 * never reads or writes outside the buffers for it. Rows without a place are not
 * appended or read back; to awa_cache_attention the rows of a page that is not
 * there are keys and values of zeros, which count in the softmax, and a sequence
 * ends where its page table does.
 */
#ifndef AWA_CACHE_H
#define AWA_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "awa_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Storage type of a cache beside AWA_F32 and AWA_BF16: 4-bit codes, 64
 * consecutive features of a row sharing a scale and a minimum. */
#define AWA_INT4 2
#define AWA_CACHE_GROUP 64 /* features that share a scale and a minimum */

/* What awa_device_status() reports (in awa_last_error's text) after a bad batch. */
#define AWA_CACHE_BAD_PAGE 71  /* a page number outside the cache, or a sequence longer than its table row */
#define AWA_CACHE_BAD_COORD 72 /* a rotation coordinate outside the table */

typedef struct awa_cache awa_cache;

/* The memory of a cache, owned by the caller. Keys (values alike) of slot s of
 * head h of page p: head_dim dense elements at
 *   k + p * page_stride + h * head_stride + s * head_dim   (elements)
 * and for AWA_INT4 head_dim / 2 bytes at
 *   k + p * page_stride + h * head_stride + s * head_dim / 2   (bytes),
 * byte i holding feature 2i in its low and 2i + 1 in its high four bits, with
 *   k_params + p * params_page_stride + h * params_head_stride + s * 2 * (head_dim / 64)
 * (bf16 elements): (scale, minimum) of each 64 features. A code c stands for
 * scale * c + minimum in fp32. Bases and strides are multiples of 16 bytes,
 * the strides below 2^40 bytes. */
typedef struct
{
    int storage;     /* AWA_F32, AWA_BF16 or AWA_INT4 */
    int heads;       /* key/value heads */
    int head_dim;    /* a multiple of 8 up to 128; AWA_INT4: 64 or 128 */
    int page_tokens; /* rows of a page: 16, 32, 64, 128 or 256 */
    int pages;
    void* k;
    void* v;
    int64_t page_stride, head_stride;
    void* k_params; /* AWA_INT4 only */
    void* v_params;
    int64_t params_page_stride, params_head_stride;
} awa_cache_params;

/* One call's rows: sequence b brings the rows row_starts[b] .. row_starts[b+1]-1
 * of the row tensors (none, if they are equal), at the positions past[b],
 * past[b] + 1, ... of the sequence. Position p lives in slot p % page_tokens of
 * page page_table[b * table_stride + p / page_tokens]. Rows outside
 * [row_starts[0], row_starts[sequences]) belong to nobody: nothing is read or
 * written for them. The three arrays are device memory. rows is below 2^30 and
 * table_width * page_tokens at most 2^30; a negative past counts as 0 in
 * awa_cache_attention and is reported by awa_cache_append and awa_cache_read. */
typedef struct
{
    int sequences;
    int rows;     /* rows that the row tensors have */
    int max_rows; /* most rows of one sequence, as far as known: chooses the kernel, not the result */
    const int* row_starts; /* [sequences + 1], ascending */
    const int* past;       /* [sequences] rows that the cache held before this call */
    const int* page_table; /* [sequences][table_width] */
    int table_width;
    int64_t table_stride;
} awa_cache_batch;

/* The rotation of q and k rows, in interleaved pairs as SeedVR2MMRoPE's
 * (awa_layers.cpp:913-953): pair i of axis a is features 2 (a pairs + i) and
 * the next, turned by table[c][i] with c the row's coordinate on that axis;
 * features past 2 axes pairs are copied. x0 c - x1 s and x1 c + x0 s, every
 * product and sum rounded to fp32. */
typedef struct
{
    const float* table; /* [max_coord][pairs][2] (cos, sin), fp32, 8-byte aligned */
    int max_coord;
    int axes;           /* 1 to 4; 2 * axes * pairs <= head_dim */
    int pairs;
    const int* coords;  /* [rows][axes]; NULL: every axis takes the row's position in its sequence */
} awa_cache_rope;

/* Checks the parameters and builds the handle on the CURRENT device (the status
 * flag, the kernels' attributes), where the memory has to lie: make it before a
 * stream capture begins. Holds no device memory of its own. */
int awa_cache_create(const awa_cache_params* params, awa_cache** out);
/* The checks of awa_cache_create without a device: for checking arguments on
 * machines without a GPU. Every call that would enqueue work rejects such a
 * cache with -1, after its own checks. */
int awa_cache_create_host(const awa_cache_params* params, awa_cache** out);
void awa_cache_destroy(awa_cache* cache);

/* Writes the batch's rows into the cache: k rotated, v as it is, each rounded
 * once to the storage type; and, if q is not NULL, q rotated into q_out.
 *   q: rows of q_heads x head_dim (dense within a row), k, v: of the cache's
 *   heads x head_dim, of in_dtype (AWA_F32 or AWA_BF16), q_out of q_out_dtype;
 *   q_out may be q itself if the types and strides agree. rope NULL: no
 *   rotation.
 * AWA_INT4: of each 64 features, minimum = min rounded down to bf16, scale =
 * (max - minimum) / 15 rounded up to bf16, code = rint((x - minimum) * (1 /
 * scale)) clamped to 0..15, each operation rounded to fp32 (all codes 0 where
 * the scale is 0); the rows have to be finite.
 * A slot that two rows of one call name holds a mixture of the two. */
int awa_cache_append(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int in_dtype, const void* q,
                     int64_t q_token_stride, const void* k, int64_t k_token_stride, const void* v,
                     int64_t v_token_stride, const awa_cache_rope* rope, int q_out_dtype, void* q_out,
                     int64_t q_out_token_stride, awa_stream_t stream);

/* The batch's rows back from the cache as the values they stand for:
 * k_out, v_out of heads x head_dim per row, of out_dtype. */
int awa_cache_read(const awa_cache* cache, const awa_cache_batch* batch, int out_dtype, void* k_out,
                   int64_t k_token_stride, void* v_out, int64_t v_token_stride, awa_stream_t stream);

/* out = softmax(scale q K^T) V of every row over the keys of its sequence that
 * it sees; the cache already holds the batch's own rows (awa_cache_append with
 * the same batch). q head i reads key/value head i / (q_heads / heads).
 *   With sinks = S, frame_tokens = F, window = W and length = past + rows of
 *   the sequence: the first S positions are the prefix; the others are cut
 *   into frames of F. A row of frame f sees the prefix and the frames f - W + 1
 *   .. f as far as they are there (W = 0: all frames up to f). A row of the
 *   prefix at position p sees positions 0 .. min(S, (p / F + 1) F) - 1.
 *   F = 1 is causal attention with a sliding window of W tokens; F > 1 lets
 *   the tokens of one video frame see one another.
 *   A row that sees nothing gets zeros. Pages that no row of the batch sees
 *   need not be there: their page_table entries are not read.
 * q and out: rows x q_heads x head_dim (dense within a row) of AWA_F32 for an
 * AWA_F32 cache (to fp32 accuracy: FFMA or six bf16 products, fp32 sums), else of
 * AWA_BF16 (16-bit operands on the tensor cores: the cache's values and the
 * probabilities, rounded once to bf16 or, many rows of 4 bits, fp16; fp32
 * accumulation and softmax statistics, the probabilities' sum taken before that
 * rounding). 16-byte aligned rows. scale: > 0. sinks and window: 0 or more,
 * frame_tokens: 1 or more. Values in the cache that some row of the batch sees
 * have to be finite; with an AWA_INT4 cache they and q are below 65504 in
 * magnitude. Of those, few rows tell values apart down to 2^-70. Many rows take
 * them as fp16 (11 bits) scaled by powers of two, one for the keys and one for
 * the values of each 64 features of a head: 2^-38 of the largest that some row
 * of the batch sees there is the least they tell apart; probabilities below
 * 2^-32 of a row's largest are dropped.
 * workspace: awa_cache_attention_workspace_bytes() bytes, 256-byte aligned
 * (NULL if that is 0), used by this call until its work is done: calls that may
 * overlap, two captured graphs among them, need one each. It holds the parts of
 * rows that several blocks work on (few rows of long caches, many rows: tens of
 * MB) and, for many rows over an AWA_INT4 cache, q and the visible pages as fp16
 * (rounded once): as many pages as the table reaches within window and prefix,
 * but no more than the cache has, of as many heads at a time as 2 GiB hold (of
 * one, if one head's are more). AWA_F32 caches and head sizes other than 64 and
 * 128 need none. */
size_t awa_cache_attention_workspace_bytes(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int sinks,
                                           int window, int frame_tokens);
int awa_cache_attention(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int dtype, const void* q,
                        int64_t q_token_stride, float scale, int sinks, int window, int frame_tokens, void* out,
                        int64_t out_token_stride, void* workspace, size_t workspace_bytes, awa_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* AWA_CACHE_H */
