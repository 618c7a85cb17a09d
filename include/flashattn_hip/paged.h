/*
 * flashattn_hip/paged.h: rotary positions and the paged K/V cache of
 * libflashattn_hip.so, for decoder layers that serve ragged batches.
 *
 * No counterpart in the reference, shrvan30/flash-attention-cuda: its caller
 * rotates q and k and keeps its own cache (README.md:9-13).
 *
 * Conventions as in flashattn_hip.h: device pointers (fp16 and bf16 data
 * and workspaces aligned to 16 bytes, int32 to 4, double to 8); asynchronous launches on `stream` (a hipStream_t; NULL is the
 * default stream); a non-zero return is an fa_status with a message in
 * fa_last_error(). Tensors are fp16 or bf16, head_dim is 64 or 128.
 */
#ifndef FLASHATTN_HIP_PAGED_H_
#define FLASHATTN_HIP_PAGED_H_

#include "../flashattn_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of these entry points (those of flashattn_hip.h are fp16). */
typedef enum fa_dtype { FA_F16 = 0, FA_BF16 = 1 } fa_dtype;

/* Rotary positions: out[b, h, n] = x[b, h, n] with pair i of its first rotary_dim
 * dims turned by positions[b, n] * inv_freq[i] (backward: by minus that) and
 * scaled by `factor`; the other dims are copied. Pair i is dims
 * (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved. With the same factor
 * the backward call gives the gradient of the forward one.
 * x is [B, H, N, head_dim] with the given strides in elements (multiples of 8, a
 * row's head_dim elements contiguous); out is contiguous and must not overlap x.
 * positions is int32 [B, N] (positions_batch_stride N) or one row for every
 * sequence (stride 0); inv_freq is rotary_dim / 2 doubles: far positions keep
 * their angle. rotary_dim is a multiple of 16 in [16, head_dim]; head_dim is 64
 * or 128. */
int fa_rope(const void *x, void *out, const int32_t *positions, const double *inv_freq, int dtype,
            int batch, int heads, int seq, int head_dim, int64_t x_batch_stride,
            int64_t x_head_stride, int64_t x_row_stride, int64_t positions_batch_stride,
            int rotary_dim, int interleaved, float factor, int backward, void *stream);

/* A paged K/V cache and the new tokens of a ragged batch on it. Pages are
 * [num_pages, H_kv, page_size, head_dim] contiguous, page_size a power of two in
 * [16, 1024]. Sequence b's key j lies in row j % page_size of page
 * page_table[b * max_pages + j / page_size]. The batch's new tokens are packed:
 * sequence b's are rows [cu_tokens[b], cu_tokens[b + 1]) of `tokens` rows, and
 * seq_lens[b] is its length with them, so its new token i sits at position
 * seq_lens[b] - (cu_tokens[b + 1] - cu_tokens[b]) + i.
 * page_table, seq_lens and cu_tokens (batch + 1 entries, the first 0, rising) are
 * int32 in device memory and never read on the host. What they hold cannot lead a
 * kernel out of the tensors: a position outside [0, max_pages * page_size) or a
 * page id outside [0, num_pages) has no key; packed rows before cu_tokens[0] and from
 * cu_tokens[batch] on belong to no sequence. At most 2^24 packed rows and 2^16
 * sequences; max_pages * page_size at most 2^27. */
typedef struct fa_paged {
  void *k_pages, *v_pages;
  const int32_t *page_table, *seq_lens, *cu_tokens;
  int dtype; /* fa_dtype */
  int batch, tokens, kv_heads, head_dim, page_size, num_pages, max_pages;
} fa_paged;

/* Packed rows [tokens, heads, head_dim]: strides in elements, multiples of 8;
 * a head's head_dim elements are contiguous. */
typedef struct fa_rows {
  const void *data;
  int64_t token_stride, head_stride;
} fa_rows;

/* Writes the new tokens' k and v into their pages (tokens without a key are
 * skipped). With rotary_dim > 0, k is turned by its position on the way (as
 * fa_rope), and q, H = `heads` query heads, is turned into q_out, contiguous
 * [tokens, H, head_dim] (rows that belong to no sequence become zero); with
 * rotary_dim 0, q, q_out and inv_freq are not used. Lengths are not changed: the
 * call can be repeated. No two tokens may have the same place, and q_out overlaps
 * no input. Where cu_tokens falls, a token still goes to one sequence at most, whose
 * bounds hold it, and to its place among that one's new tokens. */
int fa_append_paged(const fa_paged *cache, const fa_rows *k, const fa_rows *v, const fa_rows *q,
                    void *q_out, int heads, const double *inv_freq, int rotary_dim,
                    int interleaved, float factor, void *stream);

/* Bytes of device workspace fa_attend_paged needs on the current device; 0 with
 * fa_last_error() set on invalid arguments. */
size_t fa_attend_paged_workspace_bytes(int tokens, int heads, int kv_heads, int head_dim);

/* Causal attention of the new tokens' queries over the cache, their own keys
 * (written before) among it: o[t, h] = softmax over keys 0..position(t) of
 * scale * q[t, h] . k, times v, with K/V head h / (H / H_kv). out is contiguous
 * [tokens, H, head_dim] and overlaps no input; a row without a key, and one that
 * belongs to no sequence, is zero; so is every row if cu_tokens falls anywhere
 * within the packed rows. What a query does not see does not
 * reach it, infinities and NaN included; what it sees does. Scores scale q . k are held in
 * 32 bits: up to 10^7 either way. At most 128 query heads per K/V head.
 * Workspace and streams follow the rules of the split-K decode: the workspace stays
 * untouched until the launch completes, calls on one stream are ordered, replays of
 * one graph must not overlap. */
int fa_attend_paged(const fa_paged *cache, const fa_rows *q, void *out, int heads, float scale,
                    void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* FLASHATTN_HIP_PAGED_H_ */
