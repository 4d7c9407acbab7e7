/*
 * C ABI of attention over a cache of keys and values that lies in pages, of writing that cache and of reading it back
 * (gfx950).  No counterpart in the reference, which attends to q, k and v of the same length only.  Plain pointers and sizes,
 * no torch types; conventions of fused_mha.h: fp16 or bf16 tensors, device pointers on 16-byte boundaries, calls are
 * asynchronous on `stream` and allocate nothing, FUSED_MHA_OK or a negative code comes back, arguments are validated before
 * anything is launched.
 *
 * The cache: `key` and `value` of shape (pages, page_size, kv_head, d), with strides.  Position p of sequence b is slot
 * p % page_size of page page_table[b][p / page_size].  A sequence has cache_seqlens[b] keys, those of its new tokens among
 * them: new token i of n is at position cache_seqlens[b] - n + i.
 *
 * What lies in device memory is not known to the host, so the kernels keep to their bounds by themselves:
 *   - a length is taken as 0 below 0; positions past the page table or on a page that is none of the cache's (a number that is
 *     not 0 .. pages-1) are not accessed: paged_mha_write leaves those out, paged_mha_read gives NaN for them, and
 *     paged_mha_forward gives NaN for all rows that would see one, and may for other rows of the same sequence;
 *   - entries of cu_seqlens are taken as within 0 .. tokens; tokens that belong to no sequence are not read, and rows of the
 *     output that belong to none are zeroed or left as they are (paged_mha_forward).  Where entries decrease, the sequences' rows
 *     hold any numbers;
 *   - entries of the page table behind a sequence's last key, and what the cache holds there, are not looked at.
 */
#ifndef PAGED_MHA_H_
#define PAGED_MHA_H_

#include <stddef.h>

#include "fused_mha.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Codes beside those of fused_mha.h. */
#define PAGED_MHA_ERR_BAD_TYPE (-11)       /* a type that is none of the below, or scales that do not go with it */
#define PAGED_MHA_ERR_BAD_PAGE_SIZE (-12)  /* page_size is no multiple of 16 */
#define PAGED_MHA_ERR_BAD_GROUP (-13)      /* head is no multiple of kv_head */
#define PAGED_MHA_ERR_WORKSPACE (-14)      /* the workspace is too small */

#define PAGED_MHA_FP16 0
#define PAGED_MHA_BF16 1
/* 8 bits, OCP e4m3 without infinities, with a scale for each position and head: 2^(byte - 127), byte 1 .. 254. */
#define PAGED_MHA_E4M3 2

/* Element strides; rows of d elements are contiguous and begin on 16-byte boundaries.  slot < 2^24, head < 2^30. */
typedef struct paged_mha_strides {
  long long page, slot, head;
} paged_mha_strides;

typedef struct paged_mha_cache {
  void *key, *value;
  void *key_scale, *value_scale; /* (pages, page_size, kv_head) bytes with strides; NULL unless cache_type is PAGED_MHA_E4M3 */
  paged_mha_strides key_strides, value_strides, key_scale_strides, value_scale_strides;
  int pages, page_size, kv_head, d; /* d: 64 or 128 */
  int cache_type;                   /* `type` or PAGED_MHA_E4M3 */
  int type;                         /* of q, k, v and o: PAGED_MHA_FP16 or PAGED_MHA_BF16 */
} paged_mha_cache;

typedef struct paged_mha_batch {
  const int *page_table; /* batch rows of table_width, table_stride elements apart */
  long long table_stride;
  int table_width;
  const int *cache_seqlens; /* batch */
  const int *cu_seqlens;    /* batch + 1: the new tokens of sequence b are cu_seqlens[b] .. cu_seqlens[b+1]-1; NULL: see below */
  int batch;
  int tokens; /* with cu_seqlens all tokens of q, k, v and o, strides.batch is not used; without, new tokens of every sequence */
} paged_mha_batch;

/*
 * Writes k and v (tokens of the batch x kv_head x d, of cache->type) of the new tokens to their places.
 * E4M3: x is clipped to the type's largest value of four significant bits (fp16 61440, bf16 1.875 * 2^127; NaN stays NaN);
 * the scale is the least 2^e, e >= -126, for which no number of the row is over 448 * 2^e, and the row holds x / 2^e rounded to
 * nearest, ties to even: what comes back are values of the 16-bit type.
 * Places that several tokens of a call have (a page that is twice in the page table) hold one of them, or parts of several.
 */
int paged_mha_write(const paged_mha_cache *cache, const paged_mha_batch *batch, const void *key_ptr,
                    const fused_mha_strides *key_strides, const void *value_ptr, const fused_mha_strides *value_strides,
                    void *stream);

/*
 * Keys and values as dense (batch, max_seqlen, kv_head, d) tensors of cache->type; zeros behind a sequence's length.
 * cu_seqlens is not used, tokens only has to be positive.
 */
int paged_mha_read(const paged_mha_cache *cache, const paged_mha_batch *batch, int max_seqlen, void *key_ptr,
                   void *value_ptr, void *stream);

/*
 * o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j of the sequence; causal != 0: over those up to the token's own
 * position.  head is a multiple of kv_head; query head h has key head h / (head / kv_head).  A row without keys is zero,
 * one all of whose scores are -inf NaN.
 * Keys that a row does not see do not matter to it, whatever they and their values hold.
 * o is dense.  max_new: no sequence has more new tokens (0: not known); which kernel and how much workspace is taken
 * goes by it, not the result.
 * zero_rest: rows of o that belong to no sequence (tokens in front of cu_seqlens[0], and from cu_seqlens[batch] on) are zeroed
 * instead of left.
 * The workspace holds parts of long sequences that several work groups share; its contents do not matter before or after.
 */
size_t paged_mha_forward_workspace_bytes(const paged_mha_cache *cache, const paged_mha_batch *batch, int head, int max_new);
int paged_mha_forward(const paged_mha_cache *cache, const paged_mha_batch *batch, const void *query_ptr,
                      const fused_mha_strides *query_strides, void *output_ptr, int head, int max_new, float scale, int causal,
                      int zero_rest, void *workspace, size_t workspace_bytes, void *stream);

/* Static, human-readable text for a code of this file or of fused_mha.h. */
const char *paged_mha_error_string(int code);

#ifdef __cplusplus
}
#endif

#endif /* PAGED_MHA_H_ */
