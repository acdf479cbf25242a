/* A key-value cache in pages, served on an MI355X (gfx950): requests of any length share one pool of pages, each named by
 * its request's row of a page table, so that a server reserves what its requests hold and not what they might. Keys and
 * values are F32 like the caches of llama_hip_forward.h, or BF16 at half the bytes. No counterparts in the reference, which
 * runs one sequence.
 *
 * Pointers follow llama_hip_kernels.h: device memory in place (stream-ordered on the library stream, no wait),
 * registered host ranges through their device copies, other host memory copied in and out around a synchronous call.
 * The index arrays (start, length, pages) are read on the device when the call runs, so a captured call follows what they
 * hold at each replay; an index outside its range is never followed and fails at the next host-visible point
 * (llhip_synchronize, or the end of a staged call). */
#ifndef LLAMA_HIP_PAGED_H
#define LLAMA_HIP_PAGED_H

#include <stddef.h>

#include "llama_hip_requests.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef LLHIP_ENUM { PAGE_F32, PAGE_BF16 } PageType;

/* Requests 0 .. count - 1 (at most LLHIP_MAX_REQUESTS). As in RequestBatch, request r's rows are start[r] .. start[r + 1]
 * - 1 of the row buffers (none is allowed), its row j lies at position length[r] + j, and rows before start[0] and from
 * start[count] on belong to nobody and are left as they are. Position t of request r lies in page pages[r * max_pages +
 * t / page_size] at place t % page_size; entries behind the request's last position are not read, and several requests may
 * name a page that none of them stores into (a prompt's beginning that they share). The key cache and the value cache hold
 * num_pages pages each, one behind the other, a page being page_size positions of n_kv_heads heads in the selected layout
 * (kernels_kv_layout_name), as a slot of RequestBatch is. */
typedef struct {
  const int *start;  /* count + 1 */
  const int *length; /* count: positions before the request's first row */
  const int *pages;  /* count x max_pages */
  int count;
  int rows;      /* rows that the row buffers hold */
  int max_pages; /* pages that a request may have */
  int page_size; /* positions of a page */
  int num_pages; /* pages of each cache */
  int seq_len;   /* positions that a request may have, at most max_pages * page_size */
  PageType type;
} PagedBatch;

/* The rows' keys and values into their requests' pages, with RoPE on the way and, for a model that has them, the norms of
 * each head, in one launch: q_out = q's n_heads heads, normed where q_norm (head_dim weights) is given, then rotated; k's
 * n_kv_heads heads, normed where k_norm is given and rotated, and v as it is, into the pages (rounded to the nearest, ties
 * to even, for PAGE_BF16). A norm is k_rmsnorm of the head's values with epsilon, a rotation k_rope_apply (bitwise, where
 * there is no norm before it); table holds seq_len rows of k_rope_table, position by position. Rows of q, q_out, k and v lie
 * q_stride, q_out_stride and kv_stride floats apart; q_out may be q itself (of the same stride), k and v stay as they are.
 * A row whose page lies outside the caches is not stored; it fails at the next host-visible point, as do two requests whose
 * first rows go to the same page. Two rows of a call must not go to the same place of a page otherwise either: it would hold
 * values of both. q_out, the rows, the norms, both caches and the batch's arrays must not overlap otherwise; head_dim even
 * and at most 256, n_heads a multiple of n_kv_heads, at most 16 per KV head. A launch holds 2^23 blocks, each of two q heads
 * or one KV head of 8 rows (of head_dim 128; 16 of 64, 4 of 256; half as many unless head_dim and the strides are multiples
 * of 4 and the buffers 16-byte aligned): more rows are refused. */
void llhip_rope_kv_append_paged(float *q_out, size_t q_out_stride, const float *q, size_t q_stride, const float *k,
                                const float *v, size_t kv_stride, const float *table, const float *q_norm,
                                const float *k_norm, float epsilon, const PagedBatch *batch, int n_heads, int n_kv_heads,
                                int head_dim, void *key_pages, void *value_pages);

/* Causal attention of every request's rows over the positions that its pages hold: row j of request r attends to positions 0
 * .. length[r] + j (the last rows' are stored before, by llhip_rope_kv_append_paged). Rows of q lie q_stride floats apart,
 * rows of out n_heads * head_dim; scores, softmax and value sums as in k_attention: products of the F32 queries and weights
 * with the pages' values, FP32 sums; a non-finite score fails with "nonfinite value in softmax". The sums are divided by the
 * weights' at the end, which may reach 2^8 each, so n positions' values must stay below 1e36 / n. What lies in a page behind
 * the request's last position is not used, and a value that is not finite reaches the rows that see its position only, in its
 * dimension: an infinity gives infinity, whatever its weight, and NaN beside one of the other sign or beside a NaN. A request
 * with a page outside the caches fails at the next host-visible point; its rows' values are then unspecified. out must not
 * overlap q, a cache or the batch's arrays. The shapes are k_attention's: n_heads a multiple of n_kv_heads, 1 to 16 per KV
 * head, head_dim at most 256.
 *
 * Rows of K and V in whole 16-byte vectors (head_dim a multiple of 8 in BF16 pages, of 4 in F32 ones, the caches 16-byte
 * aligned) take the matrix cores, with at most 2^20 rows and 4096 KV heads; any other shape has each row read what it attends
 * to by itself, some fifty times slower. Pages of a multiple of 16 positions are the fastest (of 8: 1.15 to 1.4 times longer).
 * BF16 pages meet the F32 queries and weights as three exact BF16 parts of those, F32 pages in FP32 products, FP32 sums
 * either way; a weight below 2^-126 of its row's largest counts as 0. A call's parts meet in a workspace and counters that all
 * calls on a device share: calls ordered on the library's stream are safe, from any thread. Two that may run concurrently on one
 * GPU (graphs replayed on other streams) race, and the damage lasts: a counter that they leave off zero makes later calls' rows
 * wrong, too, until the process ends. The workspace is as large as any lengths may need: 22 MB of HBM for head_dim up to 64, 43
 * up to 256 (of up to 512 KV heads), twice that for BF16 pages of head_dim up to 128 where rows outnumber requests (and one may
 * have more than 64 query vectors of a KV head), also for a call of one short row; it stays. Run the largest batch once before
 * capturing a step, so that the workspace is there. */
void llhip_attention_paged(float *out, const float *q, size_t q_stride, const void *key_pages, const void *value_pages,
                           const PagedBatch *batch, int n_heads, int n_kv_heads, int head_dim);

#ifdef __cplusplus
}
#endif
#endif
