/* Many requests on one model, served on an MI355X (gfx950): what a server needs beside the single sequence of
 * llama_hip_forward.h. A batch of requests shares a prefix (a system prompt, a document) whose keys and values are
 * computed once; each request has a cache of its own behind it, may have a low-rank adapter of its own beside the
 * shared projections, and may bring drafted tokens that the model's logits accept or refuse. No counterparts in the
 * reference, which runs one sequence.
 *
 * Pointers follow llama_hip_kernels.h: device memory in place (stream-ordered on the library stream, no wait),
 * registered host ranges through their device copies, other host memory copied in and out around a synchronous call.
 * The index arrays (start, length, slot, adapter, tokens) are read on the device when the call runs, so a captured call
 * follows what they hold at each replay; an index outside its range is never followed and fails at the next
 * host-visible point (llhip_synchronize, or the end of a staged call), as an embedding id does. */
#ifndef LLAMA_HIP_REQUESTS_H
#define LLAMA_HIP_REQUESTS_H

#include <stddef.h>
#include <stdint.h>

#include "llama_hip_forward.h"
#include "llama_hip_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Requests 0 .. count - 1 (at most LLHIP_MAX_REQUESTS). Request r's rows are start[r] .. start[r + 1] - 1 of the row
 * buffers: its next token, or that and drafted tokens, or a prompt; none is allowed. Its row j lies at own position
 * length[r] + j, behind the `prefix` positions that all requests share, so at position prefix + length[r] + j of its
 * sequence. Rows before start[0] and from start[count] on belong to nobody and are left as they are. Its cache is slot
 * slot[r] (slot NULL: r) of key and value caches that hold `slots` of them, each seq_len positions of n_kv_heads heads
 * in the selected layout (kernels_kv_layout_name), one behind the other. */
typedef struct {
  const int *start;   /* count + 1 */
  const int *length;  /* count: own positions before the request's first row */
  const int *slot;    /* count, or NULL */
  int count;
  int rows;           /* rows that the row buffers hold */
  int prefix;         /* shared positions, 0 for none */
  int prefix_seq_len; /* positions that the prefix caches hold (the layout's strides) */
  int seq_len;        /* own positions that a slot holds */
  int slots;
} RequestBatch;
enum { LLHIP_MAX_REQUESTS = 1024 };

/* RoPE of the rows at their requests' positions, and their cache rows, in one launch: q_out = q's n_heads heads rotated
 * as k_rope_apply rotates them (bitwise), k's n_kv_heads heads rotated and v copied into the request's slot at own
 * position length[r] + j. table: prefix + seq_len rows of k_rope_table, position by position. q_out has q's stride and
 * may be q itself; k and v stay as they are. No two requests of a call may share a slot (that fails at the next
 * host-visible point; the slot's rows are then one of them's). q_out, the rows, both caches and the batch's arrays must
 * not overlap otherwise; head_dim even and at most 256. A launch holds 2^23 blocks, each of two q heads or one KV head of
 * 1024 / head_dim rows (512 / head_dim unless head_dim and the strides are multiples of 4 and the buffers 16-byte aligned):
 * more rows, over two million of 32 + 8 heads of 128, are refused. */
void llhip_rope_kv_store_requests(float *q_out, const float *q, size_t q_stride, const float *k, const float *v,
                                  size_t kv_stride, const float *table, const RequestBatch *batch, int n_heads,
                                  int n_kv_heads, int head_dim, float *key_cache, float *value_cache);

/* Causal attention of every request's rows over the shared prefix and then the request's own positions: row j of
 * request r attends to positions 0 .. prefix - 1 of prefix_key / prefix_value and to own positions 0 .. length[r] + j of
 * its slot (whose last rows llhip_rope_kv_store_requests stored). q and out hold rows of n_heads * head_dim floats;
 * scores, softmax and value sums as in k_attention (FP32-accurate; a non-finite score fails with "nonfinite value in
 * softmax"). The sums are divided by the weights' at the end, so n positions' values must stay below 3e38 / n, as there.
 * Where a tile has more than 32 query vectors (a KV head's heads of its rows), the products are of two FP16 parts, with FP32
 * sums: a factor is exact to 2^-22 of itself or, where that is more, to 2^-39 of the largest of its query vector, its K row
 * (both taken as at least 2^-100) or its group of four V rows, and a weight to 2^-24 of its row's largest, or 2^-36 over V
 * rows of about one size; V rows more than 16 to 4096 times apart in size, and smaller tiles, take FP32 products.
 *
 * Tiles are of 128 query vectors of a KV head, of all requests' rows together, and the prefix is read once for each. They are
 * formed where head_dim is a multiple of 4 and at most 128, the buffers are 16-byte aligned, the prefix and a slot of one
 * KV head (in the rows layout: of all) are below 2 GiB, and there are at most 2^20 rows, 1024 heads and 2^33 floats of q.
 * Any other shape has each row read what it attends to by itself, some ten to hundred times slower. prefix_key and
 * prefix_value may be NULL where prefix is 0; requests may share a slot here. out must not overlap q, a cache or the
 * batch's arrays. The shapes are k_attention's: n_heads a multiple of n_kv_heads, at most 16 per KV head, head_dim at
 * most 256. */
void llhip_attention_requests(float *out, const float *q, const float *prefix_key, const float *prefix_value,
                              const float *key_cache, const float *value_cache, const RequestBatch *batch, int n_heads,
                              int n_kv_heads, int head_dim);

/* Low-rank adapters of many requests beside projections that all rows share. Row i of x (m rows of k floats, leading
 * dimension ldx) has adapter adapter[i], -1 for none, out of `adapters`; for up to three segments that share x (QKV),
 * with P the product B[a] (A[a] x) scaled by scale[a]:
 *   GEMM_ADD     c = base + P            base: the shared projection's rows (k_gemm_f32, _bf16, _q8 or a k_matmul)
 *   GEMM_SWIGLU  c = silu(base + P) * (base3 + P3), for W1 and W3 projected apart (GEMM_STORE)
 * A row without an adapter has P = 0. base and base3 have c's leading dimension, and either may be c itself. A is
 * adapters x rank x k and B adapters x n x rank, row-major; rank 1 .. LLHIP_MAX_LORA_RANK, the same for the segment's
 * adapters (smaller ones padded with zeros). Sums are FP32 throughout, also over BF16 adapters (the activations are not
 * rounded); a row of x, or an adapter, that holds an infinity or a NaN gives its rows' columns NaN or infinity. Rows and
 * A on 16-byte boundaries with k a multiple of 8 (ldx of 4), at most 4096 adapters and 2^20 rows take the matrix cores;
 * other shapes take each row by itself, some ten to twenty times slower for many rows, and up to 2^23 of them. c must not
 * overlap x, the ids, any segment's adapters or scales, or another segment's c or base. */
typedef struct {
  float *c;
  int ldc;
  const float *base;  /* m x n */
  const float *base3; /* GEMM_SWIGLU only */
  const float *a, *b;
  const float *a3, *b3; /* GEMM_SWIGLU only */
  const float *scale;   /* adapters, or NULL: 1 */
  int n, rank;
  GemmKind kind; /* GEMM_ADD or GEMM_SWIGLU */
} LoraSegment;
typedef struct {
  float *c;
  int ldc;
  const float *base, *base3;
  const uint16_t *a, *b, *a3, *b3; /* BF16 bits, as bf16_from_f32 gives them */
  const float *scale;
  int n, rank;
  GemmKind kind;
} LoraBf16Segment;
enum { LLHIP_MAX_LORA_RANK = 256 };
void llhip_lora_f32(const float *x, int ldx, int m, int k, const int *adapter, int adapters, const LoraSegment *segments,
                    int count);
void llhip_lora_bf16(const float *x, int ldx, int m, int k, const int *adapter, int adapters,
                     const LoraBf16Segment *segments, int count);

/* Drafted tokens checked against the model (speculative sampling). Request r's rows start[r] .. start[r + 1] - 1 are as
 * in RequestBatch: the first row's token is known, row i's token tokens[i] of the others was drafted, and row i's
 * logits (vocab floats at logits + i * ld) judge row i + 1's token. With p = softmax(logits / temperature) of row i and q
 * the same of draft_logits' row i (the distribution that row i + 1's draft was drawn from; draft_logits NULL: the draft
 * was not drawn, q is 1 at it), the drafts are accepted in turn while uniform[2 i] * q(x) < p(x). At the first refusal the
 * next token is drawn from max(0, p - q) (from p should that be empty); with every draft accepted, from the last row's p:
 * the first token, in ascending order, at which the running sum passes uniform[2 i + 1] times the whole sum. The tokens
 * so emitted are distributed as the model's own. temperature 0 is greedy: a draft is accepted where it is the row's
 * largest logit (the lowest such token), which is also the next token; uniform and draft_logits are then not read.
 * accepted[r] receives the number of accepted drafts and next[r] the token after them; a request without rows keeps
 * both. Logits of -infinity are tokens masked out. A row that decides with a NaN, +infinity or no token left, and a
 * draft outside the vocabulary, set both to -1 and fail at the next host-visible point. Probabilities, sums and the
 * borders between tokens are FP64; uniform lies in [0, 1). draft_logits holds rows - 1 rows: a request's last row has no
 * draft behind it, and the buffer's last row is not read. accepted and next must not overlap each other or an input,
 * draft_logits taken as `rows` rows. At most LLHIP_MAX_REQUESTS requests, 2^20 rows and 2^22 tokens. */
void llhip_verify_drafts(int *accepted, int *next, const float *logits, size_t ld, const float *draft_logits,
                         size_t draft_ld, const int *tokens, const float *uniform, const int *start, int count, int rows,
                         int vocab, float temperature);

#ifdef __cplusplus
}
#endif
#endif
