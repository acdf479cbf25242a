// The C entry points of a cache in pages (include/llama_hip_paged.h): argument checks, pointer residency as for the other
// calls, one stream-ordered operation per call.
#include "common.h"
#include "llama_hip_forward.h"
#include "llama_hip_paged.h"

using namespace llhip;

namespace {

constexpr size_t kFloat = sizeof(float);

size_t value_bytes(const PagedBatch *b) { return b->type == PAGE_BF16 ? 2 : kFloat; }

// The batch's own numbers: what the host can know of it (the arrays are checked on the device).
bool batch_ok(const char *name, const PagedBatch *b) {
  if (!b || !b->start || !b->length || !b->pages)
    return raise("%s: null batch or index array", name);
  if (b->type != PAGE_F32 && b->type != PAGE_BF16)
    return raise("%s: pages of type %d, not PAGE_F32 or PAGE_BF16", name, (int)b->type);
  if (b->count > LLHIP_MAX_REQUESTS)
    return raise("%s: %d requests, at most %d are taken in one call", name, b->count, (int)LLHIP_MAX_REQUESTS);
  if (b->page_size <= 0 || b->max_pages <= 0 || b->num_pages <= 0 || b->seq_len <= 0 ||
      b->seq_len > (long long)b->max_pages * b->page_size)
    return raise("%s: %d positions of a request in at most %d pages of %d, %d pages in all", name, b->seq_len, b->max_pages,
                 b->page_size, b->num_pages);
  return true;
}

size_t table_ints(const PagedBatch *b) { return (size_t)b->count * b->max_pages; }

size_t cache_bytes(const PagedBatch *b, int n_kv_heads, int head_dim) {
  return product(product((size_t)b->num_pages * b->page_size, (size_t)n_kv_heads * head_dim), value_bytes(b));
}

// Whether a call that writes these bytes would write over the batch's arrays, which its other blocks still read.
bool over_arrays(const PagedBatch *b, const void *out, size_t bytes) {
  const size_t n = (size_t)b->count * sizeof(int);
  return overlaps(out, bytes, b->start, n + sizeof(int)) || overlaps(out, bytes, b->length, n) ||
         overlaps(out, bytes, b->pages, table_ints(b) * sizeof(int));
}

struct BatchRefs {
  Ref start, length, pages;
};

BatchRefs batch_refs(Call &call, const PagedBatch *b) {
  const size_t n = (size_t)b->count;
  return BatchRefs{call.in(b->start, (n + 1) * sizeof(int)), call.in(b->length, n * sizeof(int)),
                   call.in(b->pages, table_ints(b) * sizeof(int))};
}

PagedDev batch_dev(const Call &call, const BatchRefs &r, const PagedBatch *b, int n_kv_heads, int head_dim) {
  PagedDev d{};
  d.start = call.ptr<const int>(r.start);
  d.length = call.ptr<const int>(r.length);
  d.pages = call.ptr<const int>(r.pages);
  d.count = b->count;
  d.rows = b->rows;
  d.max_pages = b->max_pages;
  d.page_size = b->page_size;
  d.num_pages = b->num_pages;
  d.seq_len = b->seq_len;
  d.bf16 = b->type == PAGE_BF16;
  k_kv_strides(n_kv_heads, head_dim, b->page_size, &d.pos_stride, &d.head_base);
  d.page_values = (size_t)b->page_size * n_kv_heads * head_dim;
  return d;
}

// Whether rows of `an` floats at stride `as` and rows of `bn` at stride `bs`, n of each, share a float. Rows side by side
// in one buffer (QKV rows) share an extent, but not their columns.
bool rows_meet(const float *a, size_t an, size_t as, const float *b, size_t bn, size_t bs, size_t n) {
  if (!overlaps(a, ((n - 1) * as + an) * kFloat, b, ((n - 1) * bs + bn) * kFloat))
    return false;
  if (as != bs)
    return true;
  const ptrdiff_t gap = b - a;
  return !((gap >= (ptrdiff_t)an && gap + (ptrdiff_t)bn <= (ptrdiff_t)as) ||
           (-gap >= (ptrdiff_t)bn && -gap + (ptrdiff_t)an <= (ptrdiff_t)as));
}

} // namespace

extern "C" {

void llhip_rope_kv_append_paged(float *q_out, size_t q_out_stride, const float *q, size_t q_stride, const float *k,
                                const float *v, size_t kv_stride, const float *table, const float *q_norm,
                                const float *k_norm, float epsilon, const PagedBatch *batch, int n_heads, int n_kv_heads,
                                int head_dim, void *key_pages, void *value_pages) {
  const char *name = "llhip_rope_kv_append_paged";
  if (batch && (batch->count <= 0 || batch->rows <= 0))
    return;
  if (!batch_ok(name, batch))
    return;
  if (!attention_shape_ok(n_heads, n_kv_heads, head_dim) || head_dim % 2) {
    raise("%s: %d heads over %d KV heads of dimension %d are not supported (n_heads a multiple of n_kv_heads, at most "
          "16 per KV head, head_dim even and <= 256)", name, n_heads, n_kv_heads, head_dim);
    return;
  }
  const size_t dq = (size_t)n_heads * head_dim, dkv = (size_t)n_kv_heads * head_dim, rows = (size_t)batch->rows;
  if (q_out_stride < dq || q_stride < dq || kv_stride < dkv) {
    raise("%s: a row stride is shorter than its row", name);
    return;
  }
  if (!q_out || !q || !k || !v || !table || !key_pages || !value_pages) {
    raise("%s: null buffer", name);
    return;
  }
  if (q_out == q && q_out_stride != q_stride) {
    raise("%s: q_out is q at another stride (%zu and %zu)", name, q_out_stride, q_stride);
    return;
  }
  const size_t q_bytes = rows_bytes(rows, q_stride, dq), out_bytes = rows_bytes(rows, q_out_stride, dq);
  const size_t kv_bytes = rows_bytes(rows, kv_stride, dkv), norm_bytes = (size_t)head_dim * kFloat;
  const size_t cache = cache_bytes(batch, n_kv_heads, head_dim);
  if (q_bytes >= kNoRoom || out_bytes >= kNoRoom || kv_bytes >= kNoRoom || cache >= kNoRoom) {
    raise("%s: the rows or the caches take more than 2^56 bytes", name);
    return;
  }
  const size_t table_bytes = (size_t)batch->seq_len * 2 * head_dim * kFloat;
  bool bad = overlaps(key_pages, cache, value_pages, cache) ||
             (q_out != q && rows_meet(q_out, dq, q_out_stride, q, dq, q_stride, rows)) ||
             rows_meet(q_out, dq, q_out_stride, k, dkv, kv_stride, rows) ||
             rows_meet(q_out, dq, q_out_stride, v, dkv, kv_stride, rows) ||
             overlaps(table, table_bytes, q_out, out_bytes) || overlaps(q_norm, norm_bytes, q_out, out_bytes) ||
             overlaps(k_norm, norm_bytes, q_out, out_bytes) || over_arrays(batch, q_out, out_bytes);
  for (const void *c : {key_pages, value_pages})
    bad |= overlaps(c, cache, q, q_bytes) || overlaps(c, cache, q_out, out_bytes) || overlaps(c, cache, k, kv_bytes) ||
           overlaps(c, cache, v, kv_bytes) || overlaps(c, cache, table, table_bytes) ||
           overlaps(c, cache, q_norm, norm_bytes) || overlaps(c, cache, k_norm, norm_bytes) || over_arrays(batch, c, cache);
  if (bad) {
    raise("%s: q_out, the rows, the table, the norms, the caches and the batch's arrays must not overlap", name);
    return;
  }
  Call call(name);
  const BatchRefs refs = batch_refs(call, batch);
  // read too: rows that belong to no request keep what they hold
  Ref O = call.out2d(q_out, dq * kFloat, q_out_stride * kFloat, rows, true);
  Ref Q = q_out == q ? O : call.in2d(q, dq * kFloat, q_stride * kFloat, rows);
  Ref K = call.in2d(k, dkv * kFloat, kv_stride * kFloat, rows), V = call.in2d(v, dkv * kFloat, kv_stride * kFloat, rows);
  Ref T = call.in(table, table_bytes), QN = call.in(q_norm, norm_bytes), KN = call.in(k_norm, norm_bytes);
  Ref KC = call.out(key_pages, cache, true), VC = call.out(value_pages, cache, true);
  if (!call.ready())
    return;
  const AppendPagedJob job{call.ptr<float>(O), call.ptr<const float>(Q), call.ptr<const float>(K),
                           call.ptr<const float>(V), call.ptr<const float>(T),
                           q_norm ? call.ptr<const float>(QN) : nullptr, k_norm ? call.ptr<const float>(KN) : nullptr,
                           q_out_stride, q_stride, kv_stride, epsilon,
                           batch_dev(call, refs, batch, n_kv_heads, head_dim), n_heads, n_kv_heads, head_dim,
                           call.ptr<void>(KC), call.ptr<void>(VC)};
  if (launch_append_paged(job, call.stream()))
    call.finish();
}

void llhip_attention_paged(float *out, const float *q, size_t q_stride, const void *key_pages, const void *value_pages,
                           const PagedBatch *batch, int n_heads, int n_kv_heads, int head_dim) {
  const char *name = "llhip_attention_paged";
  if (batch && (batch->count <= 0 || batch->rows <= 0))
    return;
  if (!batch_ok(name, batch))
    return;
  if (n_heads <= 0 || !attention_shape_ok(n_heads, n_kv_heads, head_dim)) {
    raise("%s: %d heads over %d KV heads of dimension %d are not supported (n_heads positive and a multiple of n_kv_heads, "
          "at most 16 per KV head, head_dim <= 256)", name, n_heads, n_kv_heads, head_dim);
    return;
  }
  const size_t dq = (size_t)n_heads * head_dim, rows = (size_t)batch->rows;
  if (q_stride < dq) {
    raise("%s: a row stride is shorter than its row", name);
    return;
  }
  if (!out || !q || !key_pages || !value_pages) {
    raise("%s: null buffer", name);
    return;
  }
  const size_t q_bytes = rows_bytes(rows, q_stride, dq), out_bytes = rows_bytes(rows, dq, dq);
  const size_t cache = cache_bytes(batch, n_kv_heads, head_dim);
  if (q_bytes >= kNoRoom || cache >= kNoRoom) {
    raise("%s: the rows or the caches take more than 2^56 bytes", name);
    return;
  }
  if (overlaps(out, out_bytes, q, q_bytes) || overlaps(out, out_bytes, key_pages, cache) ||
      overlaps(out, out_bytes, value_pages, cache) || over_arrays(batch, out, out_bytes)) {
    raise("%s: out must not overlap q, a cache or the batch's arrays", name);
    return;
  }
  Call call(name);
  const BatchRefs refs = batch_refs(call, batch);
  Ref Q = call.in2d(q, dq * kFloat, q_stride * kFloat, rows);
  Ref K = call.in(key_pages, cache), V = call.in(value_pages, cache);
  Ref O = call.out(out, out_bytes, true); // read too: rows that belong to no request keep what they hold
  if (!call.ready())
    return;
  const AttentionPagedJob job{call.ptr<float>(O), call.ptr<const float>(Q), q_stride, call.ptr<const void>(K),
                              call.ptr<const void>(V), batch_dev(call, refs, batch, n_kv_heads, head_dim), n_heads,
                              n_kv_heads, head_dim};
  std::unique_lock<std::mutex> lock(scratch_mutex);
  void *scratch = nullptr;
  const size_t bytes = attention_paged_workspace(job);
  if (bytes && !scratch_room(name, bytes, &scratch, SCRATCH_PAGES))
    return;
  if (!launch_attention_paged(job, scratch, call.stream()))
    return;
  lock.unlock();
  call.finish();
}

} // extern "C"
