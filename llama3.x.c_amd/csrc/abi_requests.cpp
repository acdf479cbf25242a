// The C entry points for many requests on one model (include/llama_hip_requests.h): argument checks, pointer residency
// as for the other calls, one stream-ordered operation per call.
#include <cmath>
#include <cstring>
#include <mutex>

#include "common.h"
#include "llama_hip_requests.h"

using namespace llhip;

namespace {

constexpr size_t kFloat = sizeof(float);

bool overlaps(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  return a && b && (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// The batch's own numbers: what the host can know of it (the arrays are checked on the device).
bool batch_ok(const char *name, const RequestBatch *b) {
  if (!b || !b->start || !b->length)
    return raise("%s: null batch or index array", name);
  if (b->count > LLHIP_MAX_REQUESTS)
    return raise("%s: %d requests, at most %d are taken in one call", name, b->count, (int)LLHIP_MAX_REQUESTS);
  if (b->seq_len <= 0 || b->slots <= 0 || b->prefix < 0 || b->prefix > b->prefix_seq_len ||
      b->seq_len > INT32_MAX - b->prefix_seq_len)
    return raise("%s: a prefix of %d positions in a cache of %d, %d slots of %d positions", name, b->prefix,
                 b->prefix_seq_len, b->slots, b->seq_len);
  return true;
}

// The layout's strides for the batch, and its arrays resolved by `call`.
struct BatchRefs {
  Ref start, length, slot;
};

BatchRefs batch_refs(Call &call, const RequestBatch *b) {
  const size_t n = (size_t)b->count;
  return BatchRefs{call.in(b->start, (n + 1) * sizeof(int)), call.in(b->length, n * sizeof(int)),
                   call.in(b->slot, n * sizeof(int))};
}

RequestsDev batch_dev(const Call &call, const BatchRefs &r, const RequestBatch *b, int n_kv_heads, int head_dim) {
  RequestsDev d{};
  d.start = call.ptr<const int>(r.start);
  d.length = call.ptr<const int>(r.length);
  d.slot = b->slot ? call.ptr<const int>(r.slot) : nullptr;
  d.count = b->count;
  d.rows = b->rows;
  d.prefix = b->prefix;
  d.seq_len = b->seq_len;
  d.slots = b->slots;
  k_kv_strides(n_kv_heads, head_dim, b->seq_len, &d.pos_stride, &d.head_base);
  k_kv_strides(n_kv_heads, head_dim, b->prefix_seq_len, &d.prefix_pos_stride, &d.prefix_head_base);
  d.slot_floats = (size_t)b->seq_len * n_kv_heads * head_dim;
  return d;
}

// Whether a call that writes these bytes would write over the batch's arrays, which its other blocks still read.
bool over_arrays(const RequestBatch *b, const void *out, size_t bytes) {
  const size_t n = (size_t)b->count * sizeof(int);
  return overlaps(out, bytes, b->start, n + sizeof(int)) || overlaps(out, bytes, b->length, n) ||
         overlaps(out, bytes, b->slot, n);
}

size_t caches_bytes(const RequestBatch *b, int n_kv_heads, int head_dim) {
  return (size_t)b->slots * b->seq_len * n_kv_heads * head_dim * kFloat;
}

// The scratch of these calls, which the library stream orders: grown on demand (never during graph capture), kept for the
// process. A graph captured on it replays on it, so a buffer that a capture took is kept when a larger one follows. A call
// holds the lock until its kernels are queued, so that another thread's do not come between them.
std::mutex scratch_mutex;
void *scratch_memory = nullptr;
size_t scratch_bytes = 0;
bool scratch_captured = false;

bool workspace(const char *name, size_t bytes, void **out) {
  Device &dev = device();
  if (bytes > scratch_bytes) {
    if (dev.capturing)
      return raise("%s needs %zu bytes of workspace during graph capture; run the call once before capturing", name, bytes);
    if (scratch_memory && !scratch_captured) {
      (void)hipStreamSynchronize(dev.stream);
      (void)hipFree(scratch_memory);
      hbm_release(scratch_bytes);
    }
    scratch_memory = nullptr;
    scratch_bytes = 0;
    scratch_captured = false;
    const size_t want = bytes + bytes / 4 + 4096;
    if (!hbm_claim(want, "the request workspace"))
      return false;
    if (hipMalloc(&scratch_memory, want) != hipSuccess) {
      (void)hipGetLastError();
      hbm_release(want);
      scratch_memory = nullptr;
      return raise("%s: allocating %zu bytes of workspace failed", name, want);
    }
    scratch_bytes = want;
  }
  if (dev.capturing)
    scratch_captured = true;
  *out = scratch_memory;
  return true;
}

// One adapter call, F32 or BF16: the segment types differ in their adapters' element only.
template <class Segment>
void lora(const char *name, const float *x, int ldx, int m, int k, const int *adapter, int adapters,
          const Segment *segments, int count, bool bf16) {
  const size_t element = bf16 ? 2 : kFloat;
  if (m <= 0 || count <= 0)
    return;
  if (count > GEMM_MAX_SEGMENTS || !segments) {
    raise("%s: %d segments, 1 to %d are taken", name, count, (int)GEMM_MAX_SEGMENTS);
    return;
  }
  if (k <= 0 || ldx < k || adapters <= 0 || !x || !adapter) {
    raise("%s: rows of %d values at stride %d, %d adapters, or a null buffer", name, k, ldx, adapters);
    return;
  }
  const size_t x_bytes = ((size_t)(m - 1) * ldx + k) * kFloat;
  for (int i = 0; i < count; i++) {
    const Segment &s = segments[i];
    const bool swiglu = s.kind == GEMM_SWIGLU;
    if (s.kind != GEMM_ADD && !swiglu) {
      raise("%s: segment %d has kind %d, not GEMM_ADD or GEMM_SWIGLU", name, i, (int)s.kind);
      return;
    }
    if (s.n <= 0 || s.ldc < s.n || s.rank <= 0 || s.rank > LLHIP_MAX_LORA_RANK) {
      raise("%s: segment %d has %d columns at stride %d and rank %d (1 to %d)", name, i, s.n, s.ldc, s.rank,
            (int)LLHIP_MAX_LORA_RANK);
      return;
    }
    if (!s.c || !s.base || !s.a || !s.b || (swiglu && (!s.base3 || !s.a3 || !s.b3))) {
      raise("%s: segment %d has a null buffer", name, i);
      return;
    }
  }
  for (int i = 0; i < count; i++) {
    const Segment &s = segments[i];
    const size_t out = ((size_t)(m - 1) * s.ldc + s.n) * kFloat;
    bool bad = overlaps(s.c, out, x, x_bytes) || overlaps(s.c, out, adapter, (size_t)m * sizeof(int)) ||
               (s.base != s.c && overlaps(s.c, out, s.base, out));
    if (s.kind == GEMM_SWIGLU)
      bad |= s.base3 != s.c && overlaps(s.c, out, s.base3, out);
    for (int j = 0; j < count; j++) {
      const Segment &t = segments[j];
      const size_t other = ((size_t)(m - 1) * t.ldc + t.n) * kFloat;
      const size_t a_bytes = (size_t)adapters * t.rank * k * element, b_bytes = (size_t)adapters * t.n * t.rank * element;
      // segments side by side in one row buffer (QKV rows) share an extent: their columns must differ
      auto apart = [&](const float *p) {
        if (!overlaps(s.c, out, p, other))
          return true;
        const ptrdiff_t gap = s.c - p;
        return s.ldc == t.ldc && ((gap >= t.n && gap + s.n <= s.ldc) || (-gap >= s.n && -gap + t.n <= s.ldc));
      };
      const bool swiglu = t.kind == GEMM_SWIGLU;
      if (j != i)
        bad |= !apart(t.c) || !apart(t.base) || (swiglu && !apart(t.base3));
      bad |= overlaps(s.c, out, t.a, a_bytes) || overlaps(s.c, out, t.b, b_bytes) ||
             overlaps(s.c, out, t.scale, (size_t)adapters * kFloat);
      if (swiglu)
        bad |= overlaps(s.c, out, t.a3, a_bytes) || overlaps(s.c, out, t.b3, b_bytes);
    }
    if (bad) {
      raise("%s: segment %d's output overlaps an input or another segment", name, i);
      return;
    }
  }
  Call call(name);
  Ref X = call.in2d(x, (size_t)k * kFloat, (size_t)ldx * kFloat, (size_t)m), I = call.in(adapter, (size_t)m * sizeof(int));
  Ref C[3], B0[3], B3[3], W[3][4], S[3];
  for (int i = 0; i < count; i++) {
    const Segment &s = segments[i];
    const bool swiglu = s.kind == GEMM_SWIGLU;
    const size_t row = (size_t)s.n * kFloat, pitch = (size_t)s.ldc * kFloat;
    const size_t a_bytes = (size_t)adapters * s.rank * k * element, b_bytes = (size_t)adapters * s.n * s.rank * element;
    const bool in_place = s.base == s.c || (swiglu && s.base3 == s.c);
    C[i] = call.out2d(s.c, row, pitch, (size_t)m, in_place);
    B0[i] = s.base == s.c ? C[i] : call.in2d(s.base, row, pitch, (size_t)m);
    B3[i] = !swiglu ? Ref{} : s.base3 == s.c ? C[i] : call.in2d(s.base3, row, pitch, (size_t)m);
    W[i][0] = call.in(s.a, a_bytes);
    W[i][1] = call.in(s.b, b_bytes);
    W[i][2] = swiglu ? call.in(s.a3, a_bytes) : Ref{};
    W[i][3] = swiglu ? call.in(s.b3, b_bytes) : Ref{};
    S[i] = call.in(s.scale, (size_t)adapters * kFloat);
  }
  if (!call.ready())
    return;
  LoraJob job{};
  job.x = call.ptr<const float>(X);
  job.adapter = call.ptr<const int>(I);
  job.ldx = ldx;
  job.m = m;
  job.k = k;
  job.adapters = adapters;
  job.nseg = count;
  job.bf16 = bf16;
  for (int i = 0; i < count; i++) {
    const Segment &s = segments[i];
    const bool swiglu = s.kind == GEMM_SWIGLU;
    job.seg[i] = LoraSegmentDev{call.ptr<float>(C[i]), call.ptr<const float>(B0[i]),
                                swiglu ? call.ptr<const float>(B3[i]) : nullptr, call.ptr<const void>(W[i][0]),
                                call.ptr<const void>(W[i][1]), swiglu ? call.ptr<const void>(W[i][2]) : nullptr,
                                swiglu ? call.ptr<const void>(W[i][3]) : nullptr,
                                s.scale ? call.ptr<const float>(S[i]) : nullptr, s.ldc, s.n, s.rank, swiglu};
  }
  std::unique_lock<std::mutex> lock(scratch_mutex);
  void *scratch = nullptr;
  if (!workspace(name, lora_workspace(job), &scratch))
    return;
  if (!launch_lora(job, scratch, call.stream()))
    return;
  lock.unlock();
  call.finish();
}

} // namespace

extern "C" {

void llhip_rope_kv_store_requests(float *q_out, const float *q, size_t q_stride, const float *k, const float *v,
                                  size_t kv_stride, const float *table, const RequestBatch *batch, int n_heads,
                                  int n_kv_heads, int head_dim, float *key_cache, float *value_cache) {
  const char *name = "llhip_rope_kv_store_requests";
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
  if (q_stride < dq || kv_stride < dkv) {
    raise("%s: a row stride is shorter than its row", name);
    return;
  }
  if (!q_out || !q || !k || !v || !table || !key_cache || !value_cache) {
    raise("%s: null buffer", name);
    return;
  }
  const size_t q_bytes = ((rows - 1) * q_stride + dq) * kFloat, kv_bytes = ((rows - 1) * kv_stride + dkv) * kFloat;
  const size_t cache = caches_bytes(batch, n_kv_heads, head_dim);
  const size_t table_bytes = ((size_t)batch->prefix + batch->seq_len) * 2 * head_dim * kFloat;
  // rows side by side in one buffer (QKV rows) share an extent: k's and v's columns must not be q's
  auto apart = [&](const float *p) {
    if (!overlaps(q_out, q_bytes, p, kv_bytes))
      return true;
    const ptrdiff_t gap = p - q_out;
    return q_stride == kv_stride && ((gap >= (ptrdiff_t)dq && gap + (ptrdiff_t)dkv <= (ptrdiff_t)q_stride) ||
                                     (-gap >= (ptrdiff_t)dkv && -gap + (ptrdiff_t)dq <= (ptrdiff_t)q_stride));
  };
  bool bad = overlaps(key_cache, cache, value_cache, cache) || (q_out != q && overlaps(q_out, q_bytes, q, q_bytes)) ||
             !apart(k) || !apart(v) || overlaps(table, table_bytes, q_out, q_bytes) || over_arrays(batch, q_out, q_bytes);
  for (float *c : {key_cache, value_cache})
    bad |= overlaps(c, cache, q, q_bytes) || overlaps(c, cache, q_out, q_bytes) || overlaps(c, cache, k, kv_bytes) ||
           overlaps(c, cache, v, kv_bytes) || overlaps(c, cache, table, table_bytes) || over_arrays(batch, c, cache);
  if (bad) {
    raise("%s: q_out, the rows, the table, the caches and the batch's arrays must not overlap", name);
    return;
  }
  Call call(name);
  const BatchRefs refs = batch_refs(call, batch);
  // read too: rows that belong to no request keep what they hold
  Ref O = call.out2d(q_out, dq * kFloat, q_stride * kFloat, rows, true);
  Ref Q = q_out == q ? O : call.in2d(q, dq * kFloat, q_stride * kFloat, rows);
  Ref K = call.in2d(k, dkv * kFloat, kv_stride * kFloat, rows), V = call.in2d(v, dkv * kFloat, kv_stride * kFloat, rows);
  Ref T = call.in(table, table_bytes);
  Ref KC = call.out(key_cache, cache, true), VC = call.out(value_cache, cache, true);
  if (!call.ready())
    return;
  const RopeRequestsJob job{call.ptr<float>(O), call.ptr<const float>(Q), call.ptr<const float>(K),
                            call.ptr<const float>(V), call.ptr<const float>(T), q_stride, kv_stride,
                            batch_dev(call, refs, batch, n_kv_heads, head_dim), n_heads, n_kv_heads, head_dim,
                            call.ptr<float>(KC), call.ptr<float>(VC)};
  if (launch_rope_requests(job, call.stream()))
    call.finish();
}

void llhip_attention_requests(float *out, const float *q, const float *prefix_key, const float *prefix_value,
                              const float *key_cache, const float *value_cache, const RequestBatch *batch, int n_heads,
                              int n_kv_heads, int head_dim) {
  const char *name = "llhip_attention_requests";
  if (batch && (batch->count <= 0 || batch->rows <= 0))
    return;
  if (!batch_ok(name, batch))
    return;
  if (!attention_shape_ok(n_heads, n_kv_heads, head_dim)) {
    raise("%s: %d heads over %d KV heads of dimension %d are not supported (n_heads a multiple of n_kv_heads, at most "
          "16 per KV head, head_dim <= 256)", name, n_heads, n_kv_heads, head_dim);
    return;
  }
  if (!out || !q || !key_cache || !value_cache || (batch->prefix > 0 && (!prefix_key || !prefix_value))) {
    raise("%s: null buffer", name);
    return;
  }
  const size_t row_bytes = (size_t)batch->rows * n_heads * head_dim * kFloat;
  const size_t cache = caches_bytes(batch, n_kv_heads, head_dim);
  size_t pos_stride, head_base;
  k_kv_strides(n_kv_heads, head_dim, batch->prefix_seq_len, &pos_stride, &head_base);
  const size_t prefix_bytes =
      batch->prefix ? ((size_t)(batch->prefix - 1) * pos_stride + (size_t)(n_kv_heads - 1) * head_base + head_dim) * kFloat
                    : 0;
  if (overlaps(out, row_bytes, q, row_bytes) || overlaps(out, row_bytes, key_cache, cache) ||
      overlaps(out, row_bytes, value_cache, cache) || overlaps(out, row_bytes, prefix_key, prefix_bytes) ||
      overlaps(out, row_bytes, prefix_value, prefix_bytes) || over_arrays(batch, out, row_bytes)) {
    raise("%s: out must not overlap q, a cache or the batch's arrays", name);
    return;
  }
  Call call(name);
  const BatchRefs refs = batch_refs(call, batch);
  Ref Q = call.in(q, row_bytes);
  Ref PK = batch->prefix ? call.in(prefix_key, prefix_bytes) : Ref{};
  Ref PV = batch->prefix ? call.in(prefix_value, prefix_bytes) : Ref{};
  Ref K = call.in(key_cache, cache), V = call.in(value_cache, cache);
  Ref O = call.out(out, row_bytes, true); // read too: rows that belong to no request keep what they hold
  if (!call.ready())
    return;
  AttentionRequestsJob job{call.ptr<float>(O), call.ptr<const float>(Q),
                           batch->prefix ? call.ptr<const float>(PK) : nullptr,
                           batch->prefix ? call.ptr<const float>(PV) : nullptr, call.ptr<const float>(K),
                           call.ptr<const float>(V), batch_dev(call, refs, batch, n_kv_heads, head_dim), n_heads,
                           n_kv_heads, head_dim};
  std::unique_lock<std::mutex> lock(scratch_mutex);
  void *scratch = nullptr;
  if (!workspace(name, attention_requests_workspace(job), &scratch))
    return;
  if (!launch_attention_requests(job, scratch, call.stream()))
    return;
  lock.unlock();
  call.finish();
}

void llhip_lora_f32(const float *x, int ldx, int m, int k, const int *adapter, int adapters, const LoraSegment *segments,
                    int count) {
  lora("llhip_lora_f32", x, ldx, m, k, adapter, adapters, segments, count, false);
}

void llhip_lora_bf16(const float *x, int ldx, int m, int k, const int *adapter, int adapters,
                     const LoraBf16Segment *segments, int count) {
  lora("llhip_lora_bf16", x, ldx, m, k, adapter, adapters, segments, count, true);
}

void llhip_verify_drafts(int *accepted, int *next, const float *logits, size_t ld, const float *draft_logits,
                         size_t draft_ld, const int *tokens, const float *uniform, const int *start, int count, int rows,
                         int vocab, float temperature) {
  const char *name = "llhip_verify_drafts";
  if (count <= 0 || rows <= 0)
    return;
  const bool greedy = temperature == 0.0f;
  if (!(temperature >= 0.0f) || !std::isfinite(temperature)) {
    raise("%s: temperature %g must be finite and not negative", name, (double)temperature);
    return;
  }
  if (count > LLHIP_MAX_REQUESTS) {
    raise("%s: %d requests, at most %d are taken in one call", name, count, (int)LLHIP_MAX_REQUESTS);
    return;
  }
  if (greedy)
    draft_logits = nullptr;
  if (vocab <= 0 || ld < (size_t)vocab || (draft_logits && draft_ld < (size_t)vocab)) {
    raise("%s: rows of %d logits at strides %zu and %zu", name, vocab, ld, draft_logits ? draft_ld : ld);
    return;
  }
  if (!verify_shape_ok(rows, vocab)) {
    raise("%s: %d rows of %d tokens, at most 2^20 rows of 2^22 tokens are taken", name, rows, vocab);
    return;
  }
  if (!accepted || !next || !logits || !tokens || !start || (!greedy && !uniform)) {
    raise("%s: null buffer", name);
    return;
  }
  const size_t out_bytes = (size_t)count * sizeof(int);
  if (overlaps(accepted, out_bytes, next, out_bytes)) {
    raise("%s: accepted and next must not overlap", name);
    return;
  }
  const size_t logits_bytes = ((size_t)(rows - 1) * ld + vocab) * kFloat;
  const size_t draft_bytes = ((size_t)(rows - 1) * draft_ld + vocab) * kFloat;
  for (const int *out : {accepted, next})
    if (overlaps(out, out_bytes, logits, logits_bytes) || overlaps(out, out_bytes, draft_logits, draft_bytes) ||
        overlaps(out, out_bytes, tokens, (size_t)rows * sizeof(int)) ||
        overlaps(out, out_bytes, start, ((size_t)count + 1) * sizeof(int)) ||
        (!greedy && overlaps(out, out_bytes, uniform, (size_t)rows * 2 * kFloat))) {
      raise("%s: accepted and next must not overlap an input", name);
      return;
    }
  if (rows == 1)
    draft_logits = nullptr; // nothing is drafted
  Call call(name);
  const size_t row = (size_t)vocab * kFloat;
  Ref A = call.out(accepted, out_bytes, true), N = call.out(next, out_bytes, true); // requests without rows keep both
  Ref L = call.in2d(logits, row, ld * kFloat, (size_t)rows);
  // the buffer's last row judges nothing: its draft_logits row need not be there
  Ref D = draft_logits ? call.in2d(draft_logits, row, draft_ld * kFloat, (size_t)rows - 1) : Ref{};
  Ref T = call.in(tokens, (size_t)rows * sizeof(int)), S = call.in(start, ((size_t)count + 1) * sizeof(int));
  Ref U = greedy ? Ref{} : call.in(uniform, (size_t)rows * 2 * kFloat);
  if (!call.ready())
    return;
  const VerifyJob job{call.ptr<int>(A), call.ptr<int>(N), call.ptr<const float>(L),
                      draft_logits ? call.ptr<const float>(D) : nullptr, ld, draft_ld, call.ptr<const int>(T),
                      call.ptr<const int>(S), greedy ? nullptr : call.ptr<const float>(U), count, rows, vocab,
                      temperature};
  std::unique_lock<std::mutex> lock(scratch_mutex);
  void *scratch = nullptr;
  if (!workspace(name, verify_workspace(job), &scratch))
    return;
  if (!launch_verify(job, scratch, call.stream()))
    return;
  lock.unlock();
  call.finish();
}

} // extern "C"
