// Many requests on one model (gfx950): RoPE and cache rows at each request's own position, and attention behind a
// prefix that all requests share.
//
//   rope_requests   one thread per V dimensions of a row's two q heads or of one KV head.
//   attn_rows       attention of one row and one KV head per block, any shape: the positions walked in chunks of 64 with
//                   the running maximum and sum of the softmax.
#include <cfloat>

#include "common.h"
#include "lanes.h"

namespace llhip {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kChunk = 64;
constexpr int kMaxGroup = 16;
constexpr int kMaxHeadDim = 256;
constexpr int kMaxRequests = 1024;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

// Request r's rows, own length and slot; no rows (and bad set) where they leave the batch's buffers. A request without
// rows may hold anything else.
struct Request {
  int first, rows, length, slot;
};
__device__ __forceinline__ Request request_at(const RequestsDev &b, int r, bool &bad) {
  const int first = b.start[r], last = b.start[r + 1], length = b.length[r], slot = b.slot ? b.slot[r] : r;
  const bool rows_ok = first >= 0 && first <= last && last <= b.rows;
  const int n = rows_ok ? last - first : 0;
  const bool ok = rows_ok && (n == 0 || (length >= 0 && length <= b.seq_len - n && slot >= 0 && slot < b.slots));
  bad |= !ok;
  return Request{first, ok ? n : 0, length, slot};
}

// ---- RoPE and cache rows ----------------------------------------------------------------------------------------------

__device__ __forceinline__ void rotate(float &a, float &b, float c, float s) {
#pragma clang fp contract(off) // the products rounded before the sum, as k_rope_apply computes them
  const float x = a, y = b;
  a = x * c - y * s;
  b = x * s + y * c;
}

template <int V> struct Vec {
  float v[V];
};
template <int V> __device__ __forceinline__ Vec<V> load_vec(const float *p) {
  Vec<V> x;
  if constexpr (V == 4)
    *reinterpret_cast<float4 *>(x.v) = *reinterpret_cast<const float4 *>(p);
  else
    x.v[0] = p[0], x.v[1] = p[1];
  return x;
}
template <int V> __device__ __forceinline__ void store_vec(float *p, const Vec<V> &x) {
  if constexpr (V == 4)
    *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(x.v);
  else
    p[0] = x.v[0], p[1] = x.v[1];
}

// Block (row group, unit): unit u takes q heads 2u and 2u + 1 of the group's rows, or one KV head's k and v; thread
// (row, item) V dimensions of them. V = 4 for 16-byte aligned rows of head_dim a multiple of 4, else 2. The block finds
// its rows' requests by looking through all of them, 256 at a time: one load each where a search per row would wait for
// its log2(count) loads in turn. Block 0 also looks for two requests in one slot, in a table of slots in LDS.
template <int V> __global__ __launch_bounds__(kThreads) void rope_requests(RopeRequestsJob p, int *flags) {
  constexpr int kTable = 2 * kMaxRequests;
  __shared__ int request_of[kThreads], position_of[kThreads], slot_of[kThreads];
  __shared__ int table[kTable];
  const int items = p.head_dim / V, per_block = kThreads / items;
  const int qunits = (p.n_heads + 1) / 2, units = qunits + p.n_kv_heads;
  const int unit = blockIdx.x % units;
  const int r0 = blockIdx.x / units * per_block;
  const bool first_block = blockIdx.x == 0;
  for (int i = threadIdx.x; i < per_block; i += kThreads)
    request_of[i] = -1;
  if (first_block)
    for (int i = threadIdx.x; i < kTable; i += kThreads)
      table[i] = -1;
  __syncthreads();
  bool bad = false, twice = false;
  for (int r = threadIdx.x; r < p.batch.count; r += kThreads) {
    const Request q = request_at(p.batch, r, bad);
    const int a = max(q.first, r0), b = min(q.first + q.rows, r0 + per_block);
    for (int i = a; i < b; i++) {
      request_of[i - r0] = r;
      position_of[i - r0] = q.length + i - q.first;
      slot_of[i - r0] = q.slot;
    }
    if (first_block && q.rows) { // at most 1024 entries in a table of 2048: a free one is always found
      int at = (int)((unsigned)q.slot * 2654435761u % kTable);
      while (true) {
        const int seen = atomicCAS(&table[at], -1, q.slot);
        if (seen == -1)
          break;
        if (seen == q.slot) {
          twice = true;
          break;
        }
        at = (at + 1) % kTable;
      }
    }
  }
  if (first_block && bad)
    flags[3] = 1;
  if (first_block && twice)
    flags[4] = 1;
  __syncthreads();
  const int local = threadIdx.x / items, d = threadIdx.x % items * V;
  if (local >= per_block || request_of[local] < 0)
    return;
  const int row = r0 + local, at = position_of[local], hd = p.head_dim;
  const float *t = p.table + (size_t)(p.batch.prefix + at) * 2 * hd;
  float c[V / 2], s[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; i++)
    c[i] = t[d + 2 * i], s[i] = t[hd + d + 2 * i + 1];
  auto turn = [&](Vec<V> x) {
#pragma unroll
    for (int i = 0; i < V / 2; i++)
      rotate(x.v[2 * i], x.v[2 * i + 1], c[i], s[i]);
    return x;
  };
  if (unit < qunits) {
    const size_t src = (size_t)row * p.q_stride + (size_t)(2 * unit) * hd + d;
    const bool two = 2 * unit + 1 < p.n_heads;
    const Vec<V> x0 = load_vec<V>(p.q + src), x1 = load_vec<V>(p.q + src + (two ? hd : 0));
    store_vec<V>(p.q_out + src, turn(x0));
    if (two)
      store_vec<V>(p.q_out + src + hd, turn(x1));
  } else {
    const int g = unit - qunits;
    const size_t src = (size_t)row * p.kv_stride + (size_t)g * hd + d;
    const size_t dst = (size_t)slot_of[local] * p.batch.slot_floats + (size_t)at * p.batch.pos_stride +
                       (size_t)g * p.batch.head_base + d;
    const Vec<V> k = load_vec<V>(p.k + src), v = load_vec<V>(p.v + src);
    store_vec<V>(p.key + dst, turn(k));
    store_vec<V>(p.value + dst, v);
  }
}

// ---- attention --------------------------------------------------------------------------------------------------------

struct RequestAttn {
  float *out;
  const float *q, *prefix_key, *prefix_value, *key, *value;
  RequestsDev batch;
  int n_heads, n_kv_heads, head_dim;
  float divisor; // sqrtf(head_dim)
  int *flags;
};

// Any shape: block (row, KV head), the positions (prefix, then own) in chunks of 64. Wave w scores positions w, w + 4,
// ..: lane l holds dimensions l, l + 64, .. of the K row and of the group's query vectors, the wave's sum is the dot. Per
// chunk and head the maximum, the exponentials and their sum join the running ones, and thread (share, dimension) rescales
// its value sums by exp(m_old - m_new) and adds its share of the chunk's positions; the shares meet in LDS at the end.
__global__ __launch_bounds__(kThreads) void attn_rows(RequestAttn p, int row0) {
  __shared__ float score[kMaxGroup][kChunk];
  __shared__ float run_max[kMaxGroup], run_sum[kMaxGroup], rescale[kMaxGroup];
  __shared__ float acc[kThreads * kMaxGroup]; // [share][head][head_dim], shares * head_dim <= 256
  __shared__ int mine[3];
  const int g = blockIdx.x % p.n_kv_heads, row = row0 + blockIdx.x / p.n_kv_heads;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  if (tid == 0)
    mine[0] = -1;
  __syncthreads();
  bool bad_batch = false, bad = false;
  for (int r = tid; r < p.batch.count; r += kThreads) {
    const Request q = request_at(p.batch, r, bad_batch);
    if (row >= q.first && row < q.first + q.rows) {
      mine[0] = r;
      mine[1] = q.length + row - q.first;
      mine[2] = q.slot;
    }
  }
  if (bad_batch && blockIdx.x == 0 && row0 == 0)
    p.flags[3] = 1;
  __syncthreads();
  if (mine[0] < 0)
    return; // the row belongs to no request
  const int positions = p.batch.prefix + mine[1] + 1, slot = mine[2];
  const int kv_mul = p.n_heads / p.n_kv_heads, hd = p.head_dim;
  const float *qrow = p.q + ((size_t)row * p.n_heads + (size_t)g * kv_mul) * hd;
  constexpr int kDims = kMaxHeadDim / kWave;
  float qv[kMaxGroup][kDims];
#pragma unroll
  for (int h = 0; h < kMaxGroup; h++)
#pragma unroll
    for (int e = 0; e < kDims; e++) {
      const int d = lane + e * kWave;
      qv[h][e] = h < kv_mul && d < hd ? qrow[(size_t)h * hd + d] : 0.0f;
    }
  if (tid < kv_mul)
    run_max[tid] = -FLT_MAX, run_sum[tid] = 0.0f;
  const size_t own = (size_t)slot * p.batch.slot_floats + (size_t)g * p.batch.head_base;
  const size_t far = (size_t)g * p.batch.prefix_head_base;
  auto row_at = [&](const float *prefix, const float *cache, int t) {
    return t < p.batch.prefix ? prefix + far + (size_t)t * p.batch.prefix_pos_stride
                              : cache + own + (size_t)(t - p.batch.prefix) * p.batch.pos_stride;
  };
  const int shares = kThreads / hd, share = tid / hd, d = tid % hd;
  float o[kMaxGroup];
#pragma unroll
  for (int h = 0; h < kMaxGroup; h++)
    o[h] = 0.0f;
  for (int t0 = 0; t0 < positions; t0 += kChunk) {
    const int n = min(kChunk, positions - t0);
    for (int t = wave; t < n; t += kThreads / kWave) {
      const float *krow = row_at(p.prefix_key, p.key, t0 + t);
      float kd[kDims];
#pragma unroll
      for (int e = 0; e < kDims; e++) {
        const int dd = lane + e * kWave;
        kd[e] = dd < hd ? krow[dd] : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < kMaxGroup; h++)
        if (h < kv_mul) {
          float dot = 0.0f;
#pragma unroll
          for (int e = 0; e < kDims; e++)
            dot = fmaf(qv[h][e], kd[e], dot);
          const float s = wave_sum(dot) / p.divisor;
          bad |= !isfinite(s);
          if (lane == 0)
            score[h][t] = s;
        }
    }
    __syncthreads();
    for (int h = wave; h < kv_mul; h += kThreads / kWave) {
      const float s = lane < n ? score[h][lane] : -FLT_MAX;
      const float m_old = run_max[h], m = fmaxf(m_old, wave_max(s));
      const float e = lane < n ? expf(s - m) : 0.0f;
      score[h][lane] = e;
      const float l = wave_sum(e);
      if (lane == 0) {
        const float alpha = expf(m_old - m);
        rescale[h] = alpha;
        run_max[h] = m;
        run_sum[h] = run_sum[h] * alpha + l;
      }
    }
    __syncthreads();
    if (share < shares) {
#pragma unroll
      for (int h = 0; h < kMaxGroup; h++)
        if (h < kv_mul)
          o[h] *= rescale[h];
      for (int t = share; t < n; t += shares) {
        const float v = row_at(p.prefix_value, p.value, t0 + t)[d];
#pragma unroll
        for (int h = 0; h < kMaxGroup; h++)
          if (h < kv_mul)
            o[h] = fmaf(score[h][t], v, o[h]);
      }
    }
    __syncthreads(); // the next chunk's scores overwrite this one's
  }
  if (bad && lane == 0)
    p.flags[1] = 1;
  if (share < shares) {
#pragma unroll
    for (int h = 0; h < kMaxGroup; h++)
      if (h < kv_mul)
        acc[((size_t)share * kv_mul + h) * hd + d] = o[h];
  }
  __syncthreads();
  float *dst = p.out + ((size_t)row * p.n_heads + (size_t)g * kv_mul) * hd;
  for (int i = tid; i < kv_mul * hd; i += kThreads) {
    float total = 0.0f;
    for (int s2 = 0; s2 < shares; s2++)
      total += acc[(size_t)s2 * kv_mul * hd + i];
    dst[i] = total / run_sum[i / hd];
  }
}

} // namespace

bool launch_rope_requests(const RopeRequestsJob &job, hipStream_t stream) {
  const uintptr_t all = (uintptr_t)job.q_out | (uintptr_t)job.q | (uintptr_t)job.k | (uintptr_t)job.v |
                        (uintptr_t)job.key | (uintptr_t)job.value;
  const bool vec4 = job.head_dim % 4 == 0 && job.q_stride % 4 == 0 && job.kv_stride % 4 == 0 && (all & 15) == 0;
  const int items = job.head_dim / (vec4 ? 4 : 2), per_block = kThreads / items;
  const int units = (job.n_heads + 1) / 2 + job.n_kv_heads;
  const long long blocks = ((long long)job.batch.rows + per_block - 1) / per_block * units;
  if (blocks > (1 << 23)) // a launch holds fewer than 2^32 threads
    return raise("llhip_rope_kv_store_requests: %d rows of %d heads are too many for one launch", job.batch.rows,
                 job.n_heads);
  const auto kernel = vec4 ? rope_requests<4> : rope_requests<2>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, job, device().error_flags);
  return launch_ok("rope_requests");
}

bool launch_attention_requests(const AttentionRequestsJob &job, hipStream_t stream) {
  RequestAttn p{};
  p.out = job.out;
  p.q = job.q;
  p.prefix_key = job.prefix_key;
  p.prefix_value = job.prefix_value;
  p.key = job.key;
  p.value = job.value;
  p.batch = job.batch;
  p.n_heads = job.n_heads;
  p.n_kv_heads = job.n_kv_heads;
  p.head_dim = job.head_dim;
  p.divisor = sqrtf((float)job.head_dim);
  p.flags = device().error_flags;
  const int most = (1 << 23) / job.n_kv_heads; // rows of a launch, which holds fewer than 2^32 threads
  for (int row0 = 0; row0 < job.batch.rows; row0 += most) {
    const int n = job.batch.rows - row0 < most ? job.batch.rows - row0 : most;
    hipLaunchKernelGGL(attn_rows, dim3((unsigned)n * (unsigned)job.n_kv_heads), dim3(kThreads), 0, stream, p, row0);
    if (job.batch.rows - row0 <= most)
      break;
  }
  return launch_ok("attn_rows");
}

} // namespace llhip
