// Many requests on one model (gfx950): RoPE and cache rows at each request's own position.
//
//   rope_requests   one thread per V dimensions of a row's two q heads or of one KV head.
#include "requests_device.h"

namespace llhip {
namespace {

constexpr int kThreads = 256;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
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

} // namespace llhip
