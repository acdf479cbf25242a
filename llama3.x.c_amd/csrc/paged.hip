// A cache in pages (gfx950): the rows' keys and values into their requests' pages, with the norms of each head and RoPE on
// the way.
//
//   append_paged   block: some rows' two q heads or one KV head; a group of lanes per row and head.
#include "paged_device.h"

#include "lanes.h"

namespace llhip {
namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

// V = 4 or 2 values of a head: a lane's share of it, or one of two.
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
// Rounded to the nearest BF16 value, ties to even, as bf16_from_f32 rounds.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const v2f x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2bf));
}
template <int V> __device__ __forceinline__ void store_vec(uint16_t *p, const Vec<V> &x) {
  if constexpr (V == 4) {
    *reinterpret_cast<uint2 *>(p) = uint2{bf16_pair(x.v[0], x.v[1]), bf16_pair(x.v[2], x.v[3])};
  } else { // a row of an even number of values, the pages on 2-byte boundaries at least
    const uint32_t both = bf16_pair(x.v[0], x.v[1]);
    p[0] = (uint16_t)both, p[1] = (uint16_t)(both >> 16);
  }
}

__device__ __forceinline__ void rotate(float &a, float &b, float c, float s) {
#pragma clang fp contract(off) // the products rounded before the sum, as k_rope_apply computes them
  const float x = a, y = b;
  a = x * c - y * s;
  b = x * s + y * c;
}

// Block (row group, unit): unit u takes q heads 2u and 2u + 1 of the group's rows, or one KV head's k and v. `lanes` lanes
// (a power of two, so that a head's sum of squares is reduced within the wave) hold a row's head, V values each, or twice V
// where V = 2 and head_dim > 128. V = 4 for 16-byte aligned rows of head_dim a multiple of 4, else 2. The block finds its
// rows' requests by looking through all of them, 256 at a time: one load each where a search per row would wait for its
// log2(count) loads in turn. The last block stores nothing and looks for two requests whose first rows go to one page, in
// a table in LDS: beside the others it costs them no time.
template <int V, typename T>
__global__ __launch_bounds__(kThreads) void append_paged(AppendPagedJob p, int lanes, int *flags) {
  constexpr int kTable = 2 * kMaxRequests, kParts = V == 2 ? 2 : 1;
  __shared__ int request_of[kThreads], position_of[kThreads];
  __shared__ int table[kTable];
  const int per_block = kThreads / lanes, tid = threadIdx.x;
  const int qunits = (p.n_heads + 1) / 2, units = qunits + p.n_kv_heads;
  if (blockIdx.x == gridDim.x - 1) {
    for (int i = tid; i < kTable; i += kThreads)
      table[i] = -1;
    __syncthreads();
    bool bad = false, twice = false;
    for (int r = tid; r < p.batch.count; r += kThreads) {
      const PagedRequest q = paged_request(p.batch, r, bad);
      const int page = q.rows ? page_of(p.batch, r, q.length / p.batch.page_size) : -1;
      if (page < 0)
        continue;
      int at = (int)((unsigned)page * 2654435761u % kTable); // at most 1024 entries in 2048 places: a free one is found
      while (true) {
        const int seen = atomicCAS(&table[at], -1, page);
        if (seen == -1)
          break;
        if (seen == page) {
          twice = true;
          break;
        }
        at = (at + 1) % kTable;
      }
    }
    if (bad)
      flags[3] = 1;
    if (twice)
      flags[9] = 1;
    return;
  }
  const int unit = blockIdx.x % units, r0 = blockIdx.x / units * per_block;
  for (int i = tid; i < per_block; i += kThreads)
    request_of[i] = -1;
  __syncthreads();
  bool bad = false;
  for (int r = tid; r < p.batch.count; r += kThreads) {
    const PagedRequest q = paged_request(p.batch, r, bad);
    const int a = max(q.first, r0), b = min(q.first + q.rows, r0 + per_block);
    for (int i = a; i < b; i++) {
      request_of[i - r0] = r;
      position_of[i - r0] = q.length + i - q.first;
    }
  }
  __syncthreads();
  const int local = tid / lanes, lane = tid % lanes, hd = p.head_dim;
  const int request = request_of[local];
  if (request < 0)
    return; // the whole group of lanes
  const int row = r0 + local, at = position_of[local];
  const float *t = p.table + (size_t)at * 2 * hd;
  float c[kParts][V / 2], s[kParts][V / 2];
  int d[kParts];
  bool has[kParts];
#pragma unroll
  for (int part = 0; part < kParts; part++) {
    d[part] = (part * lanes + lane) * V;
    has[part] = d[part] < hd;
    if (!has[part])
      d[part] = 0; // loads what another lane uses, and stores nothing
#pragma unroll
    for (int i = 0; i < V / 2; i++)
      c[part][i] = t[d[part] + 2 * i], s[part][i] = t[hd + d[part] + 2 * i + 1];
  }
  struct Head {
    Vec<V> part[kParts];
  };
  auto load = [&](const float *src) {
    Head x;
#pragma unroll
    for (int part = 0; part < kParts; part++)
      x.part[part] = load_vec<V>(src + d[part]);
    return x;
  };
  // the head's norm as k_rmsnorm computes it, then the rotation
  auto turn = [&](Head &x, const float *norm) {
    if (norm) {
      float sum = 0.0f;
#pragma unroll
      for (int part = 0; part < kParts; part++)
#pragma unroll
        for (int i = 0; i < V; i++)
          sum = has[part] ? fmaf(x.part[part].v[i], x.part[part].v[i], sum) : sum;
      sum = group_reduce_add(sum, lanes);
      const float ss = 1.0f / sqrtf(sum / (float)hd + p.epsilon);
#pragma unroll
      for (int part = 0; part < kParts; part++) {
        const Vec<V> w = load_vec<V>(norm + d[part]);
#pragma unroll
        for (int i = 0; i < V; i++)
          x.part[part].v[i] = w.v[i] * (ss * x.part[part].v[i]);
      }
    }
#pragma unroll
    for (int part = 0; part < kParts; part++)
#pragma unroll
      for (int i = 0; i < V / 2; i++)
        rotate(x.part[part].v[2 * i], x.part[part].v[2 * i + 1], c[part][i], s[part][i]);
  };
  auto store = [&](auto *dst, const Head &x) {
#pragma unroll
    for (int part = 0; part < kParts; part++)
      if (has[part])
        store_vec<V>(dst + d[part], x.part[part]);
  };
  if (unit < qunits) {
    const size_t src = (size_t)row * p.q_stride + (size_t)(2 * unit) * hd;
    const size_t dst = (size_t)row * p.q_out_stride + (size_t)(2 * unit) * hd;
    const bool two = 2 * unit + 1 < p.n_heads;
    Head x0 = load(p.q + src), x1 = load(p.q + src + (two ? hd : 0));
    turn(x0, p.q_norm);
    turn(x1, p.q_norm);
    store(p.q_out + dst, x0);
    if (two)
      store(p.q_out + dst + hd, x1);
  } else {
    const int g = unit - qunits;
    const size_t src = (size_t)row * p.kv_stride + (size_t)g * hd;
    Head k = load(p.k + src);
    const Head v = load(p.v + src);
    const int page = page_of(p.batch, request, at / p.batch.page_size);
    turn(k, p.k_norm);
    if (page < 0) {
      if (lane == 0)
        flags[8] = 1;
      return;
    }
    const size_t dst = (size_t)page * p.batch.page_values + (size_t)(at % p.batch.page_size) * p.batch.pos_stride +
                       (size_t)g * p.batch.head_base;
    store((T *)p.key + dst, k);
    store((T *)p.value + dst, v);
  }
}

} // namespace

bool launch_append_paged(const AppendPagedJob &job, hipStream_t stream) {
  const uintptr_t all = (uintptr_t)job.q_out | (uintptr_t)job.q | (uintptr_t)job.k | (uintptr_t)job.v |
                        (uintptr_t)job.key | (uintptr_t)job.value | (uintptr_t)job.q_norm | (uintptr_t)job.k_norm;
  const bool vec4 = job.head_dim % 4 == 0 && job.q_stride % 4 == 0 && job.q_out_stride % 4 == 0 &&
                    job.kv_stride % 4 == 0 && (all & 15) == 0;
  int lanes = 1;
  while (lanes < kWave && lanes * (vec4 ? 4 : 2) < job.head_dim)
    lanes *= 2;
  const int per_block = kThreads / lanes, units = (job.n_heads + 1) / 2 + job.n_kv_heads;
  const long long blocks = ((long long)job.batch.rows + per_block - 1) / per_block * units + 1;
  if (blocks > (1 << 23)) // a launch holds fewer than 2^32 threads
    return raise("llhip_rope_kv_append_paged: %d rows of %d heads are too many for one launch", job.batch.rows,
                 job.n_heads);
  const auto kernel = job.batch.bf16 ? (vec4 ? append_paged<4, uint16_t> : append_paged<2, uint16_t>)
                                     : (vec4 ? append_paged<4, float> : append_paged<2, float>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, job, lanes, device().error_flags);
  return launch_ok("append_paged");
}

} // namespace llhip
