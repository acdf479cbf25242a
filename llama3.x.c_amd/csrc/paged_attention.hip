// Attention over a cache in pages (gfx950).
//
//   attn_paged_rows   any shape, one row and KV head a block.
#include <cfloat>

#include "paged_device.h"

#include "lanes.h"

namespace llhip {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kChunk = 64;
constexpr int kMaxGroup = 16;
constexpr int kMaxHeadDim = 256;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

__device__ __forceinline__ float value(const float *p) { return *p; }
__device__ __forceinline__ float value(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }

struct PagedAttn {
  AttentionPagedJob job;
  float divisor; // sqrtf(head_dim)
  int *flags;
};

// Any shape: block (row, KV head), the positions in chunks of 64, whose places in the caches are looked up together. Wave
// w scores positions w, w + 4, ..: lane l holds dimensions l, l + 64, .. of the K row and of the group's query vectors, the
// wave's sum is the dot. Per chunk and head the maximum, the exponentials and their sum join the running ones, and thread
// (share, dimension) rescales its value sums by exp(m_old - m_new) and adds its share of the chunk's positions; the shares
// meet in LDS at the end. Positions behind the row's own are never read.
template <typename T> __global__ __launch_bounds__(kThreads) void attn_paged_rows(PagedAttn p, int row0) {
  __shared__ float score[kMaxGroup][kChunk];
  __shared__ float run_max[kMaxGroup], run_sum[kMaxGroup], rescale[kMaxGroup];
  __shared__ float acc[kThreads * kMaxGroup]; // [share][head][head_dim], shares * head_dim <= 256
  __shared__ size_t place[kChunk];
  __shared__ int mine[2];
  const AttentionPagedJob &job = p.job;
  const PagedDev &b = job.batch;
  const int g = blockIdx.x % job.n_kv_heads, row = row0 + blockIdx.x / job.n_kv_heads;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  if (tid == 0)
    mine[0] = -1;
  __syncthreads();
  bool bad_batch = false, bad = false;
  for (int r = tid; r < b.count; r += kThreads) {
    const PagedRequest q = paged_request(b, r, bad_batch);
    if (row >= q.first && row < q.first + q.rows) {
      mine[0] = r;
      mine[1] = q.length + row - q.first;
    }
  }
  if (bad_batch && blockIdx.x == 0 && row0 == 0)
    p.flags[3] = 1;
  __syncthreads();
  const int request = mine[0];
  if (request < 0)
    return; // the row belongs to no request
  const int positions = mine[1] + 1;
  const int kv_mul = job.n_heads / job.n_kv_heads, hd = job.head_dim;
  const float *qrow = job.q + (size_t)row * job.q_stride + (size_t)g * kv_mul * hd;
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
  const T *keys = (const T *)job.key + (size_t)g * b.head_base, *values = (const T *)job.value + (size_t)g * b.head_base;
  const int shares = kThreads / hd, share = tid / hd, d = tid % hd;
  float o[kMaxGroup];
#pragma unroll
  for (int h = 0; h < kMaxGroup; h++)
    o[h] = 0.0f;
  for (int t0 = 0; t0 < positions; t0 += kChunk) {
    const int n = min(kChunk, positions - t0);
    if (tid < n) {
      const int t = t0 + tid, page = page_of(b, request, t / b.page_size);
      if (page < 0)
        p.flags[8] = 1;
      place[tid] = (size_t)max(page, 0) * b.page_values + (size_t)(t % b.page_size) * b.pos_stride;
    }
    __syncthreads();
    for (int t = wave; t < n; t += kThreads / kWave) {
      const T *krow = keys + place[t];
      float kd[kDims];
#pragma unroll
      for (int e = 0; e < kDims; e++) {
        const int dd = lane + e * kWave;
        kd[e] = dd < hd ? value(krow + dd) : 0.0f;
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
        const float v = value(values + place[t] + d);
#pragma unroll
        for (int h = 0; h < kMaxGroup; h++)
          if (h < kv_mul)
            o[h] = fmaf(score[h][t], v, o[h]);
      }
    }
    __syncthreads(); // the next chunk's scores and places overwrite this one's
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
  float *dst = job.out + ((size_t)row * job.n_heads + (size_t)g * kv_mul) * hd;
  for (int i = tid; i < kv_mul * hd; i += kThreads) {
    float total = 0.0f;
    for (int s2 = 0; s2 < shares; s2++)
      total += acc[(size_t)s2 * kv_mul * hd + i];
    dst[i] = total / run_sum[i / hd];
  }
}

} // namespace

size_t attention_paged_workspace(const AttentionPagedJob &) { return 0; }

bool launch_attention_paged(const AttentionPagedJob &job, void *, hipStream_t stream) {
  const PagedAttn p{job, sqrtf((float)job.head_dim), device().error_flags};
  const int most = (1 << 23) / job.n_kv_heads; // a launch holds fewer than 2^32 threads
  for (int row0 = 0; row0 < job.batch.rows; row0 += most) {
    const int n = job.batch.rows - row0 < most ? job.batch.rows - row0 : most;
    const auto kernel = job.batch.bf16 ? attn_paged_rows<uint16_t> : attn_paged_rows<float>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n * (unsigned)job.n_kv_heads), dim3(kThreads), 0, stream, p, row0);
    if (!launch_ok("attn_paged_rows"))
      return false;
  }
  return true;
}

} // namespace llhip
