// Low-rank adapters of many requests beside shared projections (gfx950): c = base + scale B (A x) per row, each row with
// the adapter that its request has.
//
//   lora_rows   any shape: one block per row and segment, A x kept in LDS.
#include "common.h"
#include "lanes.h"

namespace llhip {
namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kMaxRank = 256;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(uint16_t x) { return __uint_as_float((unsigned)x << 16); }

__device__ __forceinline__ float silu(float x) { return x * (1.0f / (1.0f + expf(-x))); }

__device__ __forceinline__ LoraSegmentDev pick(const LoraJob &p, int s) {
  return s == 0 ? p.seg[0] : s == 1 ? p.seg[1] : p.seg[2];
}

// Block (row, segment): wave w forms entries w, w + 4, .. of A x (and of A3 x), lane l over values l, l + 64, ..; then
// thread t columns t, t + 256, .. of B times them. A row without an adapter takes P = 0.
template <class T> __global__ __launch_bounds__(kThreads) void lora_rows(LoraJob p, int *flags) {
  __shared__ float low[2][kMaxRank];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const LoraSegmentDev s = pick(p, blockIdx.y);
  int id = p.adapter[row];
  if (id < -1 || id >= p.adapters) {
    flags[5] = 1;
    return;
  }
  const float *x = p.x + (size_t)row * p.ldx;
  const int parts = s.swiglu ? 2 : 1;
  if (id >= 0) {
    for (int i = wave; i < parts * s.rank; i += kThreads / kWave) {
      const int part = i / s.rank, j = i % s.rank;
      const T *a = (const T *)(part ? s.a3 : s.a) + ((size_t)id * s.rank + j) * p.k;
      float dot = 0.0f;
      for (int at = lane; at < p.k; at += kWave)
        dot = fmaf(value_of(a[at]), x[at], dot);
      dot = wave_sum(dot);
      if (lane == 0)
        low[part][j] = dot;
    }
  }
  __syncthreads();
  const float scale = id >= 0 && s.scale ? s.scale[id] : 1.0f;
  const size_t base = (size_t)row * s.ldc;
  auto product = [&](const void *b, int part, int n) {
    if (id < 0)
      return 0.0f;
    const T *w = (const T *)b + ((size_t)id * s.n + n) * s.rank;
    float sum = 0.0f;
    for (int j = 0; j < s.rank; j++)
      sum = fmaf(value_of(w[j]), low[part][j], sum);
    return scale * sum;
  };
  for (int n = tid; n < s.n; n += kThreads) {
    float y = s.base[base + n] + product(s.b, 0, n);
    if (s.swiglu)
      y = silu(y) * (s.base3[base + n] + product(s.b3, 1, n));
    s.c[base + n] = y;
  }
}

} // namespace

bool launch_lora(const LoraJob &job, hipStream_t stream) {
  if (job.m > (1 << 23))
    return raise("llhip_lora: %d rows are too many for one launch", job.m);
  const dim3 grid((unsigned)job.m, (unsigned)job.nseg);
  if (job.bf16)
    hipLaunchKernelGGL(lora_rows<uint16_t>, grid, dim3(kThreads), 0, stream, job, device().error_flags);
  else
    hipLaunchKernelGGL(lora_rows<float>, grid, dim3(kThreads), 0, stream, job, device().error_flags);
  return launch_ok("lora_rows");
}

} // namespace llhip
