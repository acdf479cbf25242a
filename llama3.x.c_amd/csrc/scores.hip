// Log probabilities of given tokens, the entropies and the likeliest tokens of rows of logits (gfx950).
//
//   score_stats   a wave each chunk of 1024 tokens of a row: the chunk's maximum, the sums of exp z and of z exp z relative to
//                 it, and, where alternatives are asked for, the maximum of each group of 64 tokens. One read. HBM-bound.
//   score_rows    block (row): the chunks joined; the alternatives from the groups that can hold them.
//
// The k likeliest tokens lie in the k groups whose maxima are largest (of equal ones the lower group's): any other group has
// k groups before it, each with a token at least as large, and lower where it is as large. So the second kernel reads
// 64 k logits and not the row.
#include <cfloat>

#include "common.h"
#include "lanes.h"
#include "llama_hip_requests.h"

namespace llhip {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 1024; // tokens of a wave, 16 a lane
constexpr int kGroup = 64;   // tokens of a maximum: those of 16 lanes' float4
constexpr int kGroups = kChunk / kGroup;
constexpr int kRankList = 512; // candidates that are ranked each against each

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

// A chunk of a row, relative to its maximum `top`: how many logits equal it (each of them exp z = 1), and the sums over the
// others of exp2(y) and of y exp2(y), y = (l - top) log2(e) / T. The ones apart, a peaked row's small rest keeps its bits:
// log S = log1p(rest) and the entropy near 0. top +infinity: the chunk holds a NaN or +infinity; -infinity: all masked.
struct Stat {
  float top;
  int ones;
  float rest, weighted;
};

struct Score {
  ScoreJob job;
  Stat *stats;   // [row][chunk]
  float *maxima; // [row][16 chunks]
  int chunks;
  float scale2; // log2(e) / T
  int *flags;
  bool vec4;
};

__global__ __launch_bounds__(kThreads) void score_stats(Score p, int row0) {
  const int row = row0 + blockIdx.y, lane = threadIdx.x % kWave, chunk = blockIdx.x * kWaves + threadIdx.x / kWave;
  const float *src = p.job.logits + (size_t)row * p.job.ld;
  const int i0 = chunk * kChunk, n = min(kChunk, p.job.vocab - i0);
  if (n <= 0)
    return;
  auto place = [&](int j) { return 4 * (lane + j / 4 * kWave) + j % 4; }; // of x[j]
  float x[16];
  if (p.vec4 && n == kChunk) { // uniform: no branch a load
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float4 v = *reinterpret_cast<const float4 *>(src + i0 + 4 * (lane + j * kWave));
      x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      x[j] = src[i0 + min(place(j), n - 1)];
#pragma unroll
    for (int j = 0; j < 16; j++)
      x[j] = place(j) < n ? x[j] : -INFINITY;
  }
  float four[4];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 16; j++)
    bad |= !(x[j] < INFINITY);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    four[j] = fmaxf(fmaxf(x[4 * j], x[4 * j + 1]), fmaxf(x[4 * j + 2], x[4 * j + 3]));
    four[j] = group_reduce_max(four[j], 16);
  }
  if (p.maxima) { // group 4 j + lane / 16, by lane 16 (lane / 16) + j
    const int j = lane % 16;
    const float mine = j == 0 ? four[0] : j == 1 ? four[1] : j == 2 ? four[2] : four[3];
    if (j < 4)
      p.maxima[((size_t)row * p.chunks + chunk) * kGroups + 4 * j + lane / 16] = mine;
  }
  float top = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3]));
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  bad = __any(bad);
  int ones = 0;
  float rest = 0.0f, weighted = 0.0f;
  if (!bad && top > -INFINITY) {
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const float y = fmaxf((x[j] - top) * p.scale2, -1e4f); // exp2 of less is 0, and 0 times it must be too
      const float e = __builtin_amdgcn_exp2f(y);
      const bool one = x[j] == top;
      ones += one;
      rest += one ? 0.0f : e;
      weighted = fmaf(y, e, weighted);
    }
    ones = group_reduce_add(ones, kWave);
    rest = wave_sum(rest);
    weighted = wave_sum(weighted);
  }
  if (lane == 0)
    p.stats[(size_t)row * p.chunks + chunk] = Stat{bad ? INFINITY : top, ones, rest, weighted};
}

__device__ __forceinline__ double wave_add(double v) {
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o);
  return v;
}

// Keys in the order of alternatives: the larger value first, of equal ones the lower place. 0 is below all.
__device__ __forceinline__ uint64_t key_of(float x, int place) {
  x += 0.0f; // -0 counts as 0
  const uint32_t b = __float_as_uint(x);
  return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~place;
}
__device__ __forceinline__ int place_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// The k largest of n different keys in LDS, in order, to best[0 .. min(n, k) - 1]; by the whole block, which has written
// the list before a barrier.
__device__ void largest(const uint64_t *list, int n, int k, uint64_t *best, uint64_t *scratch) {
  const int tid = threadIdx.x;
  if (n <= kRankList) { // each key's rank
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t mine = list[i];
      int before = 0;
      for (int j = 0; j < n; j++)
        before += list[j] > mine;
      if (before < k)
        best[before] = mine;
    }
    __syncthreads();
    return;
  }
  uint64_t last = ~0ull; // one after the other: many equal logits
  for (int i = 0; i < k; i++) {
    uint64_t mine = 0;
    for (int j = tid; j < n; j += kThreads)
      mine = list[j] < last && list[j] > mine ? list[j] : mine;
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)mine, o);
      mine = other > mine ? other : mine;
    }
    if (tid % kWave == 0)
      scratch[tid / kWave] = mine;
    __syncthreads();
    for (int w = 0; w < kWaves; w++)
      mine = scratch[w] > mine ? scratch[w] : mine;
    last = mine;
    if (tid == 0)
      best[i] = mine;
    __syncthreads();
  }
}

// What is in LDS: `list` keys of `capacity` groups or 64 top tokens.
__global__ __launch_bounds__(kThreads) void score_rows(Score p, int capacity) {
  extern __shared__ uint64_t list[];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves][2];
  __shared__ int counts[kWaves];
  __shared__ uint64_t mine_of[kThreads], best[LLHIP_MAX_TOP], scratch[kWaves];
  __shared__ uint64_t threshold;
  __shared__ int found;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, top = p.job.top;
  const float *logits = p.job.logits + (size_t)row * p.job.ld;
  const Stat *stats = p.stats + (size_t)row * p.chunks;
  const int token = p.job.tokens ? p.job.tokens[row] : -1;
  const bool inside = token >= 0 && token < p.job.vocab;
  const float given = inside ? logits[token] : 0.0f;
  const Stat first = tid < p.chunks ? stats[tid] : Stat{-INFINITY, 0, 0.0f, 0.0f};
  float most = first.top;
  for (int c = tid + kThreads; c < p.chunks; c += kThreads)
    most = fmaxf(most, stats[c].top);
  most = wave_max(most);
  if (lane == 0)
    tops[wave] = most;
  __syncthreads();
  for (int w = 0; w < kWaves; w++)
    most = fmaxf(most, tops[w]);
  const bool decides = most > -INFINITY && most < INFINITY;
  if (!decides) { // uniform
    if (tid == 0) {
      p.flags[10] = 1;
      if (p.job.logprob)
        p.job.logprob[row] = NAN;
      if (p.job.entropy)
        p.job.entropy[row] = NAN;
    }
    for (int i = tid; i < top; i += kThreads)
      p.job.top_token[(size_t)row * top + i] = -1, p.job.top_logprob[(size_t)row * top + i] = NAN;
    return;
  }
  // the row's ones, the sum of the others and the weighted sum, in units of the row's maximum
  int ones = 0;
  double rest = 0.0, weighted = 0.0;
  auto join = [&](const Stat &s) {
    const float y = fmaxf((s.top - most) * p.scale2, -1e4f);
    const bool top_chunk = s.top == most;
    const double e = (double)__builtin_amdgcn_exp2f(y), sum = (double)s.ones + (double)s.rest;
    ones += top_chunk ? s.ones : 0;
    rest += top_chunk ? (double)s.rest : e * sum;
    weighted += e * ((double)s.weighted + (double)y * sum);
  };
  join(first);
  for (int c = tid + kThreads; c < p.chunks; c += kThreads)
    join(stats[c]);
  ones = group_reduce_add(ones, kWave);
  rest = wave_add(rest);
  weighted = wave_add(weighted);
  if (lane == 0)
    counts[wave] = ones, sums[wave][0] = rest, sums[wave][1] = weighted;
  __syncthreads();
  ones = 0;
  rest = weighted = 0.0;
  for (int w = 0; w < kWaves; w++)
    ones += counts[w], rest += sums[w][0], weighted += sums[w][1];
  rest += (double)(ones - 1); // S - 1
  const double log_sum = log1p(rest), temperature = (double)p.job.temperature;
  auto logprob = [&](float l) { return (float)(((double)l - (double)most) / temperature - log_sum); };
  if (tid == 0) {
    if (p.job.logprob) {
      p.job.logprob[row] = inside ? logprob(given) : token == -1 ? 0.0f : NAN;
      if (!inside && token != -1)
        p.flags[11] = 1;
    }
    if (p.job.entropy)
      p.job.entropy[row] = (float)(log_sum - weighted * 0.6931471805599453 / (1.0 + rest));
  }
  if (top == 0)
    return;
  // the largest group maximum of each thread; the top-th of them is a bound that `top` groups reach
  const float *maxima = p.maxima + (size_t)row * p.chunks * kGroups;
  const int groups = (p.job.vocab + kGroup - 1) / kGroup;
  uint64_t mine = 0;
  for (int g = tid; g < groups; g += kThreads) {
    const uint64_t key = maxima[g] > -INFINITY ? key_of(maxima[g], g) : 0;
    mine = key > mine ? key : mine;
  }
  mine_of[tid] = mine;
  if (tid == 0)
    found = 0, threshold = 1; // 1: every key there is
  for (int i = tid; i < top; i += kThreads)
    best[i] = 0;
  __syncthreads();
  int before = 0;
  for (int j = 0; j < kThreads; j++)
    before += mine_of[j] > mine;
  if (mine && before == top - 1)
    threshold = mine;
  __syncthreads();
  const uint64_t least = threshold;
  for (int g = tid; g < groups; g += kThreads) {
    const uint64_t key = maxima[g] > -INFINITY ? key_of(maxima[g], g) : 0;
    if (key >= least) { // of at most `top` threads' groups: `capacity` keys
      const int at = atomicAdd(&found, 1);
      if (at < capacity)
        list[at] = key;
    }
  }
  __syncthreads();
  const int many = min(found, capacity);
  largest(list, many, top, best, scratch);
  // their tokens that reach the last one's maximum, then the largest of those
  const int held = min(many, top);
  const uint64_t weakest = best[held - 1];
  const float reach = many < top ? -INFINITY : value_of(weakest);
  int group = 0;
  __syncthreads(); // every thread has read `found`
  if (tid == 0)
    found = 0;
  __syncthreads();
  for (int i = wave; i < held; i += kWaves) {
    group = place_of(best[i]);
    const int at = group * kGroup + lane;
    const float x = at < p.job.vocab ? logits[at] : -INFINITY;
    if (x >= reach && x > -INFINITY)
      list[atomicAdd(&found, 1)] = key_of(x, at);
  }
  __syncthreads();
  const int tokens = found;
  __syncthreads(); // best is read
  largest(list, tokens, top, best, scratch);
  for (int i = tid; i < top; i += kThreads) {
    const bool there = i < tokens;
    p.job.top_token[(size_t)row * top + i] = there ? place_of(best[i]) : -1;
    p.job.top_logprob[(size_t)row * top + i] = there ? logprob(value_of(best[i])) : -INFINITY;
  }
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

} // namespace

size_t scores_workspace(const ScoreJob &job) {
  const size_t chunks = (size_t)job.rows * chunks_of(job.vocab);
  return chunks * sizeof(Stat) + (job.top ? chunks * kGroups * sizeof(float) : 0);
}

bool launch_scores(const ScoreJob &job, void *workspace, hipStream_t stream) {
  Score p{};
  p.job = job;
  p.chunks = chunks_of(job.vocab);
  p.stats = (Stat *)workspace;
  p.maxima = job.top ? (float *)(p.stats + (size_t)job.rows * p.chunks) : nullptr;
  const double scale2 = 1.4426950408889634 / (double)job.temperature;
  p.scale2 = scale2 < 1e38 ? (float)scale2 : 1e38f; // finite: a difference of 0 stays 0
  p.flags = device().error_flags;
  p.vec4 = job.ld % 4 == 0 && ((uintptr_t)job.logits & 15) == 0;
  const int most = 32768; // rows of a launch
  for (int row0 = 0; row0 < job.rows; row0 += most) {
    const dim3 grid((unsigned)((p.chunks + kWaves - 1) / kWaves),
                    (unsigned)(job.rows - row0 < most ? job.rows - row0 : most));
    hipLaunchKernelGGL(score_stats, grid, dim3(kThreads), 0, stream, p, row0);
    if (!launch_ok("score_stats"))
      return false;
  }
  // a thread's groups of at most `top` threads, or 64 tokens of `top` groups
  const int groups = p.chunks * kGroups, capacity = job.top * ((groups + kThreads - 1) / kThreads);
  const int keys = capacity > job.top * kGroup ? capacity : job.top * kGroup;
  static const hipError_t room = // 4 Mi tokens with 32 alternatives take 64 KB beside the rest
      hipFuncSetAttribute((const void *)score_rows, hipFuncAttributeMaxDynamicSharedMemorySize, 64 << 10);
  if (room != hipSuccess)
    return raise("score_rows: %s", hipGetErrorString(room));
  hipLaunchKernelGGL(score_rows, dim3((unsigned)job.rows), dim3(kThreads), (size_t)keys * sizeof(uint64_t), stream, p,
                     capacity);
  return launch_ok("score_rows");
}

} // namespace llhip
