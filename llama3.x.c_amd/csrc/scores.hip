// Log probabilities of given tokens, the entropies and the likeliest tokens of rows of logits (gfx950).
//
//   score_stats   a wave each chunk of 1024 tokens of a row: the chunk's maximum, the sums of exp z and of z exp z relative to
//                 it, and, where alternatives are asked for, the maximum of each group of 64 tokens. One read. HBM-bound.
//   score_rows    block (row): the chunks joined; the alternatives from the groups that can hold them.
//   score_few     both in one launch, for few rows: the last of a row's blocks to arrive joins its chunks.
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
constexpr int kPer = 16;       // maxima of a thread of score_rows, at most: rows of more than 4096 groups keep their chunks'
constexpr int kRankList = 512; // candidates that are ranked each against each
// Rows of score_few, at most: where the two forms meet over 128256 tokens. In us, one launch and two: 8 rows 6.0 and 8.1 without
// alternatives, 11.8 and 12.4 with 20; 16 rows 6.8 and 8.0, 13.0 and 13.2; 24 rows 7.6 and 8.5, 15.2 and 14.2; 64 rows 12.3 and
// 11.5, 26 and 18. (Over 32000 tokens they meet at 64 rows, 0.3 to 0.5 apart up to there.)
constexpr int kFewRows = 16;

// How many of a row's blocks have stored their chunks: zero between launches, as the last to arrive sets it back. Each in a
// cache line of its own: additions to one line wait for each other (64 rows: 12 us instead of 19).
constexpr int kLine = 32;
__device__ unsigned score_arrivals[kFewRows * kLine];

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
  float *maxima; // [row][maxima of a row], or null
  int chunks;
  int count; // maxima of a row: its groups', or its chunks'
  float scale2; // log2(e) / T
  int *flags;
  bool vec4;
};

// What one block stores and another of the same launch reads passes the XCDs' own L2s: stores of agent scope write through,
// loads of agent scope read what they wrote.
template <bool AGENT> __device__ __forceinline__ void put(float *p, float x) {
  if constexpr (AGENT)
    __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    *p = x;
}
template <bool AGENT> __device__ __forceinline__ float get(const float *p) {
  if constexpr (AGENT)
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    return *p;
}
struct Halves {
  unsigned long long lo, hi;
};
template <bool AGENT> __device__ __forceinline__ void put(Stat *p, const Stat &x) {
  if constexpr (AGENT) {
    const Halves h = __builtin_bit_cast(Halves, x);
    __hip_atomic_store((unsigned long long *)p, h.lo, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((unsigned long long *)p + 1, h.hi, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
    *p = x;
  }
}
template <bool AGENT> __device__ __forceinline__ Stat get(const Stat *p) {
  if constexpr (AGENT)
    return __builtin_bit_cast(Stat, Halves{__hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                                           __hip_atomic_load((const unsigned long long *)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)});
  else
    return *p;
}

// One chunk of a row, by a wave.
template <bool AGENT> __device__ __forceinline__ void score_chunk(const Score &p, int row, int chunk) {
  const int lane = threadIdx.x % kWave;
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
  if (p.maxima && p.count != p.chunks) { // group 4 j + lane / 16, by lane 16 (lane / 16) + j
    const int j = lane % 16, group = chunk * kGroups + 4 * j + lane / 16;
    const float mine = j == 0 ? four[0] : j == 1 ? four[1] : j == 2 ? four[2] : four[3];
    if (j < 4 && group < p.count)
      put<AGENT>(&p.maxima[(size_t)row * p.count + group], mine);
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
  if (lane == 0) {
    put<AGENT>(&p.stats[(size_t)row * p.chunks + chunk], Stat{bad ? INFINITY : top, ones, rest, weighted});
    if (p.maxima && p.count == p.chunks)
      put<AGENT>(&p.maxima[(size_t)row * p.count + chunk], top);
  }
}

__global__ __launch_bounds__(kThreads) void score_stats(Score p, int row0) {
  score_chunk<false>(p, row0 + blockIdx.y, blockIdx.x * kWaves + threadIdx.x / kWave);
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

__device__ __forceinline__ uint64_t key_max(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The k largest of n different keys in LDS to take(place among them, key); by the whole block, which has written the list
// before a barrier.
template <class Take> __device__ __forceinline__ void largest(const uint64_t *list, int n, int k, uint64_t *scratch, Take take) {
  const int tid = threadIdx.x;
  if (n <= kRankList) { // each key's rank
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t mine = list[i];
      int before = 0;
#pragma unroll 8
      for (int j = 0; j < n; j++)
        before += list[j] > mine;
      if (before < k)
        take(before, mine);
    }
    return;
  }
  uint64_t last = ~0ull; // one after the other: many equal logits
  for (int i = 0; i < k; i++) {
    uint64_t mine = 0;
    for (int j = tid; j < n; j += kThreads)
      mine = list[j] < last ? key_max(list[j], mine) : mine;
    for (int o = 32; o > 0; o >>= 1)
      mine = key_max(mine, __shfl_xor((unsigned long long)mine, o));
    __syncthreads(); // scratch is read
    if (tid % kWave == 0)
      scratch[tid / kWave] = mine;
    __syncthreads();
    for (int w = 0; w < kWaves; w++)
      mine = key_max(mine, scratch[w]);
    last = mine;
    if (tid == 0)
      take(i, mine);
  }
}

// The k-th largest of the wave's keys, or 1 (below every key) where fewer are not 0.
__device__ __forceinline__ uint64_t kth_of_wave(uint64_t mine, int k) {
  int before = 0;
  const int lo = (int)(uint32_t)mine, hi = (int)(uint32_t)(mine >> 32);
#pragma unroll
  for (int j = 0; j < kWave; j++) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane(lo, j);
    before += other > mine;
  }
  const unsigned long long is = __ballot(mine != 0 && before == k - 1);
  if (!is)
    return 1;
  const int at = __builtin_ctzll(is);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, at) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, at);
}

// A row's chunks joined, by a block. LDS holds `list` keys: those of a thread's maxima of `top` lanes a wave, 16 of each of `top` chunks, 64 of each of `top`
// groups, whichever are more.
template <bool AGENT> __device__ __forceinline__ void score_row(const Score &p, int row, uint64_t *list) {
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves][2];
  __shared__ int counts[kWaves];
  __shared__ uint64_t thresholds[kWaves], best[LLHIP_MAX_TOP], scratch[kWaves];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, top = p.job.top;
  const float *logits = p.job.logits + (size_t)row * p.job.ld;
  const Stat *stats = p.stats + (size_t)row * p.chunks;
  // what can be loaded at once is
  const int token = p.job.tokens ? p.job.tokens[row] : -1;
  const Stat first = tid < p.chunks ? get<AGENT>(&stats[tid]) : Stat{-INFINITY, 0, 0.0f, 0.0f};
  float maxima[kPer];
  if (top) {
    const float *src = p.maxima + (size_t)row * p.count;
#pragma unroll
    for (int j = 0; j < kPer; j++)
      maxima[j] = tid + j * kThreads < p.count ? get<AGENT>(&src[tid + j * kThreads]) : -INFINITY;
  }
  const bool inside = token >= 0 && token < p.job.vocab;
  const float given = inside ? logits[token] : 0.0f;
  if (tid < 3)
    found[tid] = 0;
  float most = first.top;
  for (int c = tid + kThreads; c < p.chunks; c += kThreads)
    most = fmaxf(most, get<AGENT>(&stats[c].top));
  most = wave_max(most);
  if (lane == 0)
    tops[wave] = most;
  auto key_at = [&](int j) { return maxima[j] > -INFINITY ? key_of(maxima[j], tid + j * kThreads) : 0; };
  if (top) { // the top-th of a wave's lanes' largest: a bound that `top` maxima reach
    uint64_t mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++)
      mine = key_max(mine, key_at(j));
    const uint64_t kth = kth_of_wave(mine, top);
    if (lane == 0)
      thresholds[wave] = kth;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; w++)
    most = fmaxf(most, tops[w]);
  if (!(most > -INFINITY && most < INFINITY)) { // uniform
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
  if (top) {
    uint64_t least = thresholds[0];
    for (int w = 1; w < kWaves; w++)
      least = key_max(least, thresholds[w]);
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const uint64_t key = key_at(j);
      if (key >= least)
        list[atomicAdd(&found[0], 1)] = key;
    }
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
    join(get<AGENT>(&stats[c]));
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
  int many = 0, held = 0;
  if (top) {
    many = found[0], held = min(many, top);
    largest(list, many, top, scratch, [&](int at, uint64_t key) { best[at] = key; });
  }
  const double log_sum = log1p(rest), inverse = 1.0 / (double)p.job.temperature;
  auto logprob = [&](float l) { return (float)(((double)l - (double)most) * inverse - log_sum); };
  if (tid == kThreads - 1) { // of a wave that has least to do
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
  __syncthreads(); // best is whole, and the list read
  if (p.count == p.chunks) { // the chunks' groups, then the largest of those
    for (int i = wave; i < held; i += kWaves) {
      const int chunk = place_of(best[i]);
      float x[kGroups];
#pragma unroll
      for (int j = 0; j < kGroups; j++) {
        const int at = chunk * kChunk + j * kGroup + lane;
        x[j] = at < p.job.vocab ? logits[at] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < kGroups; j++) {
        const float m = wave_max(x[j]);
        if (lane == 0 && m > -INFINITY)
          list[atomicAdd(&found[2], 1)] = key_of(m, chunk * kGroups + j);
      }
    }
    __syncthreads();
    many = found[2];
    largest(list, many, top, scratch, [&](int at, uint64_t key) { best[at] = key; });
    held = min(many, top);
    __syncthreads();
  }
  // the groups' tokens that reach the last one's maximum, then the largest of those
  const float reach = many < top ? -INFINITY : value_of(best[held - 1]);
  constexpr int kMost = LLHIP_MAX_TOP / kWaves; // groups of a wave
  float x[kMost];
  int place[kMost];
#pragma unroll
  for (int i = 0; i < kMost; i++) {
    const int which = wave + i * kWaves;
    place[i] = which < held ? place_of(best[which]) * kGroup + lane : p.job.vocab;
    x[i] = place[i] < p.job.vocab ? logits[place[i]] : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < kMost; i++)
    if (x[i] >= reach && x[i] > -INFINITY)
      list[atomicAdd(&found[1], 1)] = key_of(x[i], place[i]);
  __syncthreads();
  const int tokens = found[1];
  largest(list, tokens, top, scratch, [&](int at, uint64_t key) {
    p.job.top_token[(size_t)row * top + at] = place_of(key);
    p.job.top_logprob[(size_t)row * top + at] = logprob(value_of(key));
  });
  for (int i = tokens + tid; i < top; i += kThreads)
    p.job.top_token[(size_t)row * top + i] = -1, p.job.top_logprob[(size_t)row * top + i] = -INFINITY;
}

__global__ __launch_bounds__(kThreads) void score_rows(Score p) {
  extern __shared__ uint64_t list[];
  score_row<false>(p, blockIdx.x, list);
}

__global__ __launch_bounds__(kThreads) void score_few(Score p) {
  extern __shared__ uint64_t list[];
  __shared__ unsigned arrived;
  const int row = blockIdx.y;
  score_chunk<true>(p, row, blockIdx.x * kWaves + threadIdx.x / kWave);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the thread's stores have arrived
  __syncthreads();                                 // the block's
  if (threadIdx.x == 0)
    arrived = __hip_atomic_fetch_add(&score_arrivals[row * kLine], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != gridDim.x - 1)
    return;
  if (threadIdx.x == 0)
    __hip_atomic_store(&score_arrivals[row * kLine], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  score_row<true>(p, row, list);
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

int maxima_of(int vocab) {
  const int groups = (vocab + kGroup - 1) / kGroup;
  return groups <= kThreads * kPer ? groups : chunks_of(vocab);
}

} // namespace

size_t scores_workspace(const ScoreJob &job) {
  return (size_t)job.rows * (chunks_of(job.vocab) * sizeof(Stat) + (job.top ? maxima_of(job.vocab) * sizeof(float) : 0));
}

bool launch_scores(const ScoreJob &job, void *workspace, hipStream_t stream) {
  Score p{};
  p.job = job;
  p.chunks = chunks_of(job.vocab);
  p.count = maxima_of(job.vocab);
  p.stats = (Stat *)workspace;
  p.maxima = job.top ? (float *)(p.stats + (size_t)job.rows * p.chunks) : nullptr;
  const double scale2 = 1.4426950408889634 / (double)job.temperature;
  p.scale2 = scale2 < 1e38 ? (float)scale2 : 1e38f; // finite: a difference of 0 stays 0
  p.flags = device().error_flags;
  p.vec4 = job.ld % 4 == 0 && ((uintptr_t)job.logits & 15) == 0;
  const int per = (p.count + kThreads - 1) / kThreads, keys = job.top * (kGroup > kWaves * per ? kGroup : kWaves * per);
  static_assert(LLHIP_MAX_TOP * kGroup * sizeof(uint64_t) <= 32 << 10 && kWaves * kPer <= kGroup, "the list's room");
  const size_t list = (size_t)keys * sizeof(uint64_t);
  const unsigned blocks = (unsigned)((p.chunks + kWaves - 1) / kWaves); // of a row
  if (job.rows <= kFewRows) {
    hipLaunchKernelGGL(score_few, dim3(blocks, (unsigned)job.rows), dim3(kThreads), list, stream, p);
    return launch_ok("score_few");
  }
  const int most = 32768; // rows of a launch
  for (int row0 = 0; row0 < job.rows; row0 += most) {
    const dim3 grid(blocks, (unsigned)(job.rows - row0 < most ? job.rows - row0 : most));
    hipLaunchKernelGGL(score_stats, grid, dim3(kThreads), 0, stream, p, row0);
    if (!launch_ok("score_stats"))
      return false;
  }
  hipLaunchKernelGGL(score_rows, dim3((unsigned)job.rows), dim3(kThreads), list, stream, p);
  return launch_ok("score_rows");
}

} // namespace llhip
