// Verification of drafted tokens (gfx950): the drafts of each request accepted in turn against the target's
// probabilities, and the next token drawn from what is left.
//
//   verify_stats   a wave each chunk of 1024 tokens of a row, target and draft apart: the chunk's maximum, and the sum of
//                  exp((l - maximum) / T) (greedy: the maximum's lowest place), one read of the logits. HBM-bound.
//   verify_decide  block (request), a wave a row: which drafts are accepted, the row that the request stops at.
//   verify_rest    a wave each chunk of a request: where a draft is refused, the chunk's sum of max(0, p - q).
//   verify_pick    block (request): the chunk that holds the border of the draw, and the token in it.
//
// A draw's border falls between two of 128256 running sums, and an error of 1e-8 in one of them would turn some tokens
// of a thousand; so the exponentials, the sums and the products are FP64, which the vector unit runs at FP32's rate: an
// element's exponential takes 17 instructions, about half of the time that its logit takes to arrive. The stopping rows are
// read again, from the last-level cache.
#include <cfloat>

#include "common.h"
#include "lanes.h"

namespace llhip {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 1024; // tokens of a wave, 16 a lane
constexpr int kMaxChunks = 4096;
constexpr int kNone = INT32_MAX;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

// A chunk of a row: its largest logit, that one's lowest place (greedy; else some place of the chunk; kNone: every token is
// masked out; -1: it holds a NaN or +infinity), and the sum of the exponentials relative to it.
struct Stat {
  double sum;
  float top;
  int at;
};

// 2^(j / 32), each the nearest double. 32 of them: in LDS they lie on its 64 banks once, so that a wave's reads, wherever
// they go, do not wait for each other (64 took 8% longer).
constexpr int kPowers = 32;
__device__ const double kPowerTable[kPowers] = {
    0x1p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};

// exp(x) for x <= 0 from t = 32 x / ln 2: with n the integer nearest to t and f = t - n, 2^(n / 32) from the table and a shift,
// times the power series of 2^(f / 32) = exp(f ln 2 / 32), |f| <= 1/2, to the fifth power: the next term is below 3e-15 of
// it. Seventeen instructions an element with the sum's addition; the series alone, to the eleventh power, took 24.
struct Exp {
  const double *powers; // kPowerTable in LDS
  double scale;         // 32 / (T ln 2)
  __device__ __forceinline__ double operator()(float l, float top) const {
    const double t = fmax(((double)l - (double)top) * scale, -40000.0); // 2^-1250: zero, for l = -infinity too
    // t + 1.5 * 2^52 has n in its low bits: no conversion, which the FP64 unit runs at a quarter of an addition's rate
    const double shifted = t + 0x1.8p52, f = t - (shifted - 0x1.8p52);
    double s = 0x1.5d87fe78a6731p-35;
    s = fma(s, f, 0x1.3b2ab6fba4e77p-27);
    s = fma(s, f, 0x1.c6b08d704a0c0p-20);
    s = fma(s, f, 0x1.ebfbdff82c58fp-13);
    s = fma(s, f, 0x1.62e42fefa39efp-6);
    s = fma(s, f, 1.0);
    const int i = __double2loint(shifted);
    return ldexp(s * powers[i & (kPowers - 1)], i >> 5);
  }
};
// Loads the table; the caller's barrier makes it whole.
__device__ __forceinline__ void load_powers(double *powers) {
  if (threadIdx.x < kPowers)
    powers[threadIdx.x] = kPowerTable[threadIdx.x];
}

__device__ __forceinline__ double wave_add(double v) {
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o);
  return v;
}

// (value, place) pairs: the larger value, of equal ones the lower place; a row that decides nothing (-1) before all.
__device__ __forceinline__ void take_top(float &v, int &at, float w, int b) {
  if (w > v || (w == v && b < at))
    v = w, at = b;
}
__device__ __forceinline__ void wave_top(float &v, int &at) {
  for (int o = 32; o > 0; o >>= 1) {
    const float w = __shfl_xor(v, o);
    const int b = __shfl_xor(at, o);
    take_top(v, at, w, b);
  }
}

// A row's statistics.
struct Row {
  float top;
  int at;         // -1: decides nothing
  double inverse; // of the sum
};
// What becomes of a request: the row it stops at, and whether a draft is refused there.
enum { kGoOn, kAll, kRefused, kNothing, kOutside, kEmpty };
struct Decision {
  int what, row, token;
  Row target, draft; // of the stopping row
};

struct Verify {
  VerifyJob job;
  Stat *target, *draft; // [row][chunk]
  double *rest;         // [request][chunk]
  Decision *decisions;  // [request]
  int chunks;
  double scale; // 32 / (T ln 2)
  int *flags;
  bool vec4;
};

// The rows' chunks, one a wave: blocks (four chunks, row, 0) of the target and (.., row, 1) of the draft, whose rows that
// judge nothing (a request's last) are left out. 133 MB of logits take 37 us (3.6 TB/s; without the exponentials 29), five
// rows of 128256 tokens 5. Waves that take two, four or eight chunks in turn, the next one's logits on their way, were no
// faster (63, 65 and 66 us the whole call, 63 with one).
template <bool GREEDY> __global__ __launch_bounds__(kThreads) void verify_stats(Verify p, int row0) {
  __shared__ double powers[kPowers];
  const int row = row0 + blockIdx.y, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const bool drafted = blockIdx.z;
  if (row < p.job.start[0] || row >= p.job.start[p.job.count] || (drafted && row == p.job.rows - 1))
    return; // the last row of all judges nothing, and the draft's may not be there
  const float *src = drafted ? p.job.draft + (size_t)row * p.job.draft_ld : p.job.logits + (size_t)row * p.job.ld;
  auto place = [&](int j) { return p.vec4 ? 4 * (lane + j / 4 * kWave) + j % 4 : lane + j * kWave; }; // of x[j]
  const int chunk = blockIdx.x * kWaves + wave, i0 = chunk * kChunk, n = min(kChunk, p.job.vocab - i0);
  float x[16];
  if (p.vec4 && n == kChunk) { // uniform: no branch a load
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float4 v = *reinterpret_cast<const float4 *>(src + i0 + 4 * (lane + j * kWave));
      x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
    }
  } else if (n > 0) {
#pragma unroll
    for (int j = 0; j < 16; j++)
      x[j] = src[i0 + min(place(j), n - 1)];
#pragma unroll
    for (int j = 0; j < 16; j++)
      x[j] = place(j) < n ? x[j] : -INFINITY;
  }
  if (!GREEDY) {
    load_powers(powers);
    if (drafted) { // looked up while the logits are on their way
      bool last = false;
      for (int r = tid; r < p.job.count; r += kThreads)
        last |= p.job.start[r + 1] == row + 1;
      if (__syncthreads_or(last))
        return;
    }
    __syncthreads(); // the table is whole
  }
  if (n <= 0)
    return;
  const Exp exp{powers, p.scale};
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    bad |= !(x[j] < INFINITY);
    top = fmaxf(top, x[j]);
  }
  top = wave_max(top);
  bad = __any(bad);
  int at = bad ? -1 : top > -INFINITY ? i0 : kNone;
  double sum = 0.0;
  if constexpr (GREEDY) {
    int first = kNone;
#pragma unroll
    for (int j = 15; j >= 0; j--) // places rise with j
      first = x[j] == top ? i0 + place(j) : first;
    for (int o = 32; o > 0; o >>= 1)
      first = min(first, __shfl_xor(first, o));
    at = bad || at == kNone ? at : first;
  } else if (!bad && top > -INFINITY) {
#pragma unroll
    for (int j = 0; j < 16; j++)
      sum += exp(x[j], top);
    sum = wave_add(sum);
  }
  if (lane == 0)
    (drafted ? p.draft : p.target)[(size_t)row * p.chunks + chunk] = Stat{sum, bad ? INFINITY : top, at};
}

// A row's statistics from its chunks', by one wave; `mine` is the lane's first chunk, loaded before.
__device__ __forceinline__ Stat first_stat(const Verify &p, const Stat *stats, int row) {
  const int lane = threadIdx.x % kWave;
  return lane < p.chunks ? stats[(size_t)row * p.chunks + lane] : Stat{0.0, -INFINITY, kNone};
}
template <bool GREEDY> __device__ Row row_of(const Verify &p, const Exp &exp, const Stat *stats, int row, const Stat &mine) {
  const int lane = threadIdx.x % kWave;
  const Stat *s = stats + (size_t)row * p.chunks;
  float top = mine.top;
  int at = mine.at;
  for (int c = lane + kWave; c < p.chunks; c += kWave)
    take_top(top, at, s[c].top, s[c].at);
  wave_top(top, at);
  Row out{top, at == kNone ? -1 : at, 0.0};
  if (!GREEDY && out.at >= 0) {
    double sum = mine.sum * exp(mine.top, top);
    for (int c = lane + kWave; c < p.chunks; c += kWave)
      sum += s[c].sum * exp(s[c].top, top);
    out.inverse = 1.0 / wave_add(sum);
  }
  return out;
}

constexpr int kDecideThreads = 1024, kDecideWaves = kDecideThreads / kWave;

template <bool GREEDY> __global__ __launch_bounds__(kDecideThreads) void verify_decide(Verify p) {
  __shared__ Decision rows[kDecideWaves];
  __shared__ double powers[kPowers];
  const int r = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (!GREEDY)
    load_powers(powers);
  const Exp exp{powers, p.scale};
  const int first = p.job.start[r], last = p.job.start[r + 1];
  // a row outside start[0] .. start[count] - 1 (an array out of order) was not read and decides nothing
  const int low = p.job.start[0], high = p.job.start[p.job.count];
  __syncthreads(); // the table of powers is whole
  if (first < 0 || first >= last || last > p.job.rows) { // uniform
    if (threadIdx.x == 0) {
      const bool empty = first == last && first >= 0 && last <= p.job.rows;
      if (!empty)
        p.flags[3] = 1;
      p.decisions[r].what = kEmpty;
    }
    return;
  }
  for (int row0 = first; row0 < last; row0 += kDecideWaves) { // a row a wave
    const int row = row0 + wave;
    Decision mine{kNothing, row, 0, Row{}, Row{}};
    if (row < last && row >= low && row < high) {
      // what can be loaded at once is: then only the drafted token's logits wait for another load
      const bool drafted = row + 1 < last, drawn = drafted && !GREEDY && p.job.draft;
      mine.token = drafted ? p.job.tokens[row + 1] : 0;
      const bool inside = mine.token >= 0 && mine.token < p.job.vocab;
      const Stat t0 = first_stat(p, p.target, row), d0 = drawn ? first_stat(p, p.draft, row) : Stat{};
      const float u = !GREEDY ? p.job.uniform[2 * (size_t)row] : 0.0f;
      const float lt = !GREEDY && inside ? p.job.logits[(size_t)row * p.job.ld + mine.token] : 0.0f;
      const float ld = drawn && inside ? p.job.draft[(size_t)row * p.job.draft_ld + mine.token] : 0.0f;
      mine.target = row_of<GREEDY>(p, exp, p.target, row, t0);
      if (drawn)
        mine.draft = row_of<GREEDY>(p, exp, p.draft, row, d0);
      if (mine.target.at < 0) {
        mine.what = kNothing;
      } else if (!drafted) {
        mine.what = kAll;
      } else if (!inside) {
        mine.what = kOutside;
      } else if (GREEDY) {
        mine.what = mine.token == mine.target.at ? kGoOn : kRefused;
      } else if (drawn && mine.draft.at < 0) {
        mine.what = kNothing;
      } else {
        const double q = drawn ? exp(ld, mine.draft.top) * mine.draft.inverse : 1.0;
        mine.what = (double)u * q < exp(lt, mine.target.top) * mine.target.inverse ? kGoOn : kRefused;
      }
    }
    if (lane == 0)
      rows[wave] = mine;
    __syncthreads();
    const int here = min(kDecideWaves, last - row0);
    const unsigned long long stops = __ballot(lane < here && rows[lane % kDecideWaves].what != kGoOn);
    if (stops) { // uniform
      if (threadIdx.x == 0) {
        const Decision d = rows[__builtin_ctzll(stops)];
        if (d.what == kNothing || d.what == kOutside || GREEDY) {
          const bool ok = d.what != kNothing && d.what != kOutside;
          if (!ok)
            p.flags[d.what == kNothing ? 6 : 7] = 1;
          p.job.accepted[r] = ok ? d.row - first : -1;
          p.job.next[r] = ok ? d.target.at : -1;
        }
        p.decisions[r] = d;
      }
      return;
    }
    __syncthreads();
  }
}

// Each weight of N tokens at a request's stop, token i0 + j * step for j < N, to take(j, weight): max(0, p - q) after a
// refusal, p otherwise; zero from token `end` on.
template <int N, class Take>
__device__ __forceinline__ void weights(const Verify &p, const Exp &exp, const Decision &d, bool refused, int i0, int step,
                                        int end, Take take) {
  const float *t = p.job.logits + (size_t)d.row * p.job.ld;
  const float *q = refused && p.job.draft ? p.job.draft + (size_t)d.row * p.job.draft_ld : nullptr;
  float lt[N], lq[N];
#pragma unroll
  for (int j = 0; j < N; j++)
    lt[j] = t[min(i0 + j * step, p.job.vocab - 1)]; // no branch: the loads are in flight together
#pragma unroll
  for (int j = 0; j < N; j++)
    lq[j] = q ? q[min(i0 + j * step, p.job.vocab - 1)] : -INFINITY;
#pragma unroll
  for (int j = 0; j < N; j++) {
    lt[j] = i0 + j * step < end ? lt[j] : -INFINITY;
    lq[j] = i0 + j * step < end ? lq[j] : -INFINITY;
    const double have = exp(lt[j], d.target.top) * d.target.inverse;
    double less = 0.0;
    if (q)
      less = exp(lq[j], d.draft.top) * d.draft.inverse;
    else if (refused)
      less = i0 + j * step == d.token ? 1.0 : 0.0;
    take(j, have > less ? have - less : 0.0);
  }
}

__global__ __launch_bounds__(kThreads) void verify_rest(Verify p) {
  static_assert(kChunk / kWave == 16, "16 tokens a lane");
  __shared__ double powers[kPowers];
  const int lane = threadIdx.x % kWave, chunk = blockIdx.x * kWaves + threadIdx.x / kWave, r = blockIdx.y;
  load_powers(powers);
  const Decision d = p.decisions[r];
  if (d.what != kRefused)
    return;
  __syncthreads();
  if (chunk >= p.chunks)
    return;
  const Exp exp{powers, p.scale};
  double sum = 0.0;
  weights<16>(p, exp, d, true, chunk * kChunk + lane, kWave, min(p.job.vocab, (chunk + 1) * kChunk),
              [&](int, double w) { sum += w; });
  sum = wave_add(sum);
  if (lane == 0)
    p.rest[(size_t)r * p.chunks + chunk] = sum;
}

constexpr int kPickThreads = 256;

__global__ __launch_bounds__(kPickThreads) void verify_pick(Verify p) {
  constexpr int kWaves = kPickThreads / kWave, kTokens = kChunk / kPickThreads;
  __shared__ double mass[kMaxChunks], sums[kWaves], powers[kPowers];
  __shared__ double before, border;
  __shared__ int chunk, firsts[kWaves], lasts[kWaves];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  load_powers(powers);
  const Exp exp{powers, p.scale};
  const Decision d = p.decisions[r];
  if (d.what != kAll && d.what != kRefused)
    return; // verify_decide has answered
  __syncthreads();
  bool refused = d.what == kRefused;
  // the chunks' masses, and by one wave their running sums, 64 at a time: the whole, then the first chunk at which they
  // pass the border (at last, for a uniform of 1, the last chunk that holds anything); should the rest be empty, the
  // target's own masses
  for (;;) {
    const Stat *s = p.target + (size_t)d.row * p.chunks;
    for (int c = tid; c < p.chunks; c += kPickThreads)
      mass[c] = refused ? p.rest[(size_t)r * p.chunks + c] : s[c].sum * exp(s[c].top, d.target.top) * d.target.inverse;
    __syncthreads();
    if (wave == 0) {
      double whole = 0.0;
      for (int c = lane; c < p.chunks; c += kWave)
        whole += mass[c];
      whole = wave_add(whole);
      const double line = (double)p.job.uniform[2 * (size_t)d.row + 1] * whole;
      double run = 0.0, at = 0.0;
      int hit = -1;
      for (int c0 = 0; c0 < p.chunks; c0 += kWave) {
        const double m = c0 + lane < p.chunks ? mass[c0 + lane] : 0.0;
        double sum = m;
        for (int o = 1; o < kWave; o <<= 1) {
          const double v = __shfl_up(sum, o);
          if (lane >= o)
            sum += v;
        }
        const unsigned long long passed = __ballot(m > 0.0 && run + sum > line), any = __ballot(m > 0.0);
        const int pick = passed ? __builtin_ctzll(passed) : any ? 63 - __builtin_clzll(any) : -1;
        if (pick >= 0) {
          hit = c0 + pick;
          at = run + __shfl(sum - m, pick);
        }
        if (passed)
          break;
        run += __shfl(sum, kWave - 1);
      }
      if (lane == 0)
        chunk = hit, before = at, border = line;
    }
    __syncthreads();
    if (chunk >= 0 || !refused)
      break;
    refused = false;
  }
  // the chunk's tokens, consecutive ones a thread
  const int i0 = max(chunk, 0) * kChunk + tid * kTokens, end = min(p.job.vocab, i0 + kTokens);
  double w[kTokens], sum = 0.0;
  weights<kTokens>(p, exp, d, refused, i0, 1, end, [&](int j, double x) { sum += w[j] = x; });
  double run = sum; // of the wave's threads up to this one
  for (int o = 1; o < kWave; o <<= 1) {
    const double v = __shfl_up(run, o);
    if (lane >= o)
      run += v;
  }
  if (lane == kWave - 1)
    sums[wave] = run;
  __syncthreads();
  double at = before + (run - sum);
  for (int v = 0; v < wave; v++)
    at += sums[v];
  // the first token at which the running sum passes the border: of the threads that find one, the lowest; rounding (the
  // chunk's sum was taken in another order) may leave none, then the chunk's last token that has any weight
  int first = kNone, mostly = -1;
#pragma unroll
  for (int j = 0; j < kTokens; j++) {
    at += w[j];
    if (w[j] > 0.0) {
      mostly = i0 + j;
      if (at > border && first == kNone)
        first = i0 + j;
    }
  }
  for (int o = 32; o > 0; o >>= 1) {
    first = min(first, __shfl_xor(first, o));
    mostly = max(mostly, __shfl_xor(mostly, o));
  }
  if (lane == 0)
    firsts[wave] = first, lasts[wave] = mostly;
  __syncthreads();
  if (tid == 0) {
    for (int v = 0; v < kWaves; v++) {
      first = min(first, firsts[v]);
      mostly = max(mostly, lasts[v]);
    }
    p.job.accepted[r] = d.row - p.job.start[r];
    p.job.next[r] = first != kNone ? first : mostly;
  }
}

} // namespace

bool verify_shape_ok(int rows, int vocab) { return vocab <= kChunk * kMaxChunks && rows <= (1 << 20); }

size_t verify_workspace(const VerifyJob &job) {
  const size_t chunks = ((size_t)job.vocab + kChunk - 1) / kChunk;
  return (size_t)job.count * sizeof(Decision) + (size_t)job.rows * chunks * sizeof(Stat) * (job.draft ? 2 : 1) +
         (size_t)job.count * chunks * sizeof(double);
}

bool launch_verify(const VerifyJob &job, void *workspace, hipStream_t stream) {
  Verify p{};
  p.job = job;
  p.chunks = (job.vocab + kChunk - 1) / kChunk;
  p.decisions = (Decision *)workspace;
  p.target = (Stat *)(p.decisions + job.count);
  p.draft = p.target + (size_t)job.rows * p.chunks;
  p.rest = (double *)(job.draft ? p.draft + (size_t)job.rows * p.chunks : p.draft);
  p.scale = job.uniform ? 32.0 / ((double)job.temperature * 0.6931471805599453) : 0.0;
  p.flags = device().error_flags;
  p.vec4 = job.ld % 4 == 0 && ((uintptr_t)job.logits & 15) == 0 &&
           (!job.draft || (job.draft_ld % 4 == 0 && ((uintptr_t)job.draft & 15) == 0));
  const bool greedy = !job.uniform;
  const int most = 32768; // rows of a launch
  for (int row0 = 0; row0 < job.rows; row0 += most) {
    const dim3 grid((unsigned)((p.chunks + kWaves - 1) / kWaves), (unsigned)(job.rows - row0 < most ? job.rows - row0 : most),
                    job.draft ? 2 : 1);
    if (greedy)
      hipLaunchKernelGGL(verify_stats<true>, grid, dim3(kThreads), 0, stream, p, row0);
    else
      hipLaunchKernelGGL(verify_stats<false>, grid, dim3(kThreads), 0, stream, p, row0);
    if (!launch_ok("verify_stats"))
      return false;
  }
  if (greedy)
    hipLaunchKernelGGL(verify_decide<true>, dim3((unsigned)job.count), dim3(kDecideThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(verify_decide<false>, dim3((unsigned)job.count), dim3(kDecideThreads), 0, stream, p);
  if (!launch_ok("verify_decide"))
    return false;
  if (greedy)
    return true;
  hipLaunchKernelGGL(verify_rest, dim3((unsigned)((p.chunks + kWaves - 1) / kWaves), (unsigned)job.count), dim3(kThreads), 0, stream, p);
  if (!launch_ok("verify_rest"))
    return false;
  hipLaunchKernelGGL(verify_pick, dim3((unsigned)job.count), dim3(kPickThreads), 0, stream, p);
  return launch_ok("verify_pick");
}

} // namespace llhip
