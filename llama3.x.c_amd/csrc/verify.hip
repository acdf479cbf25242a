// Verification of drafted tokens (gfx950): the drafts of each request accepted in turn against the target's
// probabilities, and the next token drawn from what is left.
#include <cfloat>

#include "common.h"
#include "lanes.h"

namespace llhip {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 1024;

bool launch_ok(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess || raise("launching %s failed: %s", what, hipGetErrorString(e));
}

__device__ __forceinline__ double block_sum(double v, double *red) {
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0)
    red[threadIdx.x / 64] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kThreads / 64; w++)
    s += red[w];
  __syncthreads();
  return s;
}

// The largest value of a row and its lowest place; place -1 where the row decides nothing (a NaN, +infinity, or no value
// above -infinity).
struct Top {
  float value;
  int at;
};
__device__ Top block_top(const float *row, int vocab, float *rv, int *ri) {
  float best = -INFINITY;
  int at = INT32_MAX;
  bool bad = false;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const float x = row[i];
    bad |= !(x < INFINITY);
    if (x > best)
      best = x, at = i;
  }
  if (bad)
    at = -1, best = INFINITY;
  for (int o = 32; o > 0; o >>= 1) {
    const float v = __shfl_xor(best, o);
    const int a = __shfl_xor(at, o);
    if (v > best || (v == best && a < at))
      best = v, at = a;
  }
  if ((threadIdx.x & 63) == 0)
    rv[threadIdx.x / 64] = best, ri[threadIdx.x / 64] = at;
  __syncthreads();
  best = rv[0], at = ri[0];
  for (int w = 1; w < kThreads / 64; w++)
    if (rv[w] > best || (rv[w] == best && ri[w] < at))
      best = rv[w], at = ri[w];
  __syncthreads();
  if (at == INT32_MAX)
    at = -1;
  return Top{best, at};
}

// Block r: request r, row by row.
__global__ __launch_bounds__(kThreads) void verify_requests(VerifyJob p, int *flags) {
  __shared__ double red[kThreads / 64];
  __shared__ float rv[kThreads / 64];
  __shared__ int ri[kThreads / 64];
  __shared__ double run[kThreads];
  __shared__ int chosen;
  const int r = blockIdx.x, tid = threadIdx.x;
  const int first = p.start[r], last = p.start[r + 1];
  if (first < 0 || first > last || last > p.rows) {
    if (tid == 0)
      flags[3] = 1;
    return;
  }
  if (first == last)
    return;
  auto give = [&](int accepted, int next) {
    if (tid == 0)
      p.accepted[r] = accepted, p.next[r] = next;
  };
  const double t = p.temperature;
  const int vocab = p.vocab;
  for (int row = first;; row++) {
    const float *l = p.logits + (size_t)row * p.ld;
    const Top top = block_top(l, vocab, rv, ri);
    if (top.at < 0) {
      if (tid == 0)
        flags[6] = 1;
      return give(-1, -1);
    }
    const bool drafted = row + 1 < last;
    const int x = drafted ? p.tokens[row + 1] : 0;
    if (x < 0 || x >= vocab) {
      if (tid == 0)
        flags[7] = 1;
      return give(-1, -1);
    }
    if (!p.uniform) {
      if (drafted && x == top.at)
        continue;
      return give(row - first, top.at);
    }
    auto weight = [&](const float *src, float most, int i) { return exp(((double)src[i] - (double)most) / t); };
    double sum = 0.0;
    for (int i = tid; i < vocab; i += kThreads)
      sum += weight(l, top.value, i);
    const double total = block_sum(sum, red);
    double dtotal = 1.0;
    const float *dl = nullptr;
    Top dtop{0.0f, 0};
    if (drafted) {
      double qx = 1.0;
      if (p.draft) {
        dl = p.draft + (size_t)row * p.draft_ld;
        dtop = block_top(dl, vocab, rv, ri);
        if (dtop.at < 0) {
          if (tid == 0)
            flags[6] = 1;
          return give(-1, -1);
        }
        sum = 0.0;
        for (int i = tid; i < vocab; i += kThreads)
          sum += weight(dl, dtop.value, i);
        dtotal = block_sum(sum, red);
        qx = weight(dl, dtop.value, x) / dtotal;
      }
      if ((double)p.uniform[2 * row] * qx < weight(l, top.value, x) / total)
        continue;
    }
    // the draw: what max(0, p - q) leaves, or p; each thread a run of consecutive tokens
    const int per = (vocab + kThreads - 1) / kThreads, a = min(vocab, tid * per), b = min(vocab, a + per);
    auto rest = [&](int i, bool residual) {
      const double w = weight(l, top.value, i) / total;
      if (!residual)
        return w;
      const double less = dl ? weight(dl, dtop.value, i) / dtotal : (i == x ? 1.0 : 0.0);
      return w > less ? w - less : 0.0;
    };
    for (int pass = drafted ? 0 : 1; pass < 2; pass++) {
      double mass = 0.0;
      for (int i = a; i < b; i++)
        mass += rest(i, pass == 0);
      run[tid] = mass;
      if (tid == 0)
        chosen = -1;
      __syncthreads();
      if (tid == 0)
        for (int i = 1; i < kThreads; i++)
          run[i] += run[i - 1];
      __syncthreads();
      const double whole = run[kThreads - 1], border = (double)p.uniform[2 * row + 1] * whole;
      if (whole > 0.0) {
        double at = tid ? run[tid - 1] : 0.0;
        if (at <= border && run[tid] > border) { // one thread's run holds the border
          int pick = -1;
          for (int i = a; i < b; i++) {
            const double w = rest(i, pass == 0);
            at += w;
            if (w > 0.0)
              pick = i;
            if (at > border)
              break;
          }
          chosen = pick;
        }
        __syncthreads();
        if (chosen < 0) { // a uniform of 1 or more: the last token that is left
          int mostly = -1;
          for (int i = a; i < b; i++)
            if (rest(i, pass == 0) > 0.0)
              mostly = i;
          atomicMax(&chosen, mostly);
        }
        __syncthreads();
        return give(row - first, chosen);
      }
      __syncthreads();
    }
    return; // not reached: p holds its largest token's weight
  }
}

} // namespace

bool launch_verify(const VerifyJob &job, hipStream_t stream) {
  hipLaunchKernelGGL(verify_requests, dim3((unsigned)job.count), dim3(kThreads), 0, stream, job, device().error_flags);
  return launch_ok("verify_requests");
}

} // namespace llhip
