// Attention over a cache in pages (gfx950).
//
//   attn_paged        block: a slice of a KV head's walks, a walk being a tile of one request's query vectors over its
//                     positions. One pass over K and V with the softmax's running maximum and sum, products on the matrix
//                     cores; a walk that several blocks share is joined by the last of them to arrive.
//   attn_paged_rows   any shape, one row and KV head a block: 32 rows of 16 heads over 4 of 100 at 1450 positions on average take
//                     1.8 ms, where the tiled form takes 32 us for heads of 96.
//
// Measured at 32 heads over 8 KV heads of dimension 128, BF16 pages: 32 requests of one row at 2200 positions on average 65 us
// (290 MB of K and V: 4.5 TB/s), 64 at 5670 262 us (5.7 TB/s), one at 4000 13 us; five prompts' chunks, 1616 rows behind 1146
// positions on average, 115 to 125 us (310 TFLOP/s, three matrix products each). F32 pages: one row at 35000 positions 70 us
// (4.1 TB/s), 16 requests of two to seven rows 50 us, the prompts 350 us. Single rows are bound by HBM, behind 5 us of launch, plan
// and table and before 5 us of join; wide tiles by a step's 1536 cycles of matrix instructions and 950 of vector ones beside
// the reads from LDS, which overlap little; F32 prompts by the FP32 matrix instructions (103 of 157 TFLOP/s).
#include <cfloat>
#include <type_traits>

#include "paged_device.h"

#include "lanes.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

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

// x where it is not finite, else 0. A row's sum over values of which some are not finite is the sum of those, whatever their
// weights: infinity, or NaN beside one of the other sign or a NaN. A product can't tell: weights are above zero, but FP32, or
// a weight's lower part in BF16, has 0 for many of them, and 0 * infinity is NaN.
__device__ __forceinline__ float odd_only(float x) { return isfinite(x) ? 0.0f : x; }

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
  const bool failed = __syncthreads_or(bad);
  float *dst = job.out + ((size_t)row * job.n_heads + (size_t)g * kv_mul) * hd;
  for (int i = tid; i < kv_mul * hd; i += kThreads) {
    float total = 0.0f;
    for (int s2 = 0; s2 < shares; s2++)
      total += acc[(size_t)s2 * kv_mul * hd + i];
    total /= run_sum[i / hd];
    if (!isfinite(total) && !failed) {
      float odd = 0.0f;
#pragma unroll 8
      for (int t = 0; t < positions; t++) {
        const int page = max(page_of(b, request, t / b.page_size), 0);
        odd += odd_only(value(values + (size_t)page * b.page_values + (size_t)(t % b.page_size) * b.pos_stride + i % hd));
      }
      total = odd == 0.0f ? total : odd;
    }
    dst[i] = total;
  }
}

// ---- the matrix-core form ---------------------------------------------------------------------------------------------

constexpr int kWaves = kThreads / kWave;
constexpr int kStep = 32;              // positions that a wave takes at once
constexpr int kRound = kWaves * kStep; // positions that a block takes at once in a tile of up to 16 vectors
constexpr int kTileVectors = 64;       // query vectors of a tile
constexpr int kWideVectors = 128;      // of a wide one
constexpr int kMaxBlocksPerCu = 2;
constexpr int kMaxArrivals = 4096;
constexpr unsigned kNowhere = 0x7ffffff0u; // an offset past every buffer: a load reads zero there

// How many of a walk's blocks have stored their part, by the block that the walk begins in: zero between launches, as the
// last to arrive sets it back.
constexpr int kLine = 32; // each in a cache line of its own: additions to one line wait for each other
__device__ unsigned paged_arrivals[kMaxArrivals * kLine];

struct FastPaged {
  AttentionPagedJob job;
  int kv_mul, blocks; // blocks: of a KV head
  int tile_rows;      // rows of a full tile
  int tile_vectors;   // at most, of a tile: kTileVectors or kWideVectors
  int full_begin, full_position; // begin_time and position_time of a full tile
  float scale2;       // log2(e) / sqrt(hd)
  // slots of tile_vectors (HD + 2) floats, [KV head][block][0: a walk that an earlier block began, 1: one that this block
  // begins]: the vectors' sums, then their maxima and weights' sums
  float *partial;
  int *flags;
  bool pairs;   // two blocks to a CU, and an even number to a KV head: the first half of them are the CUs' first blocks
  bool fours;   // a page is a multiple of four positions
  bool q_vec;   // q in whole 16-byte vectors
  bool out_vec; // out likewise
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The thread's number, new to the compiler at each walk: else it keeps what walks derive from it in registers all along.
__device__ __forceinline__ int own_thread() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}
// Nothing moves across: a phase's registers are free before the next one's are taken.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// The walks of a KV head lie one behind the other on a line, each as long as it takes in time, and the line is cut into
// slices of equal time, one for a block: all blocks start together and end together. A walk's begin and end take as long as
// begin_time positions of a small tile.
constexpr int kBegin = 256, kWideBegin = 768;
// A slice is at least this long: shorter ones do not pay for a walk's join, and a block inside a walk has some of its
// positions however they are rounded (a round is unit * grain long).
constexpr int kMinSlice = 2 * kRound;

// Waves that walk a tile's positions together, a wave 16 vectors: four, two or one.
__device__ __forceinline__ int walkers_of(int vectors) { return vectors <= 16 ? 4 : vectors <= 32 ? 2 : 1; }
// How long a position takes: with fewer waves a tile, longer.
constexpr int kWidePosition = 4;
__device__ __forceinline__ int position_time(int vectors) {
  return vectors > kTileVectors ? kWidePosition : kWaves / walkers_of(vectors);
}

__device__ __forceinline__ int begin_time(int vectors) { return vectors > kTileVectors ? kWideBegin : kBegin; }
constexpr int kMostTime = kWidePosition > kWaves ? kWidePosition : kWaves;
static_assert(kMinSlice >= kWidePosition * kStep && kMinSlice >= kRound, "a slice holds a round");

// Where tile t of a request begins on the request's part of the line: t full tiles before it, tile i of length + (i + 1)
// tile_rows positions.
__device__ __forceinline__ long long tile_start(const FastPaged &p, int length, long long t) {
  return t * p.full_begin + p.full_position * (t * length + p.tile_rows * (t * (t + 1) / 2));
}
__device__ __forceinline__ long long request_time(const FastPaged &p, const PagedRequest &q) {
  if (q.rows == 0)
    return 0;
  const int t = ceil_div(q.rows, p.tile_rows) - 1, rest = q.rows - t * p.tile_rows;
  return tile_start(p, q.length, t) + begin_time(rest * p.kv_mul) +
         (long long)position_time(rest * p.kv_mul) * (q.length + q.rows);
}

struct Plan {
  long long line[kMaxRequests]; // where request r's walks end
  long long wave_sum[kWaves];
};

// x / y of the line's lengths (below 2^50, where the double quotient's whole part is exact), a third of the time that the
// compiler's division takes.
__device__ __forceinline__ long long whole(long long x, long long y) { return (long long)((double)x / (double)y); }

// The line's slices: as long as it is through all blocks, those of the CUs' first blocks are longer by a kFirstMore-th, those
// of the second ones shorter, which the CU's arbitration leaves behind (with equal slices the prompts' second blocks took 107 us
// beside 88; all together 131.5 us, now 126). Without wide tiles memory sets the pace, and equal slices were as good.
constexpr int kFirstMore = 5;
struct Slices {
  long long first, second; // of a block before and from `turn` on
  int turn;
  __device__ __forceinline__ long long start(int block) const {
    return block <= turn ? block * first : turn * first + (block - turn) * second;
  }
  __device__ __forceinline__ int block_of(long long x) const { // that x lies in the slice of
    return x < turn * first ? (int)whole(x, first) : turn + (int)whole(x - turn * first, second);
  }
};
__device__ __forceinline__ Slices make_slices(const FastPaged &p, long long total) {
  const long long even = whole(total + p.blocks - 1, p.blocks), more = whole(even, kFirstMore);
  if (!p.pairs || even - more < kMinSlice)
    return Slices{even > kMinSlice ? even : kMinSlice, even > kMinSlice ? even : kMinSlice, p.blocks};
  return Slices{even + more, even - more, p.blocks / 2};
}

// Fills the plan; returns the line's length.
__device__ long long make_plan(const FastPaged &p, Plan &plan) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  constexpr int kPer = kMaxRequests / kThreads; // requests of a thread, at most
  const PagedDev &b = p.job.batch;
  const int per = ceil_div(b.count, kThreads), r0 = tid * per;
  long long sum = 0, time[kPer];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    time[k] = 0;
    if (k < per && r0 + k < b.count)
      sum += time[k] = request_time(p, paged_request(b, r0 + k, bad));
  }
  if (bad && blockIdx.x == 0)
    p.flags[3] = 1;
  long long run = sum; // the threads' up to this one
  for (int o = 1; o < kWave; o <<= 1) {
    const long long v = __shfl_up(run, o);
    if (lane >= o)
      run += v;
  }
  if (lane == kWave - 1)
    plan.wave_sum[wave] = run;
  __syncthreads();
  long long at = run - sum, total = 0;
  for (int w = 0; w < kWaves; w++) {
    if (w < wave)
      at += plan.wave_sum[w];
    total += plan.wave_sum[w];
  }
#pragma unroll
  for (int k = 0; k < kPer; k++)
    if (k < per && r0 + k < b.count)
      plan.line[r0 + k] = at += time[k];
  __syncthreads();
  return total;
}

// A block's part of a walk: query vectors (row row0 + v / kv_mul, head g kv_mul + v % kv_mul for v < vectors) over positions
// t0 .. t1 - 1 of request r; row row0 + j sees positions up to last0 + j.
struct Item {
  int r, g, row0, vectors, last0;
  int t0, t1;
  int walkers;  // waves of 16 vectors
  int slot;     // of the part's sums, or -1: the part is the whole, and goes to out
};

__device__ __forceinline__ float four_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float four_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// A part's sums go past the XCDs' own L2s: stores of agent scope write through, loads of agent scope read what they wrote. (A
// release and an acquire around plain ones write back and drop a whole L2 a block: 32 requests took 134 us, not 65.) Each store
// takes its place in memory's queues, whatever its size, so the sums go out in whole rows, [vector][HD], 16 bytes a lane: as
// lanes hold them, 128 bytes each, in stores of 8 bytes the prompts took 236 us, of 16 156.
constexpr int kAgent = 16; // the cache policy's sc1
struct Slot {
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned ends; // where the maxima and weights' sums begin, in bytes
};
template <int HD> __device__ __forceinline__ Slot slot_at(const FastPaged &p, int slot) {
  const unsigned floats = (unsigned)(p.tile_vectors * (HD + 2));
  const uint64_t base = (uint64_t)(uintptr_t)p.partial + (uint64_t)uniform(slot) * floats * 4u;
  return Slot{__builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)base, (short)0, (int)(floats * 4u), 0x00020000),
              (unsigned)(p.tile_vectors * HD) * 4u};
}
__device__ __forceinline__ void put4(const Slot &s, unsigned at, const float4 &x) {
  const v4u bits = {__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(x.z), __float_as_uint(x.w)};
  __builtin_amdgcn_raw_buffer_store_b128(bits, s.rsrc, at * 16u, 0, kAgent);
}
__device__ __forceinline__ float4 get4(const Slot &s, unsigned at) {
  const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(s.rsrc, at * 16u, 0, kAgent));
  return float4{__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
}
__device__ __forceinline__ void put_end(const Slot &s, int v, float m, float l) {
  const v2u bits = {__float_as_uint(m), __float_as_uint(l)};
  __builtin_amdgcn_raw_buffer_store_b64(bits, s.rsrc, s.ends + 8u * (unsigned)v, 0, kAgent);
}
// Of a slot that differs from lane to lane.
__device__ __forceinline__ float2 load_end(const FastPaged &p, int slot, int v, int dims) {
  const float *at = p.partial + (size_t)slot * (size_t)(p.tile_vectors * (dims + 2)) + (size_t)(p.tile_vectors * dims) + 2 * v;
  const unsigned long long x = __hip_atomic_load(reinterpret_cast<const unsigned long long *>(at), __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
  return float2{__uint_as_float((unsigned)x), __uint_as_float((unsigned)(x >> 32))};
}

// exp2(x) of what moves sums from one maximum to another, x <= 0: denormal below 2^-126, where the instruction gives 0. The
// weights in such sums may be 2^8, so that 2^-118 of the largest weight would be lost, and V may hold values 10^40 apart.
__device__ __forceinline__ float exp2_far(float x) {
  const float half = __builtin_amdgcn_exp2f(0.5f * x);
  return half * half;
}

// x = a + b + c exactly, each of at most eight significant bits (truncated, so that nothing overflows): three BF16 values.
// Two x give a dword of each part.
__device__ __forceinline__ void bf16_parts(float x, float y, unsigned (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
    part[i] = __builtin_amdgcn_perm(b, a, 0x07060302); // the upper halves
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
}
__device__ __forceinline__ v4f mfma_bf16(const v4u &a, const v4u &b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Where 16 positions' K or V rows lie (page_size a multiple of 16: in one page), as a buffer: a load past the rows that
// belong to the walk reads zero, so that nothing of a page's rest, and no page behind the last, is touched.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void *cache, long long offset, int bytes) {
  const uint64_t base = (uint64_t)(uintptr_t)cache + (uint64_t)offset;
  return __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)base, (short)0, bytes, 0x00020000);
}

// Not 0 behind a value that is not finite.
__device__ __forceinline__ float mark_of(const float4 &x, float mark) {
  return fmaf(x.x, 0.0f, fmaf(x.y, 0.0f, fmaf(x.z, 0.0f, fmaf(x.w, 0.0f, mark))));
}

// 16 vectors' sums of a wave, as its lanes hold them, row by row to the part's slot or, multiplied by the inverse of the
// weights' sums, to out: through the wave's own rows of LDS, so that a store's lanes lie side by side. Returns the mark of what
// it gave to out.
template <int HD, int EV, class Row>
__device__ __forceinline__ float store_rows(const FastPaged &p, const Slot &slot, bool whole, const v4f (&o)[HD / 16],
                                            float inverse, float *rows, int lane, int hd, int v0, int count, Row row_of) {
  constexpr int kRow = HD + 4;
  const int lq = lane >> 4, lc = lane & 15;
  const float scale = whole ? inverse : 1.0f;
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int e = 0; e < HD / 16; e += 4) {
      const int d = (e / EV * 16 + 4 * lq + r) * EV + e % EV;
      *reinterpret_cast<float4 *>(rows + lc * kRow + d) =
          float4{o[e][r] * scale, o[e + 1][r] * scale, o[e + 2][r] * scale, o[e + 3][r] * scale};
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // written by one lane, read by another
  __builtin_amdgcn_wave_barrier();
  const int hd4 = hd / 4;
  float mark = 0.0f;
  for (int i = lane; i < count * hd4; i += kWave) {
    const int v = i / hd4, d = i % hd4 * 4;
    const float4 x = *reinterpret_cast<const float4 *>(rows + v * kRow + d);
    if (!whole) {
      put4(slot, (unsigned)((v0 + v) * (HD / 4) + d / 4), x);
    } else {
      mark = mark_of(x, mark);
      float *to = row_of(v0 + v) + d;
      if (p.out_vec)
        *reinterpret_cast<float4 *>(to) = x;
      else
        to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // read before it is written again
  __builtin_amdgcn_wave_barrier();
  return mark;
}

// The tile's walk: each wave has 16 of its vectors, and takes 32 positions in turn with the other waves that have the same.
//
// Lane (lq = lane / 16, lc = lane % 16). S^T = K Q^T and O^T = V^T P^T, so that a lane holds one vector's (lc) scores, weights
// and sums, and no weight changes lanes: the scores of positions 16 t + 4 lq + e are in the lane that feeds positions 16 t + 4
// lq + e to the second product, whose order of summation is free.
//   BF16: 32 dimensions, or 32 positions, an instruction; a lane's V rows (8 positions, 8 dimensions each) are turned by byte
//   permutes within the lane. Q and P as three exact parts each.
//   F32: 4 dimensions, or 4 positions, an instruction; FP32 products.
// Dimension of instruction e's row m: EV dimensions a lane, 16 lanes, further ones EV * 16 behind.
// Pages of a multiple of 16 positions hold 16 rows side by side, named by one entry of the table that a lane has looked up
// before; of others each K row and each four V rows (each V row, where four may lie in two pages) have a look of their own.
// MODE: whole heads of HD dimensions, heads of fewer, or either with pages that are no multiple of 16 positions.
// Returns the mark of what it gave to out.
enum { kWhole, kPart, kAny };
template <typename T, int HD, int MODE> __device__ float walk(const FastPaged &p, const Item &it, float *lds) {
  constexpr bool kBf16 = sizeof(T) == 2, ANY = MODE == kAny;
  constexpr int E = HD / 16, EV = E < (kBf16 ? 8 : 4) ? E : (kBf16 ? 8 : 4), kVecs = E / EV; // a V row: kVecs loads of EV
  constexpr int kSteps = kBf16 ? HD / 32 : HD / 16; // a K row: loads of 16 bytes
  constexpr int kPerLoad = kBf16 ? 8 : 4;           // dimensions of one
  constexpr int kRow = HD + 4;
  const PagedDev &b = p.job.batch;
  const int tid = own_thread(), lane = tid & (kWave - 1), wave = uniform(tid / kWave), lq = lane >> 4, lc = lane & 15;
  const int hd = MODE == kWhole ? HD : p.job.head_dim, kv_mul = p.kv_mul;
  const int v0 = wave / it.walkers * 16;    // the wave's first vector
  const int mine = min(it.vectors - v0, 16); // its vectors
  const int first = it.t0 + wave % it.walkers * kStep, stride = it.walkers * kStep;
  // positions that some of the wave's vectors see
  const int end = mine > 0 ? min(it.t1, it.last0 + (v0 + mine - 1) / kv_mul + 1) : it.t0;
  const int all_see = it.last0 + v0 / kv_mul + 1; // positions below are seen by all of them
  const bool active = lc < mine;
  const int last = active ? it.last0 + (v0 + lc) / kv_mul : -1; // the lane's vector's last position
  v4f o[E];
  float m_run = -FLT_MAX, l_run = 0.0f, odd = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e++)
    o[e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const size_t head = (size_t)it.g * b.head_base;
  // lane 2 i + t: where positions 16 t .. of the wave's step i (of 32 steps) lie, in bytes
  long long places = 0;
  auto look_up = [&](int pos) {
    const int at = min(pos + lane / 2 * stride + 16 * (lane & 1), max(end - 1, 0));
    const int number = at / b.page_size, page = page_of(b, it.r, number);
    if (page < 0)
      p.flags[8] = 1;
    places = (long long)(((size_t)max(page, 0) * b.page_values + (size_t)((at - number * b.page_size) & ~15) * b.pos_stride +
                          head) * sizeof(T));
  };
  auto place = [&](int i) {
    const int lo = __builtin_amdgcn_readlane((int)places, i), hi = __builtin_amdgcn_readlane((int)(places >> 32), i);
    return (long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
  };
  // any page size: where position t lies, in values
  auto place_any = [&](int t) {
    const int at = min(t, max(end - 1, 0)), number = at / b.page_size, page = page_of(b, it.r, number);
    if (page < 0)
      p.flags[8] = 1;
    return (size_t)max(page, 0) * b.page_values + (size_t)(at - number * b.page_size) * b.pos_stride + head;
  };
  const unsigned row_bytes = (unsigned)b.pos_stride * (unsigned)sizeof(T);
  const unsigned k_row = (unsigned)lc * row_bytes, v_row = (unsigned)(4 * lq) * row_bytes;
  auto k_off = [&](int s) {
    const int d = (4 * s + lq) * kPerLoad;
    return d < hd ? k_row + (unsigned)(d * sizeof(T)) : kNowhere;
  };
  auto v_off = [&](int e, int u) {
    const int d = (u * 16 + lc) * EV;
    return d < hd ? v_row + (unsigned)e * row_bytes + (unsigned)(d * sizeof(T)) : kNowhere;
  };
  v4u kr[2][kSteps];
  unsigned vr[8][kVecs][EV * sizeof(T) / 4]; // positions 16 (j / 4) + 4 lq + j % 4
  auto load_rows = [&](int pos, int i, auto take) { // both 16-row buffers of the step at pos, the wave's i-th since look_up
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const int rows = min(end - (pos + 16 * t), 16);
      const int bytes = rows > 0 ? (int)((unsigned)(rows - 1) * row_bytes + (unsigned)(hd * sizeof(T))) : 0;
      take(t, place(min(2 * i + t, kWave - 1)), bytes);
    }
  };
  auto load_k = [&](int pos, int i) {
    if constexpr (ANY) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const T *row = (const T *)p.job.key + place_any(pos + 16 * t + lc);
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          const int d = (4 * s + lq) * kPerLoad;
          kr[t][s] = *reinterpret_cast<const v4u *>(row + (d < hd ? d : 0)); // there Q is zero
        }
      }
    } else {
      load_rows(pos, i, [&](int t, long long offset, int bytes) {
        const auto rsrc = rows_of(p.job.key, offset, bytes);
#pragma unroll
        for (int s = 0; s < kSteps; s++)
          kr[t][s] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rsrc, k_off(s), 0, 0));
      });
    }
  };
  auto load_v = [&](int pos, int i) {
    if constexpr (ANY) {
      size_t four = 0; // where the first of four positions lies
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int t = pos + 16 * (j / 4) + 4 * lq + j % 4;
        if (j % 4 == 0 || !p.fours) // uniform
          four = place_any(t);
        // the same page holds the next three; behind the end the first is read again
        const T *row = (const T *)p.job.value + four + (p.fours && t < end ? (size_t)(j % 4) * b.pos_stride : 0);
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
          const int d = (u * 16 + lc) * EV;
          if constexpr (EV * sizeof(T) == 16) {
            const v4u x = *reinterpret_cast<const v4u *>(row + (d < hd ? d : 0));
#pragma unroll
            for (int c = 0; c < 4; c++)
              vr[j][u][c] = t < end ? x[c] : 0u;
          } else {
            const v2u x = *reinterpret_cast<const v2u *>(row + (d < hd ? d : 0));
#pragma unroll
            for (int c = 0; c < 2; c++)
              vr[j][u][c] = t < end ? x[c] : 0u;
          }
        }
      }
    } else {
      load_rows(pos, i, [&](int t, long long offset, int bytes) {
        const auto rsrc = rows_of(p.job.value, offset, bytes);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int u = 0; u < kVecs; u++) {
            if constexpr (EV * sizeof(T) == 16) {
              const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rsrc, v_off(e, u), 0, 0));
#pragma unroll
              for (int c = 0; c < 4; c++)
                vr[4 * t + e][u][c] = x[c];
            } else {
              const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(rsrc, v_off(e, u), 0, 0));
#pragma unroll
              for (int c = 0; c < 2; c++)
                vr[4 * t + e][u][c] = x[c];
            }
          }
      });
    }
  };
  // the query vectors on their way with the first step's rows, then scaled, in the order in which K's dimensions come
  constexpr int kParts = kBf16 ? 3 : 1;
  v4u qp[kSteps][kParts];
  {
    const int v = active ? v0 + lc : 0;
    const float *src = p.job.q + (size_t)(it.row0 + v / kv_mul) * p.job.q_stride + ((size_t)it.g * kv_mul + v % kv_mul) * hd;
    float x[kSteps][kPerLoad];
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const int d = (4 * s + lq) * kPerLoad;
      const float *at = src + (d < hd ? d : 0);
      if (p.q_vec) {
#pragma unroll
        for (int c = 0; c < kPerLoad; c += 4) {
          const float4 four = *reinterpret_cast<const float4 *>(at + c);
          x[s][c] = four.x, x[s][c + 1] = four.y, x[s][c + 2] = four.z, x[s][c + 3] = four.w;
        }
      } else {
#pragma unroll
        for (int c = 0; c < kPerLoad; c++)
          x[s][c] = at[c];
      }
    }
    if constexpr (!ANY)
      look_up(first);
    load_k(first, 0);
    load_v(first, 0);
    fence();
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const bool there = active && (4 * s + lq) * kPerLoad < hd;
#pragma unroll
      for (int c = 0; c < kPerLoad; c++)
        x[s][c] = there ? x[s][c] * p.scale2 : 0.0f;
      if constexpr (kBf16) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          unsigned part[3];
          bf16_parts(x[s][2 * c], x[s][2 * c + 1], part);
#pragma unroll
          for (int k = 0; k < 3; k++)
            qp[s][k][c] = part[k];
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
          qp[s][0][c] = __float_as_uint(x[s][c]);
      }
    }
  }
  int i = 0; // the step's number since look_up
  unsigned odd_values = 0;
  for (int pos = first; pos < end; pos += stride) {
    v4f sc[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      if constexpr (kBf16) {
#pragma unroll
        for (int k = 2; k >= 0; k--)
#pragma unroll
          for (int t = 0; t < 2; t++)
            sc[t] = mfma_bf16(kr[t][s], qp[s][k], sc[t]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int t = 0; t < 2; t++)
            sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[t][s][c]), __uint_as_float(qp[s][0][c]), sc[t],
                                                         0, 0, 0);
      }
    }
    fence();
    if constexpr (!ANY)
      if (++i == kWave / 2) { // uniform
        look_up(pos + stride);
        i = 0;
      }
    load_k(pos + stride, i);
    fence();
    // weights
    float w[8], top = -FLT_MAX;
#pragma unroll
    for (int j = 0; j < 8; j++)
      w[j] = sc[j / 4][j % 4];
    if (pos + kStep > all_see || pos + kStep > end || mine < 16) { // a lane without a vector sees nothing
      const int seen = min(last, end - 1) - pos - 4 * lq;
#pragma unroll
      for (int j = 0; j < 8; j++)
        w[j] = 16 * (j / 4) + j % 4 <= seen ? w[j] : -FLT_MAX;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      odd = fmaf(w[j], 0.0f, odd);
      top = fmaxf(top, w[j]);
    }
    // the maximum moves only where weights would pass 2^8: rare, and the sums keep their bits
    if (__any(top > m_run + 8.0f)) {
      const float m = fmaxf(m_run, four_max(top)), alpha = exp2_far(m_run - m);
      l_run *= alpha;
      m_run = m;
#pragma unroll
      for (int e = 0; e < E; e++)
        o[e] *= alpha;
    }
    const float base = m_run > -FLT_MAX ? m_run : 0.0f; // a masked score, -FLT_MAX, has no weight where a lane has seen no other
#pragma unroll
    for (int j = 0; j < 8; j++) {
      w[j] = __builtin_amdgcn_exp2f(w[j] - base);
      l_run += w[j]; // this lane's positions; the four lanes of a vector meet at the end
    }
    // A V value that is not finite must reach the vectors that see its position alone, and 0 * infinity would carry it to
    // those that do not: where some do not, the product takes 0 in its place, and it is added to those that do at the end.
    if (pos + kStep > all_see && all_see < end) {
      // an exponent of ones, plus one, carries into the sign's place
      unsigned met = 0;
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
#pragma unroll
          for (unsigned c = 0; c < EV * sizeof(T) / 4; c++) {
            unsigned &x = vr[j][u][c];
            if constexpr (kBf16) {
              const unsigned carry = ((x & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u;
              met |= carry;
              x &= ~((carry << 16) - carry);
            } else {
              const int carry = (int)((x & 0x7f800000u) + 0x00800000u) >> 31;
              met |= (unsigned)carry;
              x &= ~(unsigned)carry;
            }
          }
          asm volatile("" : "+v"(met)); // one after the other: registers
        }
      odd_values |= met;
    }
    if constexpr (kBf16) {
      v4u wp[3];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        unsigned part[3];
        bf16_parts(w[2 * c], w[2 * c + 1], part);
#pragma unroll
        for (int k = 0; k < 3; k++)
          wp[k][c] = part[k];
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        v4u vt;
#pragma unroll
        for (int c = 0; c < 4; c++)
          vt[c] = __builtin_amdgcn_perm(vr[2 * c + 1][e / EV][e % EV / 2], vr[2 * c][e / EV][e % EV / 2],
                                        e % 2 ? 0x07060302 : 0x05040100);
#pragma unroll
        for (int k = 2; k >= 0; k--)
          o[e] = mfma_bf16(vt, wp[k], o[e]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < E; e++)
          o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j][e / EV][e % EV]), w[j], o[e], 0, 0, 0);
    }
    fence();
    load_v(pos + stride, i);
    fence();
  }
  if (odd != 0.0f)
    p.flags[1] = 1;
  if (__any(odd_values != 0)) {
    for (int pos = first; pos < end; pos += stride) // the steps above
      for (int t = pos + kStep > all_see ? pos : end; t < min(pos + kStep, end); t++) {
        const T *row = (const T *)p.job.value + place_any(t);
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int d = (e / EV * 16 + 4 * lq + r) * EV + e % EV;
            const float x = value(row + (d < hd ? d : 0));
            o[e][r] += d < hd && t <= last && !isfinite(x) ? x : 0.0f;
          }
      }
  }
  // vector v's place in out
  auto target = [&](int v) {
    return p.job.out + ((size_t)(it.row0 + v / kv_mul) * p.job.n_heads + (size_t)it.g * kv_mul + v % kv_mul) * hd;
  };
  auto store = [&](float *dst, const float4 &x) {
    if (p.out_vec) {
      *reinterpret_cast<float4 *>(dst) = x;
    } else {
      dst[0] = x.x, dst[1] = x.y, dst[2] = x.z, dst[3] = x.w;
    }
  };
  const bool whole = it.slot < 0;
  const Slot slot = slot_at<HD>(p, max(it.slot, 0));
  float mark = 0.0f;
  constexpr int kFours = E / 4; // a lane's r-th row: kFours groups of four dimensions
  const float l = four_sum(l_run), inverse = 1.0f / l;
  if (it.walkers > 1) { // the waves' sums meet in LDS: [wave][vector][HD values, maximum, sum]
    float *dst = lds + (size_t)(wave * 16 + lc) * kRow;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int f = 0; f < kFours; f++) {
        const int e = 4 * f, d = (e / EV * 16 + 4 * lq + r) * EV + e % EV;
        *reinterpret_cast<float4 *>(dst + d) = float4{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
      }
    if (lq == 0)
      dst[HD] = m_run, dst[HD + 1] = l;
    __syncthreads();
    const int hd4 = hd / 4;
    for (int i = tid; i < it.vectors * hd4; i += kThreads) {
      const int v = i / hd4, d4 = i % hd4;
      const float *src = lds + (size_t)(v / 16 * it.walkers * 16 + v % 16) * kRow;
      float m = -FLT_MAX, whole_l = 0.0f;
      for (int w = 0; w < it.walkers; w++)
        m = fmaxf(m, src[(size_t)w * 16 * kRow + HD]);
      float4 sum = float4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int w = 0; w < it.walkers; w++) {
        const float *at = src + (size_t)w * 16 * kRow;
        const float scale = exp2_far(at[HD] - m);
        const float4 x = *reinterpret_cast<const float4 *>(at + 4 * d4);
        whole_l = fmaf(scale, at[HD + 1], whole_l);
        sum = float4{fmaf(scale, x.x, sum.x), fmaf(scale, x.y, sum.y), fmaf(scale, x.z, sum.z), fmaf(scale, x.w, sum.w)};
      }
      if (whole) {
        const float4 x = float4{sum.x / whole_l, sum.y / whole_l, sum.z / whole_l, sum.w / whole_l};
        mark = mark_of(x, mark);
        store(target(v) + 4 * d4, x);
      } else {
        put4(slot, (unsigned)(v * (HD / 4) + d4), sum);
        if (d4 == 0)
          put_end(slot, v, m, whole_l);
      }
    }
  } else if (mine > 0) { // uniform
    if (!whole && lq == 0 && active)
      put_end(slot, v0 + lc, m_run, l);
    mark = store_rows<HD, EV>(p, slot, whole, o, inverse, lds + (size_t)wave * 16 * kRow, lane, hd, v0, mine, target);
  }
  return mark;
}

// A tile of more than 64 vectors over BF16 pages: each wave has 32 of them and takes all positions. A step's K and V rows are
// loaded once for the block, V turned on the way, and staged in LDS as the instructions take them: a K row's 16 bytes and a V
// operand's serve six instructions each (three parts of two sets of 16 vectors).
template <int HD> struct WideStage {
  static constexpr int kKRow = HD + 8; // values: a row's 16 bytes lie four banks behind the row before's
  uint16_t k[kStep * kKRow];
  v4u v[HD / 16][kWave]; // [instruction][lane]: eight positions of a dimension
};
template <int HD, int MODE> __device__ float walk_wide(const FastPaged &p, const Item &it, float *lds) {
  typedef WideStage<HD> Stage;
  static_assert(2 * sizeof(Stage) <= kWaves * 16 * (HD + 4) * sizeof(float), "two stages in the sums' place");
  Stage *const stages = reinterpret_cast<Stage *>(lds); // two: a step is staged while the one before is computed
  constexpr int E = HD / 16, EV = E, kSteps = HD / 32, kRow = HD + 4, NT = 2;
  constexpr int kKLanes = HD / 8, kKLoads = kStep * kKLanes / kThreads; // lanes of a K row, loads a thread
  static_assert(kKLoads >= 1 && kThreads / kKLanes % 16 == 0, "a K load's rows in one tile of 16");
  const PagedDev &b = p.job.batch;
  const int tid = own_thread(), lane = tid & (kWave - 1), wave = uniform(tid / kWave), lq = lane >> 4, lc = lane & 15;
  const int hd = MODE == kWhole ? HD : p.job.head_dim, kv_mul = p.kv_mul;
  const int v0 = wave * 16 * NT, mine = min(it.vectors - v0, 16 * NT);
  const int all_see = it.last0 + 1;                          // positions below are seen by all of the tile's vectors
  const int wave_sees = it.last0 + v0 / kv_mul + 1;          // by the wave's
  const int end = it.t1;
  int last[NT];
  v4f o[NT][E];
  float m_run[NT], l_run[NT], odd = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; n++) {
    last[n] = 16 * n + lc < mine ? it.last0 + (v0 + 16 * n + lc) / kv_mul : -1;
    m_run[n] = -FLT_MAX, l_run[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++)
      o[n][e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const size_t head = (size_t)it.g * b.head_base;
  long long places = 0; // as in walk, of 32 steps
  auto look_up = [&](int pos) {
    const int at = min(pos + 16 * lane, end - 1), number = at / b.page_size, page = page_of(b, it.r, number);
    if (page < 0)
      p.flags[8] = 1;
    places = (long long)(((size_t)max(page, 0) * b.page_values + (size_t)((at - number * b.page_size) & ~15) * b.pos_stride +
                          head) * sizeof(uint16_t));
  };
  const unsigned row_bytes = (unsigned)b.pos_stride * 2u;
  // 16 rows, tile t of the step at pos, the i-th since look_up
  auto rows_at = [&](const void *cache, int pos, int i, int t) {
    const int at = min(2 * i + t, kWave - 1);
    const int lo = __builtin_amdgcn_readlane((int)places, at), hi = __builtin_amdgcn_readlane((int)(places >> 32), at);
    const int rows = min(end - (pos + 16 * t), 16);
    const int bytes = rows > 0 ? (int)((unsigned)(rows - 1) * row_bytes + (unsigned)(hd * 2)) : 0;
    return rows_of(cache, (long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo), bytes);
  };
  // a thread's K values: row tid / kKLanes of every 256 / kKLanes, dimensions 8 (tid % kKLanes) ..; its V values: dimensions
  // EV lc .. of positions j = 2 wave, 2 wave + 1 of its lane group's eight
  v4u kr[kKLoads];
  unsigned vr[2][EV / 2];
  const int k_dim = 8 * (tid % kKLanes), k_row = tid / kKLanes;
  const unsigned k_at = k_dim < hd ? (unsigned)(k_row % 16) * row_bytes + (unsigned)k_dim * 2u : kNowhere;
  const unsigned v_at = EV * lc < hd ? (unsigned)(4 * lq + 2 * (wave & 1)) * row_bytes + (unsigned)(EV * lc) * 2u : kNowhere;
  auto place_any = [&](int t) { // as in walk
    const int at = min(t, end - 1), number = at / b.page_size, page = page_of(b, it.r, number);
    if (page < 0)
      p.flags[8] = 1;
    return (size_t)max(page, 0) * b.page_values + (size_t)(at - number * b.page_size) * b.pos_stride + head;
  };
  auto load = [&](int pos, int i) {
    if constexpr (MODE == kAny) {
      const int k_dims = k_dim < hd ? k_dim : 0, v_dims = EV * lc < hd ? EV * lc : 0; // there Q is zero, or nothing is stored
#pragma unroll
      for (int u = 0; u < kKLoads; u++)
        kr[u] = *reinterpret_cast<const v4u *>((const uint16_t *)p.job.key + place_any(pos + k_row + u * (kThreads / kKLanes)) + k_dims);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int t = pos + 16 * (wave / 2) + 4 * lq + 2 * (wave & 1) + j;
        const uint16_t *row = (const uint16_t *)p.job.value + place_any(t) + v_dims;
        if constexpr (EV == 8) {
          const v4u x = *reinterpret_cast<const v4u *>(row);
#pragma unroll
          for (int c = 0; c < 4; c++)
            vr[j][c] = t < end ? x[c] : 0u;
        } else {
          const v2u x = *reinterpret_cast<const v2u *>(row);
#pragma unroll
          for (int c = 0; c < 2; c++)
            vr[j][c] = t < end ? x[c] : 0u;
        }
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < kKLoads; u++)
      kr[u] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(
                                          rows_at(p.job.key, pos, i, kKLoads > 1 ? u : uniform(k_row / 16)), k_at, 0, 0));
    const auto rsrc = rows_at(p.job.value, pos, i, wave / 2);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const unsigned at = v_at == kNowhere ? kNowhere : v_at + (unsigned)j * row_bytes;
      if constexpr (EV == 8) {
        const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
#pragma unroll
        for (int c = 0; c < 4; c++)
          vr[j][c] = x[c];
      } else {
        const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, 0));
#pragma unroll
        for (int c = 0; c < 2; c++)
          vr[j][c] = x[c];
      }
    }
  };
  unsigned odd_values = 0;
  auto stage = [&](Stage &sh, int pos) {
#pragma unroll
    for (int u = 0; u < kKLoads; u++)
      *reinterpret_cast<v4u *>(&sh.k[(k_row + u * (kThreads / kKLanes)) * Stage::kKRow + k_dim]) = kr[u];
    if (pos + kStep > all_see) { // as in walk: a value that is not finite is added behind it
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int c = 0; c < EV / 2; c++) {
          const unsigned carry = ((vr[j][c] & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u;
          odd_values |= carry;
          vr[j][c] &= ~((carry << 16) - carry);
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++)
      reinterpret_cast<unsigned *>(&sh.v[e][lane])[wave] =
          __builtin_amdgcn_perm(vr[1][e / 2], vr[0][e / 2], e % 2 ? 0x07060302 : 0x05040100);
  };
  int i = 0; // the number since look_up of the step that is loaded next
  v4u qp[NT][kSteps][3];
  {
    float x[NT][kSteps][8]; // on their way with the first step's rows
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int v = 16 * n + lc < mine ? v0 + 16 * n + lc : 0;
      const float *src = p.job.q + (size_t)(it.row0 + v / kv_mul) * p.job.q_stride + ((size_t)it.g * kv_mul + v % kv_mul) * hd;
#pragma unroll
      for (int s = 0; s < kSteps; s++) {
        const int d = 32 * s + 8 * lq;
        const float *at = src + (d < hd ? d : 0);
        if (p.q_vec) {
          const float4 a = reinterpret_cast<const float4 *>(at)[0], c = reinterpret_cast<const float4 *>(at)[1];
          x[n][s][0] = a.x, x[n][s][1] = a.y, x[n][s][2] = a.z, x[n][s][3] = a.w;
          x[n][s][4] = c.x, x[n][s][5] = c.y, x[n][s][6] = c.z, x[n][s][7] = c.w;
        } else {
#pragma unroll
          for (int c = 0; c < 8; c++)
            x[n][s][c] = at[c];
        }
      }
    }
    if constexpr (MODE != kAny)
      look_up(it.t0);
    load(it.t0, i++);
    fence();
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int s = 0; s < kSteps; s++) {
        const bool there = 16 * n + lc < mine && 32 * s + 8 * lq < hd;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          unsigned part[3];
          bf16_parts(there ? x[n][s][2 * c] * p.scale2 : 0.0f, there ? x[n][s][2 * c + 1] * p.scale2 : 0.0f, part);
#pragma unroll
          for (int k = 0; k < 3; k++)
            qp[n][s][k][c] = part[k];
        }
      }
  }
  stage(stages[0], it.t0);
  load(it.t0 + kStep, i++);
  int turn = 0;
  constexpr int kAheadK = 4 < 2 * kSteps ? 4 : 2 * kSteps, kAheadV = 2;
  for (int pos = it.t0; pos < end; pos += kStep, turn ^= 1) {
    const Stage &sh = stages[turn];
    __syncthreads(); // the step is staged, the one before it computed
    v4f sc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int t = 0; t < 2; t++)
        sc[n][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // each operand is read four (two) uses ahead: left to itself the compiler reads one, waits for it and uses it
    v4u a[2 * kSteps];
    auto read_k = [&](int i) {
      a[i] = *reinterpret_cast<const v4u *>(&sh.k[(16 * (i % 2) + lc) * Stage::kKRow + 32 * (i / 2) + 8 * lq]);
    };
#pragma unroll
    for (int i = 0; i < kAheadK; i++)
      read_k(i);
    fence();
#pragma unroll
    for (int i = 0; i < 2 * kSteps; i++) {
      if (i + kAheadK < 2 * kSteps)
        read_k(i + kAheadK);
#pragma unroll
      for (int k = 2; k >= 0; k--)
#pragma unroll
        for (int n = 0; n < NT; n++)
          sc[n][i % 2] = mfma_bf16(a[i], qp[n][i / 2][k], sc[n][i % 2]);
      fence();
    }
    stage(stages[turn ^ 1], pos + kStep);
    if (MODE != kAny && i == kWave / 2) { // uniform
      look_up(pos + 2 * kStep);
      i = 0;
    }
    load(pos + 2 * kStep, i++);
    v4u wp[NT][3];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float w[8], top = -FLT_MAX;
#pragma unroll
      for (int j = 0; j < 8; j++)
        w[j] = sc[n][j / 4][j % 4];
      if (pos + kStep > wave_sees || pos + kStep > end || mine < 16 * NT) { // a lane without a vector sees nothing
        const int seen = min(last[n], end - 1) - pos - 4 * lq;
#pragma unroll
        for (int j = 0; j < 8; j++)
          w[j] = 16 * (j / 4) + j % 4 <= seen ? w[j] : -FLT_MAX;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        odd = fmaf(w[j], 0.0f, odd);
        top = fmaxf(top, w[j]);
      }
      if (__any(top > m_run[n] + 8.0f)) { // as in walk
        const float m = fmaxf(m_run[n], four_max(top)), alpha = exp2_far(m_run[n] - m);
        l_run[n] *= alpha;
        m_run[n] = m;
#pragma unroll
        for (int e = 0; e < E; e++)
          o[n][e] *= alpha;
      }
      const float base = m_run[n] > -FLT_MAX ? m_run[n] : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        w[j] = __builtin_amdgcn_exp2f(w[j] - base);
        l_run[n] += w[j];
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        unsigned part[3];
        bf16_parts(w[2 * c], w[2 * c + 1], part);
#pragma unroll
        for (int k = 0; k < 3; k++)
          wp[n][k][c] = part[k];
      }
    }
    v4u v[E];
#pragma unroll
    for (int e = 0; e < kAheadV; e++)
      v[e] = sh.v[e][lane];
    fence();
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (e + kAheadV < E)
        v[e + kAheadV] = sh.v[e + kAheadV][lane];
#pragma unroll
      for (int k = 2; k >= 0; k--)
#pragma unroll
        for (int n = 0; n < NT; n++)
          o[n][e] = mfma_bf16(v[e], wp[n][k], o[n][e]);
      fence();
    }
  }
  if (odd != 0.0f)
    p.flags[1] = 1;
  if (__syncthreads_or(odd_values != 0)) {
    for (int t = it.t0 + (max(all_see - it.t0, 0) & ~(kStep - 1)); t < end; t++) { // of the steps that some do not see whole
      const int number = t / b.page_size, page = max(page_of(b, it.r, number), 0);
      const uint16_t *row = (const uint16_t *)p.job.value + (size_t)page * b.page_values +
                            (size_t)(t - number * b.page_size) * b.pos_stride + head;
#pragma unroll
      for (int e = 0; e < E; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int d = (4 * lq + r) * EV + e;
          const float x = value(row + (d < hd ? d : 0));
#pragma unroll
          for (int n = 0; n < NT; n++)
            o[n][e][r] += d < hd && t <= last[n] && !isfinite(x) ? x : 0.0f;
        }
    }
  }
  const bool whole = it.slot < 0;
  const Slot slot = slot_at<HD>(p, max(it.slot, 0));
  __syncthreads(); // the stages' place is free
  float mark = 0.0f;
  auto target = [&](int v) {
    return p.job.out + ((size_t)(it.row0 + v / kv_mul) * p.job.n_heads + (size_t)it.g * kv_mul + v % kv_mul) * hd;
  };
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const float l = four_sum(l_run[n]), inverse = 1.0f / l;
    if (16 * n >= mine)
      continue; // uniform
    if (!whole && lq == 0 && 16 * n + lc < mine)
      put_end(slot, v0 + 16 * n + lc, m_run[n], l);
    mark += store_rows<HD, EV>(p, slot, whole, o[n], inverse, lds + (size_t)wave * 16 * kRow, lane, hd, v0 + 16 * n,
                               min(mine - 16 * n, 16), target);
  }
  return mark;
}

// A tile that gave out something not finite: each of its rows gets what its positions' values hold, in the dimensions where
// one is not finite. Threads (share, dimension), the shares' positions interleaved; LDS free before and behind.
template <typename T> __device__ __forceinline__ void give_odd(const FastPaged &p, const Item &it, float *lds) {
  const PagedDev &b = p.job.batch;
  const int tid = threadIdx.x, hd = p.job.head_dim, shares = kThreads / hd, share = tid / hd, d = tid % hd;
  auto at = [&](int t) {
    const int page = max(page_of(b, it.r, t / b.page_size), 0);
    return odd_only(value((const T *)p.job.value + (size_t)page * b.page_values + (size_t)(t % b.page_size) * b.pos_stride +
                          (size_t)it.g * b.head_base + d));
  };
  float odd = 0.0f;
  if (share < shares)
    for (int t = share; t <= it.last0; t += 8 * shares) { // eight on their way at once; the last one again does no harm
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        x[i] = at(min(t + i * shares, it.last0));
#pragma unroll
      for (int i = 0; i < 8; i++)
        odd += x[i];
    }
  lds[tid] = odd;
  __syncthreads();
  if (share == 0) {
    for (int s = 1; s < shares; s++)
      odd += lds[s * hd + d];
    for (int j = 0; j < it.vectors / p.kv_mul; j++) {
      odd += j ? at(it.last0 + j) : 0.0f;
      for (int h = 0; h < p.kv_mul && odd != 0.0f; h++)
        p.job.out[((size_t)(it.row0 + j) * p.job.n_heads + (size_t)it.g * p.kv_mul + h) * hd + d] = odd;
    }
  }
  __syncthreads();
}

// A block's part of a walk with what of the line its join needs.
struct Part {
  Item it;
  long long w0, end; // where the walk begins and ends on the line
  int begin, unit, grain;
  bool shared, begins; // with other blocks; in this one's slice
};
// The parts of the line's lo .. hi - 1, in order.
template <class Visit>
__device__ __forceinline__ void each_part(const FastPaged &p, const Plan &plan, int g, long long lo, long long hi, Visit visit) {
  const PagedDev &b = p.job.batch;
  const int kv_mul = p.kv_mul;
  int r = 0; // the first request whose walks end behind lo
  for (int step = kMaxRequests; step > 0; step >>= 1)
    if (r + step <= b.count && plan.line[r + step - 1] <= lo)
      r += step;
  for (long long base = r ? plan.line[r - 1] : 0; r < b.count && base < hi; base = plan.line[r], r++) {
    bool bad = false;
    const PagedRequest q = paged_request(b, r, bad);
    if (q.rows == 0)
      continue;
    const int tiles = ceil_div(q.rows, p.tile_rows);
    int t = 0; // the last tile that begins at or before lo
    if (base < lo)
      for (int step = 1 << 20; step > 0; step >>= 1)
        if (t + step < tiles && base + tile_start(p, q.length, t + step) <= lo)
          t += step;
    for (; t < tiles; t++) {
      const long long w0 = base + tile_start(p, q.length, t);
      if (w0 >= hi)
        break;
      const int row = t * p.tile_rows, rows = min(q.rows - row, p.tile_rows);
      const int positions = q.length + row + rows;
      Part part;
      Item &it = part.it;
      it.vectors = rows * kv_mul;
      it.walkers = walkers_of(it.vectors);
      const int begin = begin_time(it.vectors), unit = position_time(it.vectors), grain = it.walkers * kStep;
      const long long end = w0 + begin + (long long)unit * positions;
      // the position that lies at x of the line, in whole rounds
      auto position_at = [&](long long x) {
        if (x >= end)
          return positions;
        const int at = x <= w0 + begin ? 0 : (int)((x - w0 - begin) / unit);
        return min(at / grain * grain, positions);
      };
      it.t0 = w0 >= lo ? 0 : position_at(lo);
      it.t1 = position_at(hi);
      if (it.t0 >= it.t1)
        continue; // the rounds leave this block none of it
      it.r = r, it.g = g;
      it.row0 = q.first + row, it.last0 = q.length + row;
      part.w0 = w0, part.end = end, part.begin = begin, part.unit = unit, part.grain = grain;
      part.shared = it.t0 > 0 || it.t1 < positions;
      part.begins = w0 >= lo;
      visit(part);
    }
  }
}

template <typename T, int HD, int MODE, bool WIDE>
__global__ __launch_bounds__(kThreads, HD > 128 ? 1 : kMaxBlocksPerCu) void attn_paged(FastPaged p) {
  constexpr int kRow = HD + 4;
  __shared__ Plan plan;
  __shared__ __align__(16) float lds[kWaves * 16 * kRow];
  __shared__ unsigned arrived;
  // which parts' results, as this block gave them out, are not all finite: 1 those of a walk that is its own, 2 those of one
  // that an earlier block began, 4 those of one that goes on in the next
  __shared__ unsigned odd;
  if (threadIdx.x == 0)
    odd = 0;
  const int tid = threadIdx.x, g = blockIdx.x % p.job.n_kv_heads, block = blockIdx.x / p.job.n_kv_heads;
  const int hd = p.job.head_dim, kv_mul = p.kv_mul;
  const long long total = make_plan(p, plan);
  const Slices slices = make_slices(p, total);
  const long long lo = slices.start(block), hi = slices.start(block + 1) < total ? slices.start(block + 1) : total;
  if (lo >= total)
    return;
  each_part(p, plan, g, lo, hi, [&](Part &mine) {
    Item &it = mine.it;
    auto slot_of = [&](int blk, bool begins) { return (g * p.blocks + blk) * 2 + begins; };
    it.slot = uniform(mine.shared ? slot_of(block, mine.begins) : -1);
    __syncthreads(); // LDS is free
    float mark;
    if constexpr (WIDE) {
      if (it.vectors > kTileVectors)
        mark = walk_wide<HD, MODE>(p, it, lds);
      else
        mark = walk<T, HD, MODE>(p, it, lds);
    } else {
      mark = walk<T, HD, MODE>(p, it, lds);
    }
    if (!mine.shared) {
      if (mark != 0.0f)
        atomicOr(&odd, 1u);
      return;
    }
    const long long w0 = mine.w0, end = mine.end;
    const int begin = mine.begin, unit = mine.unit, grain = mine.grain;
    // the walk's blocks: from .. last_block
    const int first = slices.block_of(w0), last_block = slices.block_of(end - 1);
    // the first block whose slice ends behind the walk's first round
    const int from = min(max(first, slices.block_of(w0 + begin + unit * grain - 1)), last_block), parts = last_block - from + 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the thread's sums have arrived
    __syncthreads();                                 // the block's
    if (tid == 0)
      arrived = __hip_atomic_fetch_add(&paged_arrivals[(g * p.blocks + first) * kLine], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != (unsigned)(parts - 1))
      return;
    if (tid == 0)
      __hip_atomic_store(&paged_arrivals[(g * p.blocks + first) * kLine], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The parts of some vectors at a time: each part's share of the vector's sums, exp2(m - the largest) / the whole l, into
    // LDS, then the sums in the parts' order, whoever comes last. A part's place by its number.
    auto part = [&](int k) { return slot_at<HD>(p, slot_of(from + k, from + k == first)); };
    const int hd4 = hd / 4, some = kWaves * 16 * kRow / parts;
    mark = 0.0f;
    for (int v0 = 0; v0 < it.vectors; v0 += some) {
      const int n = min(some, it.vectors - v0), items = n * hd4;
      __syncthreads(); // LDS is free
      constexpr int kFew = 8;
      if (parts <= kFew) { // a thread a vector, its loads together
        for (int v = tid; v < n; v += kThreads) {
          float2 x[kFew];
#pragma unroll
          for (int k = 0; k < kFew; k++)
            x[k] = load_end(p, slot_of(from + min(k, parts - 1), from + min(k, parts - 1) == first), v0 + v, HD);
          float m = -FLT_MAX, l = 0.0f;
#pragma unroll
          for (int k = 0; k < kFew; k++)
            m = fmaxf(m, x[k].x);
#pragma unroll
          for (int k = 0; k < kFew; k++) {
            x[k].x = exp2_far(x[k].x - m);
            l = k < parts ? fmaf(x[k].x, x[k].y, l) : l;
          }
          const float inverse = 1.0f / l;
#pragma unroll
          for (int k = 0; k < kFew; k++)
            if (k < parts)
              lds[v * parts + k] = x[k].x * inverse;
        }
      } else {
        for (int v = tid / kWave; v < n; v += kWaves) {
          float m = -FLT_MAX, l = 0.0f;
          for (int k = tid % kWave; k < parts; k += kWave) {
            const float2 end_of = load_end(p, slot_of(from + k, from + k == first), v0 + v, HD);
            lds[v * parts + k] = end_of.x;
            const float top = fmaxf(m, end_of.x);
            l = l * __builtin_amdgcn_exp2f(m - top) + end_of.y * __builtin_amdgcn_exp2f(end_of.x - top);
            m = top;
          }
          const float top = wave_max(m), inverse = 1.0f / wave_sum(l * __builtin_amdgcn_exp2f(m - top));
          for (int k = tid % kWave; k < parts; k += kWave)
            lds[v * parts + k] = exp2_far(lds[v * parts + k] - top) * inverse;
        }
      }
      __syncthreads();
      // I of the thread's items and K parts at a time: as many loads are in flight
      auto add_up = [&](auto of_items, auto of_parts) {
        constexpr int I = decltype(of_items)::value, K = decltype(of_parts)::value;
        for (int i0 = tid; i0 < items; i0 += I * kThreads) {
          int v[I], d[I];
          unsigned at[I];
          float4 sum[I];
#pragma unroll
          for (int j = 0; j < I; j++) {
            const int i = i0 + j * kThreads;
            v[j] = i / hd4, d[j] = i % hd4 * 4;
            at[j] = (unsigned)((v0 + v[j]) * (HD / 4) + d[j] / 4);
            if (i >= items)
              v[j] = 0, d[j] = -1, at[j] = kNowhere / 16; // reads zero
            sum[j] = float4{0.0f, 0.0f, 0.0f, 0.0f};
          }
          for (int k0 = 0; k0 < parts; k0 += K) {
            float4 x[K][I];
#pragma unroll
            for (int k = 0; k < K; k++) {
              const Slot slot = part(min(k0 + k, parts - 1));
#pragma unroll
              for (int j = 0; j < I; j++)
                x[k][j] = get4(slot, k0 + k < parts ? at[j] : kNowhere / 16);
            }
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
              for (int j = 0; j < I; j++) {
                const float scale = lds[v[j] * parts + min(k0 + k, parts - 1)];
                sum[j] = float4{fmaf(scale, x[k][j].x, sum[j].x), fmaf(scale, x[k][j].y, sum[j].y),
                                fmaf(scale, x[k][j].z, sum[j].z), fmaf(scale, x[k][j].w, sum[j].w)};
              }
          }
#pragma unroll
          for (int j = 0; j < I; j++)
            if (d[j] >= 0) {
              mark = mark_of(sum[j], mark);
              const int vector = v0 + v[j];
              float *to = p.job.out + ((size_t)(it.row0 + vector / kv_mul) * p.job.n_heads + (size_t)g * kv_mul + vector % kv_mul) * hd + d[j];
              if (p.out_vec)
                *reinterpret_cast<float4 *>(to) = sum[j];
              else
                to[0] = sum[j].x, to[1] = sum[j].y, to[2] = sum[j].z, to[3] = sum[j].w;
            }
        }
      };
      if (items > 2 * kThreads)
        add_up(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
      else if (parts > 16 && items <= kThreads)
        add_up(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
      else if (parts > 4)
        add_up(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
      else
        add_up(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
    }
    if (mark != 0.0f)
      atomicOr(&odd, mine.begins ? 4u : 2u);
  });
  // What is not finite is looked for behind all parts, rare as it is: inside the loop its registers cost one F32 row at 35000
  // positions 73 us instead of 70. The flags are written, by a barrier that does not wait for the rows' stores.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  if (__builtin_expect(odd != 0, 0)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the thread's rows are stored
    __syncthreads();                                 // the block's
    each_part(p, plan, g, lo, hi, [&](Part &mine) {
      if (odd & (mine.shared ? mine.begins ? 4u : 2u : 1u))
        give_odd<T>(p, mine.it, lds);
    });
  }
}

int tile_dims(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// The matrix-core form takes the job: K and V rows in whole 16-byte vectors, offsets within 16 rows of 32 bits, positions
// within int arithmetic of the steps, and a line below 2^50.
bool tiled(const AttentionPagedJob &job) {
  const size_t size = job.batch.bf16 ? 2 : 4;
  return job.head_dim * size % 16 == 0 && (((uintptr_t)job.key | (uintptr_t)job.value) & 15) == 0 &&
         job.batch.pos_stride * size * 16 < ((size_t)1 << 30) && job.batch.seq_len < (1 << 30) && job.batch.rows <= (1 << 20) && job.n_kv_heads <= kMaxArrivals;
}

int blocks_of(const AttentionPagedJob &job) {
  const int all = (job.head_dim > 128 ? 1 : kMaxBlocksPerCu) * device().cu_count, cap = kMaxArrivals / job.n_kv_heads;
  const int n = all / job.n_kv_heads;
  return n < 1 ? 1 : n < cap ? n : cap;
}

typedef void (*FastKernel)(FastPaged);
template <typename T, int HD> FastKernel kernel_of(int mode, bool wide) {
  if constexpr (sizeof(T) == 2 && HD <= 128)
    if (wide)
      return mode == kWhole  ? attn_paged<T, HD, kWhole, true>
             : mode == kPart ? attn_paged<T, HD, kPart, true>
                             : attn_paged<T, HD, kAny, true>;
  return mode == kWhole  ? attn_paged<T, HD, kWhole, false>
         : mode == kPart ? attn_paged<T, HD, kPart, false>
                         : attn_paged<T, HD, kAny, false>;
}
template <typename T> FastKernel kernel_of(int dims, int mode, bool wide) {
  return dims == 64 ? kernel_of<T, 64>(mode, wide) : dims == 128 ? kernel_of<T, 128>(mode, wide) : kernel_of<T, 256>(mode, wide);
}

// Blocks of a KV head that the batch may need, whatever its arrays hold: a small one's are fewer than fill the device.
int blocks_for(const AttentionPagedJob &job, int tile_rows) {
  const long long rows = job.batch.rows, count = job.batch.count;
  const long long tiles = (rows + tile_rows - 1) / tile_rows + (rows < count ? rows : count);
  const long long line = tiles * (kWideBegin + kMostTime * (long long)job.batch.seq_len);
  const int all = blocks_of(job);
  return line / kMinSlice < all ? (int)(line / kMinSlice) + 1 : all;
}

int mode_of(const AttentionPagedJob &job) {
  return job.batch.page_size % 16 ? kAny : job.head_dim == tile_dims(job.head_dim) ? kWhole : kPart;
}

// The kernel with wide tiles, where some request may have more than 64 vectors.
bool wide_tiles(const AttentionPagedJob &job) {
  const long long vectors = (long long)job.batch.rows * (job.n_heads / job.n_kv_heads);
  return job.batch.bf16 && job.head_dim <= 128 && job.batch.rows > job.batch.count && vectors > kTileVectors;
}

bool launch_rows(const AttentionPagedJob &job, hipStream_t stream) {
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

} // namespace

size_t attention_paged_workspace(const AttentionPagedJob &job) {
  if (!tiled(job))
    return 0;
  return (size_t)job.n_kv_heads * blocks_of(job) * 2 * (wide_tiles(job) ? kWideVectors : kTileVectors) *
         (tile_dims(job.head_dim) + 2) * sizeof(float);
}

bool launch_attention_paged(const AttentionPagedJob &job, void *workspace, hipStream_t stream) {
  if (!tiled(job))
    return launch_rows(job, stream);
  const int dims = tile_dims(job.head_dim);
  FastPaged p{};
  p.job = job;
  p.kv_mul = job.n_heads / job.n_kv_heads;
  const bool wide = wide_tiles(job);
  p.tile_vectors = wide ? kWideVectors : kTileVectors;
  p.tile_rows = p.tile_vectors / p.kv_mul;
  p.full_begin = wide ? kWideBegin : kBegin;
  p.full_position = wide ? kWidePosition : kWaves / (p.tile_rows * p.kv_mul <= 16 ? 4 : p.tile_rows * p.kv_mul <= 32 ? 2 : 1);
  p.blocks = blocks_for(job, p.tile_rows);
  p.pairs = wide && p.blocks % 2 == 0 && p.blocks * job.n_kv_heads == kMaxBlocksPerCu * device().cu_count;
  p.scale2 = (float)(1.4426950408889634 / sqrt((double)job.head_dim));
  p.partial = (float *)workspace;
  p.flags = device().error_flags;
  p.fours = job.batch.page_size % 4 == 0;
  p.q_vec = job.q_stride % 4 == 0 && ((uintptr_t)job.q & 15) == 0;
  p.out_vec = ((uintptr_t)job.out & 15) == 0;
  const int mode = mode_of(job);
  const FastKernel kernel = job.batch.bf16 ? kernel_of<uint16_t>(dims, mode, wide) : kernel_of<float>(dims, mode, false);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(p.blocks * job.n_kv_heads)), dim3(kThreads), 0, stream, p);
  return launch_ok("attn_paged");
}

} // namespace llhip
