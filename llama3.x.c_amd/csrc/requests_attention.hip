// Attention of many requests behind a prefix that all of them share (gfx950).
//
//   attn_requests        block: a slice of a KV head's walks, a walk being a tile of query vectors over the prefix (all
//                        requests' rows together, so that the prefix is read once a tile) or over a request's own
//                        positions. One pass over K and V with the softmax's running maximum and sum; 128 vectors a wide
//                        tile, whose products are FP16 parts on the matrix cores, up to 32 a narrow one, with FP32 products.
//   attn_requests_merge  a row's partial sums, rescaled to their largest maximum.
//   attn_rows            any shape, one row at a time: 32 rows of 8 heads over 4 KV heads of 256 behind 2048 positions take
//                        2.4 ms, where their K and V once would take 24 us.
//
// Measured at 32 heads over 8 KV heads of dimension 128, both launches: 32 requests of one row behind 2048 positions, 502 own
// ones on average, 48 us (148 MB of K and V: 3.1 TB/s); 64 behind 8192 with 594 99 us (378 MB: 3.8 TB/s); 16 with two to
// seven rows behind 4096 with 916 65 us; five prompts, 923 rows, behind 1024 93 us. With 32 heads over 8 of 64: the 32 rows
// 27.6 us, the 16 requests' drafts 42, the prompts 94. Wide walks are bound by their
// instructions: a step takes the two waves of a SIMD 5600 cycles, 4300 of vector and 3100 of matrix instructions, which overlap
// little (over the whole kernel the vector unit is 50% busy, the matrix cores 30%, LDS less); narrow ones by HBM.
#include <cfloat>
#include <type_traits>

#include "requests_device.h"

#include "lanes.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

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

// ---- the matrix-core form ---------------------------------------------------------------------------------------------

constexpr int kUnit = 32;         // positions of a step
constexpr int kTileVectors = 128; // query vectors of a wide tile
// At most, of a narrow one: 16 requests with 8 to 28 vectors take 65.9 us (with 16: 67.4, their wide tiles mostly empty),
// requests of four vectors the same; FP32 products for more than 32 would take longer than the wide tile's.
constexpr int kNarrowVectors = 32;
constexpr int kBlocksPerCu = 2; // as LDS and registers allow
constexpr int kTable = 128;     // requests that a block keeps in LDS; it reads the others again
// A block's shortest slice, in WalkTime's units: one row behind 200 positions takes 11.9 us (700: 12.4, 1500: 13.2).
constexpr int kMinSlice = 1024;
constexpr float kMasked = -0x1p126f; // a masked score, -FLT_MAX, lies so far below that its weight is zero, also where a
                                     // lane has seen nothing else

// Where a row's partial sums lie: those of its tile over the prefix, and over its own positions, by the blocks first ..
// last that took the tile's walk.
struct RowSlots {
  int prefix_first, prefix_last, prefix_v;
  int own_first, own_last, own_v; // own_first -1: the row belongs to no request
  int slot, last;                 // cache slot and last own position
};

struct FastAttn {
  float *out;
  const float *q, *prefix_key, *prefix_value, *key, *value;
  RequestsDev batch;
  int n_heads, n_kv_heads, kv_mul, hd;
  int tile_rows, narrow_rows; // rows of a wide tile, and at most of a narrow one
  int blocks;                 // of a KV head
  float scale2;               // log2(e) / sqrtf(hd)
  // slots of hd + 4 floats: [prefix, own][row][head] where a walk begins, [KV head][block][vector of the tile] where a
  // block goes on with the walk of the one before
  float *partial;
  RowSlots *rows;
  int *flags;
};

// What every block works out for itself from the batch's arrays. The walks of a KV head (a tile of query vectors over the
// prefix, or over a request's own positions) lie one behind the other on a line, each as long as it takes in time, and
// the line is cut into slices of one length, one for a block: all blocks start together and end together. (Walks cut into
// about equal shares of their own, one to a block, left a third of the blocks' time idle behind the first round.)
struct Plan {
  long long line[kMaxRequests]; // where request r's own walks end
  long long prefix, full;       // the prefix's part of the line, and of one full tile in it
  long long slice, total;
  int total_rows, first_row, end_row; // of the requests: their rows' number, the lowest, one past the highest
  long long wave_sum[kThreads / kWave];
  Request table[kTable]; // the first requests, for the blocks' walks
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// How long a walk over so many positions takes a block, two of them on a CU, in units of 8.6 ns: 1.1 us for 32 positions
// with up to 16 vectors, 1.9 with up to 32 (two waves walk a tile instead of four), 3.3 to 4 in a wide tile, and 6 to 10 us
// to begin and end.
struct WalkTime {
  int begin, position;
};
__device__ __host__ __forceinline__ constexpr WalkTime walk_time_of(int vectors) {
  return vectors <= 16 ? WalkTime{680, 4} : vectors <= kNarrowVectors ? WalkTime{900, 7} : WalkTime{1120, 12};
}
__device__ __forceinline__ long long walk_time(int vectors, int positions) {
  const WalkTime t = walk_time_of(vectors);
  return t.begin + (long long)t.position * positions;
}
// A request's own walks: one narrow tile, or full wide ones and the rest, tile t over the positions up to its last row's.
__device__ __forceinline__ int own_tiles(const FastAttn &p, int rows) {
  return rows * p.kv_mul <= kNarrowVectors ? 1 : ceil_div(rows, p.tile_rows);
}
__device__ __forceinline__ long long tile_start(const FastAttn &p, int length, long long t) {
  constexpr WalkTime wide = walk_time_of(kTileVectors);
  return t * wide.begin + wide.position * (t * length + p.tile_rows * (t * (t + 1) / 2));
}
__device__ __forceinline__ long long own_time(const FastAttn &p, const Request &q) {
  if (q.rows == 0)
    return 0;
  const int t = own_tiles(p, q.rows) - 1;
  return tile_start(p, q.length, t) + walk_time((q.rows - t * p.tile_rows) * p.kv_mul, q.length + q.rows);
}

// x / y of the line's lengths (below 2^50, where the double quotient's whole part is exact), a third of the time that the
// compiler's division takes.
__device__ __forceinline__ long long whole(long long x, long long y) { return (long long)((double)x / (double)y); }

__device__ void make_plan(const FastAttn &p, Plan &plan) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  constexpr int kPer = kMaxRequests / kThreads; // requests of a thread, at most
  const int per = ceil_div(p.batch.count, kThreads), r0 = tid * per;
  if (tid == 0) { // as the arrays say, if they are right
    plan.first_row = p.batch.start[0];
    plan.end_row = p.batch.start[p.batch.count];
    plan.total_rows = 0;
  }
  long long sum = 0, time[kPer];
  int total_rows = 0, first_row = p.batch.rows, end_row = 0;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    time[k] = 0;
    if (k < per && r0 + k < p.batch.count) {
      const Request q = request_at(p.batch, r0 + k, bad);
      if (r0 + k < kTable)
        plan.table[r0 + k] = q;
      total_rows = min(total_rows + q.rows, INT32_MAX / kThreads);
      if (q.rows) {
        first_row = min(first_row, q.first);
        end_row = max(end_row, q.first + q.rows);
      }
      sum += time[k] = own_time(p, q);
    }
  }
  long long run = sum; // the threads' up to this one
  for (int o = 1; o < kWave; o <<= 1) {
    const long long v = __shfl_up(run, o);
    if (lane >= o)
      run += v;
  }
  if (lane == kWave - 1)
    plan.wave_sum[wave] = run;
  if (__syncthreads_or(bad)) { // what is left of them
    if (blockIdx.x == 0 && tid == 0)
      p.flags[3] = 1;
    if (tid == 0)
      plan.first_row = p.batch.rows, plan.end_row = 0;
    __syncthreads();
    atomicAdd(&plan.total_rows, total_rows);
    atomicMin(&plan.first_row, first_row);
    atomicMax(&plan.end_row, end_row);
    __syncthreads();
  }
  // requests over each other's rows (and some start above the next, so bad is set): none is taken
  const bool none = plan.total_rows > p.batch.rows;
  const int rows = none || !p.batch.prefix ? 0 : max(plan.end_row - plan.first_row, 0);
  const int tiles = ceil_div(rows, p.tile_rows);
  const long long full = walk_time(p.tile_rows * p.kv_mul, p.batch.prefix);
  const long long prefix =
      tiles ? (tiles - 1) * full + walk_time((rows - (tiles - 1) * p.tile_rows) * p.kv_mul, p.batch.prefix) : 0;
  long long at = prefix + run - sum, total = prefix;
  for (int w = 0; w < kThreads / kWave; w++) {
    if (w < wave)
      at += plan.wave_sum[w];
    total += plan.wave_sum[w];
  }
#pragma unroll
  for (int k = 0; k < kPer; k++)
    if (k < per && r0 + k < p.batch.count)
      plan.line[r0 + k] = none ? 0 : at += time[k];
  if (tid == 0) {
    plan.prefix = prefix;
    plan.full = full;
    plan.total = none ? 0 : total;
    plan.slice = max(whole(total + p.blocks - 1, p.blocks), (long long)kMinSlice);
  }
  __syncthreads();
}

// Query vectors (row row0 + v / kv_mul, head g * kv_mul + v % kv_mul for v < vectors) over positions t0 .. t1 - 1 of one
// cache; row row0 + j sees positions up to last0 + j (the prefix: all).
struct Item {
  const float *key, *value;
  size_t pos_stride;
  int row0, vectors, g;
  int t0, t1;
  int last0; // INT_MAX: every position is seen by every row
  size_t slot0; // vector v's slot is slot0 + (v / kv_mul) * slot_row + v % kv_mul
  int slot_row;
};
__device__ __forceinline__ float *slot_of(const FastAttn &p, const Item &it, int v) {
  return p.partial + (it.slot0 + (size_t)(v / p.kv_mul) * it.slot_row + v % p.kv_mul) * (size_t)(p.hd + 4);
}

// Nothing moves across: each phase's registers are free before the next one's are taken (moved freely, the phases of a
// step need more than the 256 registers that two waves a SIMD leave each).
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long uniform(long long x) {
  return (long long)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

// The thread's number, new to the compiler at each walk: else it keeps what both walks derive from it in registers all along
// a block's walks (43 of them spilled).
__device__ __forceinline__ int own_thread() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The end of a partial sum's slot: maximum (base 2), sum of the weights, and, where the item met a V value that is not
// finite, its positions t0 .. t1 - 1 (else t1 = 0). Such a value must reach exactly the rows that see its position, and 0 *
// infinity would carry it to those that do not; so the products take 0 in its place, and the merge adds it.
__device__ __forceinline__ float4 slot_end(float m, float l, bool met, const Item &it) {
  return float4{m, l, __int_as_float(it.t0), __int_as_float(met ? it.t1 : 0)};
}

__device__ __forceinline__ v4f mfma_f16(const v4i &a, const v4i &b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// x * scale = h + l to 22 bits and more, two FP16 parts, for |x * scale| <= 2^15: two values a dword.
__device__ __forceinline__ void f16_pair(float a, float b, float scale, int &h, int &l) {
  const v2f x = {a * scale, b * scale};
  const v2h hi = __builtin_convertvector(x, v2h);
  const v2f rest = {__builtin_fmaf(a, scale, -(float)hi[0]), __builtin_fmaf(b, scale, -(float)hi[1])};
  h = __builtin_bit_cast(int, hi);
  l = __builtin_bit_cast(int, __builtin_convertvector(rest, v2h));
}

// The power of two that brings values up to `top` to at most 2^15 (top in [2^e, 2^(e+1)): 2^(14 - e)), and e, which is at
// least `least`; top must be finite.
__device__ __forceinline__ float f16_scale(float top, int least, int &e) {
  e = max((int)(__float_as_uint(top) >> 23) - 127, least);
  return __uint_as_float((unsigned)(127 + 14 - e) << 23);
}

// Four values of a query vector, zero past the head's dimensions.
__device__ __forceinline__ float4 load4(const float *row, int d, int hd) {
  return d < hd ? *reinterpret_cast<const float4 *>(row + d) : float4{0.0f, 0.0f, 0.0f, 0.0f};
}

// K or V rows t0 .. t1 - 1 of an item as a buffer: a load past them reads zero, and a row's place is a 32-bit offset that a
// step advances by one addition (a 64-bit address a load took a third of a step's vector instructions).
struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned stride; // bytes
};
__device__ __forceinline__ Rows rows_of(const float *cache, const Item &it, int hd) {
  const uint64_t base = (uint64_t)(uintptr_t)(cache + (size_t)it.t0 * it.pos_stride);
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)base);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(base >> 32));
  const unsigned stride = __builtin_amdgcn_readfirstlane((unsigned)it.pos_stride * 4u);
  const int n = __builtin_amdgcn_readfirstlane(it.t1 - it.t0);
  const int bytes = n > 0 ? (n - 1) * (int)stride + hd * 4 : 0;
  return Rows{__builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)(((uint64_t)hi << 32) | lo), (short)0, bytes, 0x00020000),
              stride};
}
// Dimensions d .. d + 3 at byte offset `at` of its row's start, `rows` rows further; zero past the head's dimensions.
template <bool FULL> __device__ __forceinline__ float4 row4(const Rows &r, unsigned at, int rows, int d, int hd) {
  const unsigned off = at + 4u * (unsigned)d;
  return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r.rsrc, FULL || d < hd ? off : 0x7FFFFFF0u,
                                                                          (unsigned)rows * r.stride, 0));
}

// The largest or the sum of a query vector's four lanes (lane, and 16, 32 and 48 lanes away), on the vector unit.
__device__ __forceinline__ float four_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float four_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Narrow: at most 16 vectors a wave. The four waves walk 32-position steps in turn when the item has one tile of 16
// vectors; with two tiles (or four) each tile has two waves (one) that walk all the steps, the rows that another wave has
// read coming from the caches. K and V rows go straight into registers in the order the matrix instructions take them,
// with no copy in LDS, and the waves' sums meet at the end. The products are FP32 ones on the matrix cores, the cheapest
// form where a K or V value meets so few vectors: the 128 instructions of a step take 4096 cycles, while BF16 parts take
// 1536 and 3800 on the vector unit to split the values.
template <int HD, bool FULL> __device__ void walk_narrow(const FastAttn &p, const Item &it, unsigned char *lds) {
  constexpr int kSteps = HD / 32, kDt = HD / 16, kWaves = kThreads / kWave, kRow = HD + 4;
  const int tid = own_thread(), lane = tid & (kWave - 1), wave = tid / kWave, lq = lane >> 4, lc = lane & 15;
  const int hd = p.hd;
  const int tiles = it.vectors <= 16 ? 1 : 2, walkers = kWaves / tiles; // waves of a tile
  const int v_mine = 16 * (wave / walkers) + lc; // this lane's vector
  const bool active = v_mine < it.vectors;
  float4 x[kSteps][2]; // dimensions 32 st + 8 lq .. + 7, on their way with the first step's rows
  const float *src = p.q + ((size_t)(it.row0 + (active ? v_mine / p.kv_mul : 0)) * p.n_heads + (size_t)it.g * p.kv_mul +
                            (active ? v_mine % p.kv_mul : 0)) * hd;
#pragma unroll
  for (int st = 0; st < kSteps; st++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int d = 32 * st + 8 * lq + 4 * h;
      x[st][h] = *reinterpret_cast<const float4 *>(src + (FULL || d < hd ? d : 0));
    }
  fence();
  const int last = !active ? -1 : it.last0 == INT32_MAX ? INT32_MAX : it.last0 + v_mine / p.kv_mul;
  v4f o[kDt];
  float m_run = -FLT_MAX, l_run = 0.0f, odd = 0.0f;
  bool met = false; // a value that is not finite
#pragma unroll
  for (int d = 0; d < kDt; d++)
    o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  float4 kr[2][kSteps][2], vr[2][4][HD / 64];
  const Rows keys = rows_of(it.key, it, hd), values = rows_of(it.value, it, hd);
  unsigned k_at = (unsigned)(wave % walkers * kUnit + lc) * keys.stride;
  unsigned v_at = (unsigned)(wave % walkers * kUnit + 4 * lq) * values.stride;
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int st = 0; st < kSteps; st++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          kr[t][st][h] = row4<FULL>(keys, k_at, 16 * t, 32 * st + 8 * lq + 4 * h, hd);
    k_at += (unsigned)(walkers * kUnit) * keys.stride;
  };
  auto load_v = [&]() {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
          vr[t][e][j] = row4<FULL>(values, v_at, 16 * t + e, 64 * j + 4 * lc, hd);
    v_at += (unsigned)(walkers * kUnit) * values.stride;
  };
  const int stride = walkers * kUnit;
  const int end = 16 * (wave / walkers) < it.vectors ? it.t1 : it.t0; // a tile without vectors walks nothing
  int t0 = it.t0 + wave % walkers * kUnit;
  load_k(); // zeros past the end
  load_v();
  fence();
  float qr[kSteps][8];
#pragma unroll
  for (int st = 0; st < kSteps; st++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float scale = active && (FULL || 32 * st + 8 * lq + 4 * h < hd) ? p.scale2 : 0.0f;
      qr[st][4 * h] = x[st][h].x * scale, qr[st][4 * h + 1] = x[st][h].y * scale, qr[st][4 * h + 2] = x[st][h].z * scale,
      qr[st][4 * h + 3] = x[st][h].w * scale;
    }
  auto of = [](const float4 &x, int e) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; };
  for (; t0 < end; t0 += stride) {
    // S^T = K Q^T: instruction (st, i) takes dimension 32 st + 8 lq + i from lane group lq; two sums a position tile
    v4f sc[2][2];
#pragma unroll
    for (int t = 0; t < 2; t++)
      sc[t][0] = sc[t][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < kSteps; st++)
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int t = 0; t < 2; t++)
          sc[t][i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(of(kr[t][st][i / 4], i % 4), qr[st][i], sc[t][i & 1], 0, 0, 0);
    fence();
    load_k(); // zeros past the end: a branch would have the next wait take these loads in
    fence();
    float pv[8], top = -FLT_MAX;
    const int seen = min(it.t1 - 1, last) - t0 - 4 * lq; // of the lane's positions 16 t + e
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        pv[4 * t + e] = 16 * t + e <= seen ? sc[t][0][e] + sc[t][1][e] : -FLT_MAX;
        odd = fmaf(pv[4 * t + e], 0.0f, odd);
        top = fmaxf(top, pv[4 * t + e]);
      }
    top = four_max(top);
    const float m_new = fmaxf(m_run, top);
    if (__any(m_new > m_run)) { // else nothing of the sums changes
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int d = 0; d < kDt; d++)
        o[d] *= alpha;
    }
    const float base = fmaxf(m_new, kMasked);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      pv[i] = __builtin_amdgcn_exp2f(pv[i] - base);
      l_run += pv[i]; // this lane's positions; the four lanes of a vector meet at the end
    }
    float nonfinite = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < HD / 64; j++) {
          const float4 x = vr[t][e][j];
          nonfinite = fmaf(x.x, 0.0f, fmaf(x.y, 0.0f, fmaf(x.z, 0.0f, fmaf(x.w, 0.0f, nonfinite))));
        }
    if (__any(nonfinite != 0.0f)) { // NaN: some value of the step is not finite
      met = true;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int j = 0; j < HD / 64; j++) {
            float4 &x = vr[t][e][j];
            x = float4{finite(x.x) ? x.x : 0.0f, finite(x.y) ? x.y : 0.0f, finite(x.z) ? x.z : 0.0f,
                       finite(x.w) ? x.w : 0.0f};
          }
    }
    // O^T += V^T P^T: instruction (t, e) takes position 16 t + 4 lq + e from lane group lq, which is where the weights
    // are; tile 4 j + c holds dimensions 64 j + 4 m + c
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int d = 0; d < kDt; d++)
          o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(of(vr[t][e][d / 4], d % 4), pv[4 * t + e], o[d], 0, 0, 0);
    fence();
    load_v();
    fence();
  }
  if (odd != 0.0f)
    p.flags[1] = 1;
  // the waves' sums: [wave][vector][HD values, maximum, sum]
  float *sums = reinterpret_cast<float *>(lds);
  {
    const float l = four_sum(l_run);
    float *dst = sums + (size_t)(wave * 16 + lc) * kRow;
#pragma unroll
    for (int j = 0; j < HD / 64; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        *reinterpret_cast<float4 *>(dst + 64 * j + 4 * (4 * lq + e)) =
            float4{o[4 * j][e], o[4 * j + 1][e], o[4 * j + 2][e], o[4 * j + 3][e]};
    if (lq == 0)
      dst[HD] = m_run, dst[HD + 1] = l;
  }
  met = __syncthreads_or(met);
  const int hd4 = hd / 4;
  for (int i = tid; i < it.vectors * hd4; i += kThreads) {
    const int v = i / hd4, d4 = i % hd4;
    const float *src = sums + (size_t)(v / 16 * walkers * 16 + v % 16) * kRow;
    float m = -FLT_MAX;
    for (int w = 0; w < walkers; w++)
      m = fmaxf(m, src[(size_t)w * 16 * kRow + HD]);
    float l = 0.0f;
    float4 sum = float4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = 0; w < walkers; w++) {
      const float *at = src + (size_t)w * 16 * kRow;
      const float scale = __builtin_amdgcn_exp2f(at[HD] - m);
      const float4 x = *reinterpret_cast<const float4 *>(at + 4 * d4);
      l = fmaf(scale, at[HD + 1], l);
      sum = float4{fmaf(scale, x.x, sum.x), fmaf(scale, x.y, sum.y), fmaf(scale, x.z, sum.z), fmaf(scale, x.w, sum.w)};
    }
    float *dst = slot_of(p, it, v);
    *reinterpret_cast<float4 *>(dst + 4 * d4) = sum;
    if (d4 == 0)
      *reinterpret_cast<float4 *>(dst + hd) = slot_end(m, l, met, it);
  }
}

// Wide: up to 128 query vectors, 32 a wave; a step's K and V rows are split once for the block and staged in LDS. A
// product x y is taken as hh + hl + lh of two FP16 parts each (22 bits and more), three matrix instructions where exact
// BF16 parts take six. The parts need values near 2^15: each query vector and each K row is scaled by a power of two of
// its own, taken out of the score again; each group of four V rows likewise, and its exponent ev joins the score before
// the exponential, so that the weights are exp2(s + ev - m) and meet V 2^-ev, with m the running maximum of s + ev. The
// softmax's sum takes them times 2^-ev. A value is so exact to 2^-22 of itself, or to 2^-39 of the largest of its query
// vector, K row or four V rows.
//
// A weight is exact to 2^-22 of itself, or to 2^-25 where the largest is 2^11 or more; so, with the ev of a walk within 3
// kSpread of each other, to 2^(12 - 36) of the row's largest (to 2^-36 where they are the same). An element far above the
// others would raise its rows' ev and leave the other rows' weights too few bits, in every dimension. So a wave compares the
// exponents of its V rows with those of its first step, and at the end of a walk they are compared with each other: where
// they lie further apart, or below what ev takes, the block does the walk again in narrow tiles, whose FP32 products have no
// such limits. That takes longer (one element of 10^6 in a prefix: 923 prompt rows 94 -> 290 us, 64 requests 98 -> 180), and
// is rare: the largest of four rows of a head differs by far less.
// (Kept per walk as a smallest and a largest ev, in registers, scalars or LDS, the same check spilled 10 to 17 registers: 64
// requests 98 -> 112 us.)
//
// V parts lie transposed, a dimension's 32 slots in 64 bytes, its 16-byte units where v_unit puts them: a matrix operand's
// read takes one unit of 16 dimensions, a staging write half a unit of every fourth one, and both spread over the banks.
constexpr int kSpread = 4, kNoExponent = -(1 << 20);
template <int HD> struct WideStage {
  static constexpr int kKRow = HD + 8;
  uint16_t k[2][kUnit * kKRow];
  uint16_t v[2][HD * kUnit];
  float k_back[kUnit]; // 2^(e - 14): undoes a K row's scale
  float v_exp[kUnit];  // ev
  float v_back[kUnit]; // 2^-ev
};
__device__ __forceinline__ int v_unit(int dim, int unit) { // in halves
  const int four = dim >> 2;
  return ((four << 2) | ((dim ^ four) & 3)) * kUnit + 8 * ((unit ^ four ^ (dim >> 4)) & 3);
}

template <int HD, bool FULL> __device__ bool walk_wide(const FastAttn &p, const Item &it, unsigned char *lds) {
  typedef WideStage<HD> Stage;
  Stage *const stages = reinterpret_cast<Stage *>(lds); // two: a step is staged while the one before is computed
  constexpr int kSteps = HD / 32, kDt = HD / 16, kLeastK = -100, kLeastV = -60;
  constexpr int kItems = kUnit * HD / 8 / kThreads; // K staging items of eight values a thread
  constexpr int kLanes = HD / 8;                    // a K row's
  constexpr int kVLanes = HD / 4;
  static_assert(kItems >= 1 && kUnit / 4 * kVLanes <= kThreads, "staging items");
  const int tid = own_thread(), lane = tid & (kWave - 1), wave = tid / kWave, lq = lane >> 4, lc = lane & 15;
  const int hd = p.hd;
  constexpr bool kAllStage = kUnit / 4 * kVLanes == kThreads;
  const bool v_stager = kAllStage || tid < kUnit / 4 * kVLanes;
  const int vg = tid / kVLanes, vd = 4 * (tid % kVLanes); // V item: positions 4 vg .. + 3, dimensions vd .. + 3
  float4 kr[kItems][2], vr[4];
  bool met = false;           // a value that is not finite
  int ev_first = kNoExponent; // the largest exponent of the wave's V rows of the first step that are not zero
  bool spread = false;        // that of others lies further from it than kSpread
  const Rows keys = rows_of(it.key, it, hd), values = rows_of(it.value, it, hd);
  unsigned k_at = (unsigned)(tid / kLanes) * keys.stride, v_at = (unsigned)(4 * vg) * values.stride;
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < kItems; u++) {
      const int d = 8 * (tid % kLanes);
      kr[u][0] = row4<FULL>(keys, k_at, u * (kThreads / kLanes), d, hd);
      kr[u][1] = row4<FULL>(keys, k_at, u * (kThreads / kLanes), d + 4, hd);
    }
    if (v_stager)
#pragma unroll
      for (int e = 0; e < 4; e++)
        vr[e] = row4<FULL>(values, v_at, e, vd, hd);
    k_at += kUnit * keys.stride;
    v_at += kUnit * values.stride;
  };
  auto peak = [](const float4 &x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); };
  auto stage = [&](Stage &sh, auto first) {
#pragma unroll
    for (int u = 0; u < kItems; u++) {
      const int i = tid + u * kThreads, row = i / kLanes, d = 8 * (i % kLanes);
      const float4 a = kr[u][0], b = kr[u][1];
      // a row with an infinity keeps it: its scores are not finite, whatever the scale
      const float top = fminf(group_reduce_max(fmaxf(peak(a), peak(b)), kLanes), FLT_MAX);
      int e;
      const float scale = f16_scale(top, kLeastK, e);
      v4i h, l;
      int th, tl;
      f16_pair(a.x, a.y, scale, th, tl), h[0] = th, l[0] = tl;
      f16_pair(a.z, a.w, scale, th, tl), h[1] = th, l[1] = tl;
      f16_pair(b.x, b.y, scale, th, tl), h[2] = th, l[2] = tl;
      f16_pair(b.z, b.w, scale, th, tl), h[3] = th, l[3] = tl;
      *reinterpret_cast<v4i *>(&sh.k[0][row * Stage::kKRow + d]) = h;
      *reinterpret_cast<v4i *>(&sh.k[1][row * Stage::kKRow + d]) = l;
      sh.k_back[row] = __uint_as_float((unsigned)(127 - 14 + e) << 23); // by all of the row's lanes: no branch
    }
    if (v_stager) {
      float top = fmaxf(fmaxf(peak(vr[0]), peak(vr[1])), fmaxf(peak(vr[2]), peak(vr[3])));
      top = group_reduce_max(top, kVLanes);
      int ev;
      const float scale = f16_scale(top > 0.0f ? top : 1.0f, kLeastV, ev); // rows of zeros take no extreme exponent
      const int exponent = (int)(__float_as_uint(top) >> 23) - 127; // ev, but not raised to kLeastV
      if constexpr (decltype(first)::value) {
        const int mine = top > 0.0f ? exponent : kNoExponent;
#pragma unroll
        for (int o = 0; o < kWave; o += kVLanes)
          ev_first = max(ev_first, __builtin_amdgcn_readlane(mine, o));
        spread = mine != kNoExponent && mine < ev_first - kSpread;
      } else {
        spread |= top > 0.0f && (unsigned)(exponent - ev_first + kSpread) > 2u * kSpread;
      }
      // slot of position 16 t + 4 q + e: 8 q + 4 t + e, so the four of this item are half of unit vg % 4
      auto put = [&](int d, float x0, float x1, float x2, float x3) {
        int h0, l0, h1, l1;
        f16_pair(x0, x1, scale, h0, l0);
        f16_pair(x2, x3, scale, h1, l1);
        const int at = v_unit(vd + d, vg % 4) + 4 * (vg / 4);
        *reinterpret_cast<int2 *>(&sh.v[0][at]) = int2{h0, h1};
        *reinterpret_cast<int2 *>(&sh.v[1][at]) = int2{l0, l1};
      };
      put(0, vr[0].x, vr[1].x, vr[2].x, vr[3].x);
      put(1, vr[0].y, vr[1].y, vr[2].y, vr[3].y);
      put(2, vr[0].z, vr[1].z, vr[2].z, vr[3].z);
      put(3, vr[0].w, vr[1].w, vr[2].w, vr[3].w);
      const int e = 4 * vg + tid % 4;
      sh.v_exp[e] = (float)ev;
      sh.v_back[e] = __uint_as_float(ev < 127 ? (unsigned)(127 - ev) << 23 : 1u << 22);
    }
  };
  // the loaded V values that are not finite become 0
  auto check = [&]() {
    float odd = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++)
      odd = fmaf(vr[e].x, 0.0f, fmaf(vr[e].y, 0.0f, fmaf(vr[e].z, 0.0f, fmaf(vr[e].w, 0.0f, odd))));
    if (__any(v_stager && odd != 0.0f)) {
      met = true;
#pragma unroll
      for (int e = 0; e < 4; e++)
        vr[e] = float4{finite(vr[e].x) ? vr[e].x : 0.0f, finite(vr[e].y) ? vr[e].y : 0.0f,
                       finite(vr[e].z) ? vr[e].z : 0.0f, finite(vr[e].w) ? vr[e].w : 0.0f};
    }
  };
  // the wave's query vectors, dimensions 32 st + 8 lq .. + 7 of vector 32 wave + 16 n + lc: on their way with the first
  // step's rows, then their parts
  float4 x[2][kSteps][2];
  int last[2];
#pragma unroll
  for (int n = 0; n < 2; n++) {
    const int v = 32 * wave + 16 * n + lc;
    const bool active = v < it.vectors;
    last[n] = !active ? -1 : it.last0 == INT32_MAX ? INT32_MAX : it.last0 + v / p.kv_mul;
    const float *src = p.q + ((size_t)(it.row0 + (active ? v / p.kv_mul : 0)) * p.n_heads + (size_t)it.g * p.kv_mul +
                              (active ? v % p.kv_mul : 0)) * hd;
#pragma unroll
    for (int st = 0; st < kSteps; st++)
#pragma unroll
      for (int k = 0; k < 2; k++)
        x[n][st][k] = load4(src, active ? 32 * st + 8 * lq + 4 * k : hd, hd);
  }
  fence();
  load(); // zeros past the end
  fence();
  v4i qh[2][kSteps], ql[2][kSteps];
  float q_back[2], m_run[2], l_run[2], odd = 0.0f;
  const bool busy = 32 * wave < it.vectors; // a wave without vectors only stages
  v4f o[2][kDt];
#pragma unroll
  for (int n = 0; n < 2; n++) {
    float top = 0.0f;
#pragma unroll
    for (int st = 0; st < kSteps; st++)
      top = fmaxf(top, fmaxf(peak(x[n][st][0]), peak(x[n][st][1])));
    top = fminf(four_max(top), FLT_MAX);
    int e;
    const float scale = f16_scale(top, kLeastK, e);
    q_back[n] = __uint_as_float((unsigned)(127 - 14 + e) << 23) * p.scale2;
#pragma unroll
    for (int st = 0; st < kSteps; st++) {
      const float4 a = x[n][st][0], b = x[n][st][1];
      int th, tl;
      f16_pair(a.x, a.y, scale, th, tl), qh[n][st][0] = th, ql[n][st][0] = tl;
      f16_pair(a.z, a.w, scale, th, tl), qh[n][st][1] = th, ql[n][st][1] = tl;
      f16_pair(b.x, b.y, scale, th, tl), qh[n][st][2] = th, ql[n][st][2] = tl;
      f16_pair(b.z, b.w, scale, th, tl), qh[n][st][3] = th, ql[n][st][3] = tl;
    }
    m_run[n] = -FLT_MAX, l_run[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDt; d++)
      o[n][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  v4f sc[2][2];
  auto score = [&](const Stage &sh) {
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int t = 0; t < 2; t++)
        sc[n][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < kSteps; st++) {
      v4i kh[2], kl[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const int at = (16 * t + lc) * Stage::kKRow + 32 * st + 8 * lq;
        kh[t] = *reinterpret_cast<const v4i *>(&sh.k[0][at]);
        kl[t] = *reinterpret_cast<const v4i *>(&sh.k[1][at]);
      }
#pragma unroll
      for (int k = 0; k < 3; k++) // the three products in turn over four sums: none waits for the one before
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int n = 0; n < 2; n++)
            sc[n][t] = mfma_f16(k == 0 ? kl[t] : kh[t], k == 1 ? ql[n][st] : qh[n][st], sc[n][t]);
    }
  };
  auto weigh_and_add = [&](const Stage &sh, int t0) {
    v4i ph[2], pl[2];
    auto of = [](const float4 &x, int e) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; };
#pragma unroll
    for (int n = 0; n < 2; n++) {
      float pv[8], top = -FLT_MAX;
      const int seen = min(it.t1 - 1, last[n]) - t0 - 4 * lq; // of the lane's positions 16 t + e
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const float4 k_back = *reinterpret_cast<const float4 *>(&sh.k_back[16 * t + 4 * lq]);
        const float4 v_exp = *reinterpret_cast<const float4 *>(&sh.v_exp[16 * t + 4 * lq]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float x = fmaf(sc[n][t][e], of(k_back, e) * q_back[n], of(v_exp, e));
          pv[4 * t + e] = 16 * t + e <= seen ? x : -FLT_MAX;
          odd = fmaf(pv[4 * t + e], 0.0f, odd);
          top = fmaxf(top, pv[4 * t + e]);
        }
      }
      // the running maximum moves only when a score passes it by 2^4, which the weights' range leaves room for: nearly
      // all steps then need no exchange between lanes and no rescale
      if (__any(top > m_run[n] + 4.0f)) {
        const float m_new = fmaxf(m_run[n], four_max(top)), alpha = __builtin_amdgcn_exp2f(m_run[n] - m_new);
        l_run[n] *= alpha;
        m_run[n] = m_new;
#pragma unroll
        for (int d = 0; d < kDt; d++)
          o[n][d] *= alpha;
      }
      const float base = fmaxf(m_run[n], kMasked) - 11.0f; // weights up to 2^15, the largest at least 2^11
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const float4 v_back = *reinterpret_cast<const float4 *>(&sh.v_back[16 * t + 4 * lq]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pv[4 * t + e] = __builtin_amdgcn_exp2f(pv[4 * t + e] - base);
          sum = fmaf(pv[4 * t + e], of(v_back, e), sum);
        }
      }
      l_run[n] += sum;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        int th, tl;
        f16_pair(pv[2 * i], pv[2 * i + 1], 1.0f, th, tl);
        ph[n][i] = th, pl[n][i] = tl;
      }
    }
    fence();
    // the products in turn over four sums, as above; the next operands are on their way meanwhile
    v4i vh[2][2], vl[2][2];
    auto fetch = [&](int d, int buffer) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int at = v_unit(16 * (d + i) + lc, lq);
        vh[buffer][i] = *reinterpret_cast<const v4i *>(&sh.v[0][at]);
        vl[buffer][i] = *reinterpret_cast<const v4i *>(&sh.v[1][at]);
      }
    };
    fetch(0, 0);
#pragma unroll
    for (int d = 0; d < kDt; d += 2) {
      const int now = d / 2 % 2;
      if (d + 2 < kDt)
        fetch(d + 2, now ^ 1);
      fence();
#pragma unroll
      for (int k = 0; k < 3; k++)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int n = 0; n < 2; n++)
            o[n][d + i] = mfma_f16(k == 0 ? vl[now][i] : vh[now][i], k == 1 ? pl[n] : ph[n], o[n][d + i]);
      fence();
    }
  };
  if (it.t0 < it.t1) {
    check();
    stage(stages[0], std::true_type());
    load();
    __syncthreads();
  }
  int turn = 0;
  for (int t0 = it.t0; t0 < it.t1; t0 += kUnit, turn ^= 1) {
    check();
    fence();
    if (busy) {
      score(stages[turn]);
      // the next step's stage was read before the last barrier; past the end it takes zeros that nobody reads
      stage(stages[turn ^ 1], std::false_type());
      fence();
      load();
      fence();
      weigh_and_add(stages[turn], t0);
    } else {
      stage(stages[turn ^ 1], std::false_type());
      load();
    }
    __syncthreads();
  }
  // the waves' findings, where the stages were
  int2 *const found = reinterpret_cast<int2 *>(lds);
  const bool apart = __any(spread);
  if (lane == 0)
    found[wave] = int2{ev_first, (apart ? 2 : 0) | (met ? 1 : 0)};
  __syncthreads();
  int low = INT32_MAX, high = kNoExponent, flags = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; w++) {
    const int2 f = found[w];
    low = min(low, f.x == kNoExponent ? INT32_MAX : f.x);
    high = max(high, f.x);
    flags |= f.y;
  }
  if (flags & 2 || high - kSpread > low || low - kSpread < kLeastV) // uniform
    return false;
  met = flags & 1;
  if (odd != 0.0f && (last[0] >= 0 || last[1] >= 0))
    p.flags[1] = 1;
#pragma unroll
  for (int n = 0; n < 2; n++) {
    const float l = four_sum(l_run[n]);
    const int v = 32 * wave + 16 * n + lc;
    if (v >= it.vectors)
      continue;
    float *dst = slot_of(p, it, v);
    const float back = 0x1p-25f; // 2^14 of the V rows, 2^11 of the weights
#pragma unroll
    for (int d = 0; d < kDt; d++)
      if (16 * d + 4 * lq < hd)
        *reinterpret_cast<float4 *>(dst + 16 * d + 4 * lq) =
            float4{o[n][d][0] * back, o[n][d][1] * back, o[n][d][2] * back, o[n][d][3] * back};
    if (lq == 0)
      *reinterpret_cast<float4 *>(dst + hd) = slot_end(m_run[n], l * 0x1p-11f, met, it);
  }
  return true;
}

// LDS: the plan, then the walk's.
constexpr size_t kPlanLds = (sizeof(Plan) + 15) / 16 * 16;
template <int HD> constexpr size_t fast_lds() {
  constexpr size_t narrow_sums = (size_t)(kThreads / kWave) * 16 * (HD + 4) * 4, stages = 2 * sizeof(WideStage<HD>);
  return kPlanLds + (narrow_sums > stages ? narrow_sums : stages);
}
static_assert(kBlocksPerCu * fast_lds<128>() <= 160 * 1024, "blocks of a CU");

// Positions 0 .. e - 1 of a walk that lies at a .. a + time - 1 on the line: the first one behind the cut at x.
__device__ __forceinline__ int cut_at(long long x, long long a, long long time, int e) {
  return x <= a ? 0 : x >= a + time ? e : (int)((double)(x - a) / (double)time * e) / kUnit * kUnit;
}

// Where row `row` finds its partial sums, for the merge.
__device__ void find_slots(const FastAttn &p, const Plan &plan, int r0) {
  __shared__ int owner[kThreads];
  const int tid = threadIdx.x, row = r0 + tid;
  owner[tid] = -1;
  __syncthreads();
  bool bad = false;
  if (plan.total > 0)
    for (int r = tid; r < p.batch.count; r += kThreads) {
      const Request q = request_at(p.batch, r, bad);
      for (int i = max(q.first, r0); i < min(q.first + q.rows, r0 + kThreads); i++)
        owner[i - r0] = r;
    }
  __syncthreads();
  if (row >= p.batch.rows)
    return;
  RowSlots at{};
  at.own_first = -1;
  if (owner[tid] >= 0) {
    const Request q = request_at(p.batch, owner[tid], bad);
    const int j = row - q.first, tile = own_tiles(p, q.rows) == 1 ? 0 : j / p.tile_rows;
    const int rows = min(p.tile_rows, q.rows - tile * p.tile_rows), end = q.length + tile * p.tile_rows + rows;
    const long long a = plan.line[owner[tid]] - own_time(p, q) + tile_start(p, q.length, tile);
    at.own_first = (int)whole(a, plan.slice);
    at.own_last = (int)whole(a + walk_time(rows * p.kv_mul, end) - 1, plan.slice);
    at.own_v = (j - tile * p.tile_rows) * p.kv_mul;
    at.slot = q.slot;
    at.last = q.length + j;
    if (p.batch.prefix) {
      const int i = row - plan.first_row, t = i / p.tile_rows;
      const long long b = t * plan.full, e = min(b + plan.full, plan.prefix);
      at.prefix_first = (int)whole(b, plan.slice);
      at.prefix_last = (int)whole(e - 1, plan.slice);
      at.prefix_v = (i - t * p.tile_rows) * p.kv_mul;
    }
  }
  p.rows[row] = at;
}

// Blocks: p.blocks for each KV head (the head fastest, so that consecutive blocks, which go to the XCDs in turn, give an XCD
// the same heads' rows, and that the two blocks of a CU come from different parts of the line), then ceil(rows / 256) that
// write down each row's slots for the merge (in front they kept blocks with slices from starting with the others).
template <int HD, bool FULL> __global__ __launch_bounds__(kThreads, kBlocksPerCu) void attn_requests(FastAttn p) {
  extern __shared__ __align__(16) unsigned char lds[];
  Plan &plan = *reinterpret_cast<Plan *>(lds);
  make_plan(p, plan);
  const int tid = threadIdx.x;
  const int i = blockIdx.x, g = i % p.n_kv_heads, block = i / p.n_kv_heads;
  if (block >= p.blocks) {
    find_slots(p, plan, (i - p.blocks * p.n_kv_heads) * kThreads);
    return;
  }
  const long long x0 = uniform(block * plan.slice), x1 = uniform(min(block * plan.slice + plan.slice, plan.total));
  const size_t begins = (size_t)p.batch.rows * p.n_heads; // slots of the walks that begin in a block, prefix and own each
  int r = -1, part = -1; // the part of a wide tile that is done again in narrow ones, by its first row
  for (long long x = x0; x < x1;) {
    Item it;
    long long a, time; // the walk's place
    int end;           // its positions
    const bool prefix = x < plan.prefix;
    if (prefix) {
      const int tile = (int)whole(x, plan.full);
      a = tile * plan.full;
      time = min(plan.full, plan.prefix - a);
      end = p.batch.prefix;
      it.row0 = plan.first_row + tile * p.tile_rows;
      it.vectors = min(p.tile_rows, plan.end_row - it.row0) * p.kv_mul;
      it.key = p.prefix_key + (size_t)g * p.batch.prefix_head_base;
      it.value = p.prefix_value + (size_t)g * p.batch.prefix_head_base;
      it.pos_stride = p.batch.prefix_pos_stride;
      it.last0 = INT32_MAX;
    } else {
      if (r < 0) {
        int lo = 0, hi = p.batch.count - 1; // the first request whose walks end behind x
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (plan.line[mid] > x)
            hi = mid;
          else
            lo = mid + 1;
        }
        r = lo;
      }
      while (plan.line[r] <= x) // requests without rows; the last one's end is the line's
        r++;
      bool bad = false;
      const Request q = r < kTable ? plan.table[r] : request_at(p.batch, r, bad);
      const long long begin = plan.line[r] - own_time(p, q);
      int tile = 0;
      for (int hi = own_tiles(p, q.rows) - 1; tile < hi;) { // the last tile that begins at or before x
        const int mid = (tile + hi + 1) / 2;
        if (begin + tile_start(p, q.length, mid) <= x)
          tile = mid;
        else
          hi = mid - 1;
      }
      const int j0 = tile * p.tile_rows, rows = min(p.tile_rows, q.rows - j0);
      const size_t cache = (size_t)q.slot * p.batch.slot_floats + (size_t)g * p.batch.head_base;
      end = q.length + j0 + rows;
      a = begin + tile_start(p, q.length, tile);
      time = walk_time(rows * p.kv_mul, end);
      it.row0 = q.first + j0;
      it.vectors = rows * p.kv_mul;
      it.key = p.key + cache;
      it.value = p.value + cache;
      it.pos_stride = p.batch.pos_stride;
      it.last0 = q.length + j0;
    }
    a = uniform(a);
    time = uniform(time);
    r = uniform(r);
    it.g = g;
    it.row0 = uniform(it.row0);
    it.vectors = uniform(it.vectors);
    it.last0 = uniform(it.last0);
    it.t0 = uniform(cut_at(x, a, time, end));
    it.t1 = uniform(cut_at(x1, a, time, end));
    if (a >= x0) {
      it.slot0 = (prefix ? 0 : begins) + (size_t)it.row0 * p.n_heads + (size_t)g * p.kv_mul;
      it.slot_row = p.n_heads;
    } else {
      it.slot0 = 2 * begins + ((size_t)g * p.blocks + block) * kTileVectors;
      it.slot_row = p.kv_mul;
    }
    if (x != x0 || part >= 0)
      __syncthreads(); // the walk before is done with its LDS
    if (it.t0 == it.t1) { // a cut within the first step's positions: nothing is left for this side of it
      const int quads = p.hd / 4 + 1;
      for (int e = tid; e < it.vectors * quads; e += kThreads)
        *reinterpret_cast<float4 *>(slot_of(p, it, e / quads) + 4 * (e % quads)) =
            float4{e % quads == quads - 1 ? -FLT_MAX : 0.0f, 0.0f, 0.0f, 0.0f};
    } else if (it.vectors > kNarrowVectors && part < 0) {
      if (!walk_wide<HD, FULL>(p, it, lds + kPlanLds)) {
        part = 0; // V rows too far apart in size for its parts
        continue;
      }
    } else {
      int next = -1;
      if (part >= 0) {
        const int rows = uniform(it.vectors / p.kv_mul), n = min(rows - part, p.narrow_rows);
        it.row0 += part;
        it.vectors = n * p.kv_mul;
        it.last0 = prefix ? INT32_MAX : it.last0 + part;
        it.slot0 += (size_t)part * it.slot_row;
        next = part + n < rows ? part + n : -1;
      }
      walk_narrow<HD, FULL>(p, it, lds + kPlanLds);
      part = next;
      if (part >= 0)
        continue;
    }
    x = a + time;
  }
}

// A thread per (row, head, four dimensions): the row's partial sums over the prefix and over its own positions, rescaled to
// their largest maximum and added in order.
__global__ __launch_bounds__(kThreads) void attn_requests_merge(FastAttn p) {
  const unsigned hd4 = (unsigned)p.hd / 4;
  const unsigned idx = blockIdx.x * kThreads + threadIdx.x, vec = idx / hd4; // at most 2^31: 32-bit divisions
  const int d4 = (int)(idx % hd4), row = (int)(vec / (unsigned)p.n_heads), head = (int)(vec % (unsigned)p.n_heads);
  if (row >= p.batch.rows)
    return;
  const int g = head / p.kv_mul, h = head % p.kv_mul;
  const RowSlots mine = p.rows[row];
  if (mine.own_first < 0)
    return;
  const int shared = p.batch.prefix ? mine.prefix_last - mine.prefix_first + 1 : 0;
  const int count = shared + mine.own_last - mine.own_first + 1;
  const size_t slot = (size_t)(p.hd + 4), begins = (size_t)p.batch.rows * p.n_heads;
  auto slot_at = [&](int s) {
    const bool prefix = s < shared;
    const int k = prefix ? s : s - shared, block = (prefix ? mine.prefix_first : mine.own_first) + k;
    const size_t at = k == 0 ? (prefix ? 0 : begins) + (size_t)vec
                             : 2 * begins + ((size_t)g * p.blocks + block) * kTileVectors +
                                   (prefix ? mine.prefix_v : mine.own_v) + h;
    return p.partial + at * slot;
  };
  float m = -FLT_MAX, l = 0.0f;
  float4 o = float4{0.0f, 0.0f, 0.0f, 0.0f};
  bool met = false;
  constexpr int kAhead = 4; // sums whose loads are in flight together (8: prompts 2 us more, decode steps the same)
  for (int s0 = 0; s0 < count; s0 += kAhead) {
    float4 end[kAhead], x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const int s = min(s0 + k, count - 1);
      const float *src = slot_at(s);
      end[k] = *reinterpret_cast<const float4 *>(src + p.hd);
      x[k] = *reinterpret_cast<const float4 *>(src + 4 * d4);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      top = fmaxf(top, end[k].x); // the last share again past the count: the same maximum
    const float alpha = __builtin_amdgcn_exp2f(m - top);
    l *= alpha;
    o = float4{o.x * alpha, o.y * alpha, o.z * alpha, o.w * alpha};
    m = top;
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (s0 + k < count) {
        const float w = __builtin_amdgcn_exp2f(end[k].x - m);
        l = fmaf(w, end[k].y, l);
        o = float4{fmaf(w, x[k].x, o.x), fmaf(w, x[k].y, o.y), fmaf(w, x[k].z, o.z), fmaf(w, x[k].w, o.w)};
        met |= __float_as_int(end[k].w) != 0;
      }
  }
  if (met) { // V values that are not finite, whatever their weights: a positive one changes neither infinity nor NaN
    for (int s = 0; s < count; s++) {
      const float *src = slot_at(s);
      const bool prefix = s < shared;
      const int t0 = max(__float_as_int(src[p.hd + 2]), 0), t1 = __float_as_int(src[p.hd + 3]);
      const float *v = prefix ? p.prefix_value + (size_t)g * p.batch.prefix_head_base
                              : p.value + (size_t)mine.slot * p.batch.slot_floats + (size_t)g * p.batch.head_base;
      const size_t stride = prefix ? p.batch.prefix_pos_stride : p.batch.pos_stride;
      for (int t = t0; t < min(t1, prefix ? p.batch.prefix : mine.last + 1); t++) {
        const float4 y = *reinterpret_cast<const float4 *>(v + (size_t)t * stride + 4 * d4);
        o = float4{finite(y.x) ? o.x : o.x + y.x, finite(y.y) ? o.y : o.y + y.y, finite(y.z) ? o.z : o.z + y.z,
                   finite(y.w) ? o.w : o.w + y.w};
      }
    }
  }
  *reinterpret_cast<float4 *>(p.out + (size_t)vec * p.hd + 4 * d4) = float4{o.x / l, o.y / l, o.z / l, o.w / l};
}

} // namespace

// The matrix-core form takes head dimensions up to 128 in whole groups of four, with 16-byte aligned rows: its loads are of
// 16 bytes, and a head of 256 would need twice the registers for its query parts and value sums.
bool attention_requests_fast(const AttentionRequestsJob &job) {
  const RequestsDev &b = job.batch;
  const uintptr_t all = (uintptr_t)job.out | (uintptr_t)job.q | (uintptr_t)job.prefix_key | (uintptr_t)job.prefix_value |
                        (uintptr_t)job.key | (uintptr_t)job.value;
  // a walk's rows lie within 2^31 bytes, which its loads' 32-bit offsets reach
  const bool near = (size_t)b.prefix * b.prefix_pos_stride < (1u << 29) && (size_t)b.seq_len * b.pos_stride < (1u << 29);
  // the merge's launch holds fewer than 2^32 threads
  const bool few = (uint64_t)b.rows * job.n_heads * job.head_dim / 4 <= (1u << 31);
  return job.head_dim <= 128 && job.head_dim % 4 == 0 && (all & 15) == 0 && b.rows <= (1 << 20) && job.n_heads <= 1024 &&
         near && few;
}

// Blocks of a KV head: what the chip holds at once, or as many as the longest line that the buffers' sizes allow gives
// slices of kMinSlice.
static int fast_blocks(const AttentionRequestsJob &job) {
  const RequestsDev &b = job.batch;
  const long long cus = device().cu_count > 0 ? device().cu_count : 256, kv_mul = job.n_heads / job.n_kv_heads;
  const long long tile_rows = kTileVectors / kv_mul, tiles = (b.rows + tile_rows - 1) / tile_rows;
  const long long own = (b.count < b.rows ? b.count : b.rows) + tiles; // own tiles
  constexpr WalkTime wide = walk_time_of(kTileVectors);                // the longest
  const long long line = (b.prefix ? tiles * (wide.begin + (long long)wide.position * b.prefix) : 0) +
                         own * (wide.begin + (long long)wide.position * b.seq_len);
  const long long most = (line + kMinSlice - 1) / kMinSlice, held = kBlocksPerCu * cus / job.n_kv_heads;
  return (int)(most < held ? most : held > 1 ? held : 1);
}

// Slots: one for each vector of the prefix's walks and of the requests' own, and a tile's for each block, which goes on with
// one walk at most.
static size_t fast_slots(const AttentionRequestsJob &job) {
  return 2 * (size_t)job.batch.rows * job.n_heads + (size_t)job.n_kv_heads * fast_blocks(job) * kTileVectors;
}

size_t attention_requests_workspace(const AttentionRequestsJob &job) {
  if (!attention_requests_fast(job))
    return 0;
  return fast_slots(job) * (size_t)(job.head_dim + 4) * sizeof(float) + (size_t)job.batch.rows * sizeof(RowSlots);
}

bool launch_attention_fast(const AttentionRequestsJob &job, void *workspace, hipStream_t stream) {
  FastAttn p{};
  p.out = job.out;
  p.q = job.q;
  p.prefix_key = job.prefix_key;
  p.prefix_value = job.prefix_value;
  p.key = job.key;
  p.value = job.value;
  p.batch = job.batch;
  p.n_heads = job.n_heads;
  p.n_kv_heads = job.n_kv_heads;
  p.kv_mul = job.n_heads / job.n_kv_heads;
  p.hd = job.head_dim;
  p.tile_rows = kTileVectors / p.kv_mul;
  p.narrow_rows = kNarrowVectors / p.kv_mul;
  p.blocks = fast_blocks(job);
  p.scale2 = 1.4426950408889634f / sqrtf((float)job.head_dim);
  p.rows = (RowSlots *)workspace;
  p.partial = (float *)(p.rows + job.batch.rows);
  p.flags = device().error_flags;
  const long long blocks = (long long)p.blocks * p.n_kv_heads + (job.batch.rows + kThreads - 1) / kThreads;
  const bool full = job.head_dim == 64 || job.head_dim == 128;
  const auto kernel = job.head_dim <= 64 ? (full ? attn_requests<64, true> : attn_requests<64, false>)
                                         : (full ? attn_requests<128, true> : attn_requests<128, false>);
  const size_t lds = job.head_dim <= 64 ? fast_lds<64>() : fast_lds<128>();
  static const hipError_t allowed = [] {
    hipError_t e = hipSuccess;
    auto allow = [&](const void *k, size_t bytes) {
      if (e == hipSuccess)
        e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    allow((const void *)attn_requests<64, true>, fast_lds<64>());
    allow((const void *)attn_requests<64, false>, fast_lds<64>());
    allow((const void *)attn_requests<128, true>, fast_lds<128>());
    allow((const void *)attn_requests<128, false>, fast_lds<128>());
    return e;
  }();
  if (allowed != hipSuccess)
    return raise("allowing the attention kernel its LDS failed: %s", hipGetErrorString(allowed));
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), lds, stream, p);
  if (!launch_ok("attn_requests"))
    return false;
  const long long threads = (long long)job.batch.rows * job.n_heads * (job.head_dim / 4);
  hipLaunchKernelGGL(attn_requests_merge, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream,
                     p);
  return launch_ok("attn_requests_merge");
}

bool launch_attention_requests(const AttentionRequestsJob &job, void *workspace, hipStream_t stream) {
  if (attention_requests_fast(job))
    return launch_attention_fast(job, workspace, stream);
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
