// Low-rank adapters of many requests beside shared projections (gfx950): c = base + scale B (A x) per row, each row with
// the adapter that its request has.
//
//   lora_shrink   block (share of K, tile of 32 rows with one adapter, eight 16-entry tiles of A): the share's part of A x on
//                 the BF16 matrix cores. The tiles are found in the adapter array by the blocks themselves.
//   lora_join     the shares' parts added, for batches whose columns would each read them again.
//   lora_expand   block (columns, tile of rows): base + scale B (A x), and for W1 and W3 their gate, read and written once.
//   lora_rows     any shape: one block per row and segment, A x kept in LDS. 32 rows of 4097 values, rank 16, beside QKV take
//                 87 us, 1100 of rank 64 beside W1 and W3 1790.
//
// Measured (BF16 but for the first): one row of 2048 values, rank 8, beside Wo 9.5 us; 32 rows of 4096, rank 16, beside QKV
// 13 us (7 and 6.5); 1100 rows of 4096, rank 64, beside W1 and W3 of 14336 81 us (21, 5 and 58: the expansion moves 189 MB of
// base rows and outputs and 18 MB of adapters at 3.6 TB/s). Few rows are bound by the two launches and the loads that wait
// for each other in them, many by HBM.
//
// The products are FP32-accurate: a value x is split exactly into three BF16 parts (8 bits each), and x y is taken as the
// six products of parts above 2^-24 of it, or three where y is a BF16 adapter's value.
#include "common.h"
#include "lanes.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

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

// ---- tiles of rows on the matrix cores --------------------------------------------------------------------------------

constexpr int kTileRows = 32;
constexpr int kMaxAdapters = 4096; // of the tiled form: their rows are counted in LDS

// The launch: A's of all segments (and A3's) as one list of matrices, their rows in 16-entry tiles side by side in A x.
struct Tiled {
  LoraJob job;
  int matrices;               // A and A3 of the segments, in order
  int first_tile[7];          // of each matrix, and the number of all
  int shares;                 // of K, in lora_shrink's partial sums
  int steps;                  // of 32 values in K
  bool skip_plain;            // rows without an adapter stay as they are
  int tiles;                  // row tiles at most
  int width;                  // floats of a row of A x: 16 * first_tile[matrices]
  int columns;                // of an lora_expand block: a multiple of 128
  struct Tile {
    int adapter, rows;        // -1: none; 0 rows: no tile
    int row[kTileRows];
  } *tile;
  float *low;                 // [share][tile][32][width]
  float *joined;              // [tile][32][width], or low's only share
  int *flags;
};

__device__ __forceinline__ const void *matrix_a(const Tiled &p, int i, int &rank) {
  for (int s = 0; s < p.job.nseg; s++) {
    const LoraSegmentDev seg = pick(p.job, s);
    rank = seg.rank;
    if (i == 0)
      return seg.a;
    i--;
    if (seg.swiglu) {
      if (i == 0)
        return seg.a3;
      i--;
    }
  }
  return nullptr;
}

// Eight values as three BF16 parts whose sum they are exactly (value 2 w in the low half of dword w).
__device__ __forceinline__ void parts_of(const float (&v)[8], v4i &ph, v4i &pm, v4i &pl) {
#pragma unroll
  for (int w = 0; w < 4; w++) {
    unsigned u[2][3];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const float x = v[2 * w + k];
      u[k][0] = __float_as_uint(x);
      const float r1 = x - __uint_as_float(u[k][0] & 0xFFFF0000u);
      u[k][1] = __float_as_uint(r1);
      u[k][2] = __float_as_uint(r1 - __uint_as_float(u[k][1] & 0xFFFF0000u));
    }
    ph[w] = (int)__builtin_amdgcn_perm(u[1][0], u[0][0], 0x07060302u);
    pm[w] = (int)__builtin_amdgcn_perm(u[1][1], u[0][1], 0x07060302u);
    pl[w] = (int)__builtin_amdgcn_perm(u[1][2], u[0][2], 0x07060302u);
  }
}
__device__ __forceinline__ v4f mfma(const v4i &a, const v4i &b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Eight values of an adapter's row as matrix operands: the BF16 bits as they are, or three parts of the FP32 values.
template <class T> struct Operand;
template <> struct Operand<uint16_t> {
  v4i h;
  __device__ __forceinline__ void load(const uint16_t *p) { h = *reinterpret_cast<const v4i *>(p); }
  __device__ __forceinline__ void load_some(const uint16_t *p, int n) { // the first n
    uint16_t v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      v[i] = p[i < n ? i : 0];
#pragma unroll
    for (int w = 0; w < 4; w++)
      h[w] = (int)((2 * w < n ? v[2 * w] : 0u) | (2 * w + 1 < n ? (unsigned)v[2 * w + 1] << 16 : 0u));
  }
  __device__ __forceinline__ void keep(bool ok) {
#pragma unroll
    for (int w = 0; w < 4; w++)
      h[w] = ok ? h[w] : 0;
  }
  __device__ __forceinline__ v4f times(const v4i &bh, const v4i &bm, const v4i &bl, v4f c) const {
    c = mfma(h, bl, c);
    c = mfma(h, bm, c);
    return mfma(h, bh, c);
  }
};
template <> struct Operand<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
  }
  __device__ __forceinline__ void load_some(const float *p, int n) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      v[i] = p[i < n ? i : 0];
#pragma unroll
    for (int i = 0; i < 8; i++)
      v[i] = i < n ? v[i] : 0.0f;
    a = float4{v[0], v[1], v[2], v[3]}, b = float4{v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ void keep(bool ok) {
    a = ok ? a : float4{0.0f, 0.0f, 0.0f, 0.0f};
    b = ok ? b : float4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __device__ __forceinline__ v4f times(const v4i &bh, const v4i &bm, const v4i &bl, v4f c) const {
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    v4i h, m, l;
    parts_of(v, h, m, l);
    c = mfma(l, bh, c);
    c = mfma(h, bl, c);
    c = mfma(m, bm, c);
    c = mfma(m, bh, c);
    c = mfma(h, bm, c);
    return mfma(h, bh, c);
  }
};

struct ShrinkLds {
  int count[kMaxAdapters + 1]; // rows of each adapter, and of none
  int wave_sum[kThreads / kWave], hit[2], rows;
  Tiled::Tile tile;
};

// The batch's tile number b, of at most 64 rows: a lane a row. A row whose place among its adapter's rows is 0 or 32 begins
// a tile; tile b begins with the b-th such row. (Counting as below took 1.4 us more.)
__device__ void find_tile_of_64(const Tiled &p, ShrinkLds &sh, int b, bool &bad) {
  const int lane = threadIdx.x & (kWave - 1), m = p.job.m;
  const int id = lane < m ? p.job.adapter[lane] : INT32_MIN;
  const bool known = id >= -1 && id < p.job.adapters;
  bad = lane < m && !known;
  unsigned long long same = 0;
#pragma unroll
  for (int j = 0; j < kWave; j++)
    same |= (unsigned long long)(__builtin_amdgcn_readlane(id, j) == id) << j;
  const int place = __popcll(same & ((1ull << lane) - 1));
  const bool begins = known && place % kTileRows == 0 && !(id == -1 && p.skip_plain);
  unsigned long long begin = __ballot(begins);
  for (int i = 0; i < b && begin; i++)
    begin &= begin - 1;
  if (threadIdx.x == 0)
    sh.tile.rows = 0;
  __syncthreads();
  if (begin == 0)
    return; // fewer tiles
  const int first = __builtin_ctzll(begin), from = __shfl(place, first);
  const bool mine = known && id == __builtin_amdgcn_readlane(id, first) && place >= from && place < from + kTileRows;
  const unsigned long long rows = __ballot(mine);
  if (threadIdx.x < kWave) { // one wave writes
    if (mine)
      sh.tile.row[place - from] = lane;
    if (lane == first)
      sh.tile.adapter = id, sh.tile.rows = __popcll(rows);
  }
}

// Of any number of rows: the rows of one adapter in their order, 32 a tile, the adapters in theirs and the rows without one
// last. Rows with an id outside the table are in none (bad). A thread looks through a run of rows. Every block of
// lora_shrink does so, which grows with the square of the rows: 1100, 17600 and 70400 rows of 4096 values, rank 16, spend 15,
// 198 and 1106 us in A x, where x once is 4, 58 and 233.
__device__ void find_tile(const Tiled &p, ShrinkLds &sh, int b, bool &bad) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, m = p.job.m, bins = p.job.adapters + 1;
  for (int i = tid; i < bins; i += kThreads)
    sh.count[i] = 0;
  if (tid == 0)
    sh.hit[0] = -1, sh.tile.rows = 0;
  __syncthreads();
  auto bin_of = [&](int id) { return id == -1 ? bins - 1 : id >= 0 && id < bins - 1 ? id : -1; };
  for (int i = tid; i < m; i += kThreads) {
    const int bin = bin_of(p.job.adapter[i]);
    bad |= bin < 0;
    if (bin >= 0)
      atomicAdd(&sh.count[bin], 1);
  }
  __syncthreads();
  // a sum over the threads before this one
  auto before = [&](int v) {
    int run = v;
    for (int o = 1; o < kWave; o <<= 1) {
      const int u = __shfl_up(run, o);
      if (lane >= o)
        run += u;
    }
    if (lane == kWave - 1)
      sh.wave_sum[wave] = run;
    __syncthreads();
    run -= v;
    for (int w = 0; w < wave; w++)
      run += sh.wave_sum[w];
    return run;
  };
  const int per = (bins + kThreads - 1) / kThreads, b0 = min(tid * per, bins), b1 = min(b0 + per, bins);
  auto tiles_of = [&](int bin) {
    return bin == bins - 1 && p.skip_plain ? 0 : (sh.count[bin] + kTileRows - 1) / kTileRows;
  };
  int tiles = 0;
  for (int i = b0; i < b1; i++)
    tiles += tiles_of(i);
  int run = before(tiles);
  if (b >= run && b < run + tiles) // one thread's adapters hold the tile
    for (int i = b0; i < b1; i++) {
      const int n = tiles_of(i);
      if (b >= run && b < run + n)
        sh.hit[0] = i, sh.hit[1] = b - run;
      run += n;
    }
  __syncthreads();
  const int bin = sh.hit[0];
  if (bin < 0)
    return; // fewer tiles; uniform
  const int from = sh.hit[1] * kTileRows, rows = min(kTileRows, sh.count[bin] - from);
  if (tid == 0)
    sh.tile.adapter = bin == bins - 1 ? -1 : bin, sh.tile.rows = rows;
  const int each = (m + kThreads - 1) / kThreads, i0 = min(tid * each, m), i1 = min(i0 + each, m);
  int found = 0;
  for (int i = i0; i < i1; i++)
    found += bin_of(p.job.adapter[i]) == bin;
  int at = before(found);
  if (at < from + rows && at + found > from)
    for (int i = i0; i < i1; i++)
      if (bin_of(p.job.adapter[i]) == bin) {
        if (at >= from && at < from + rows)
          sh.tile.row[at - from] = i;
        at++;
      }
}

// One block's part of A x for RT * 16 rows and NR 16-entry tiles of A (the last ones repeated past the launch's number).
template <class T, int NR, int RT>
__device__ __forceinline__ void shrink(const Tiled &p, const Tiled::Tile &tile, int t0, int share, int b, float *red) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, lq = lane >> 4, lc = lane & 15;
  const T *a[NR];
  int all = p.first_tile[p.matrices];
#pragma unroll
  for (int i = 0; i < NR; i++) {
    const int t = min(t0 + i, all - 1);
    int matrix = 0, rank;
    while (t >= p.first_tile[matrix + 1])
      matrix++;
    const T *base = (const T *)matrix_a(p, matrix, rank);
    const int r = min(16 * (t - p.first_tile[matrix]) + lc, rank - 1); // entries past the rank are met by zeros in B
    a[i] = base + ((size_t)tile.adapter * rank + r) * p.job.k + 8 * lq;
  }
  const float *x[RT];
#pragma unroll
  for (int t = 0; t < RT; t++)
    x[t] = p.job.x + (size_t)tile.row[min(16 * t + lc, tile.rows - 1)] * p.job.ldx + 8 * lq;
  v4f acc[NR][RT];
#pragma unroll
  for (int i = 0; i < NR; i++)
#pragma unroll
    for (int t = 0; t < RT; t++)
      acc[i][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int parts = p.shares * (kThreads / kWave), part = share * (kThreads / kWave) + wave;
  const int s0 = (int)((long long)p.steps * part / parts), s1 = (int)((long long)p.steps * (part + 1) / parts);
  // a step's operands, the next one's on their way while this one's products are formed
  struct Step {
    Operand<T> w[NR];
    float4 xa[RT], xb[RT];
  };
  auto load = [&](Step &st, int s) {
    const bool inside = 32 * s + 8 * lq < p.job.k;
    const int at = inside ? 32 * s : -8 * lq; // past K the row's first values: A's are set to zero
#pragma unroll
    for (int t = 0; t < RT; t++)
      st.xa[t] = *reinterpret_cast<const float4 *>(x[t] + at), st.xb[t] = *reinterpret_cast<const float4 *>(x[t] + at + 4);
#pragma unroll
    for (int i = 0; i < NR; i++)
      st.w[i].load(a[i] + at);
  };
  auto add = [&](Step &st, int s) {
    if (p.job.k % 32) // uniform
#pragma unroll
      for (int i = 0; i < NR; i++)
        st.w[i].keep(32 * s + 8 * lq < p.job.k);
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const float v[8] = {st.xa[t].x, st.xa[t].y, st.xa[t].z, st.xa[t].w, st.xb[t].x, st.xb[t].y, st.xb[t].z, st.xb[t].w};
      v4i h, m, l;
      parts_of(v, h, m, l);
#pragma unroll
      for (int i = 0; i < NR; i++)
        acc[i][t] = st.w[i].times(h, m, l, acc[i][t]);
    }
  };
  Step one;
  if constexpr (NR <= 4) {
    Step two;
    if (s0 < s1) {
      load(one, s0);
      for (int s = s0; s < s1; s += 2) {
        load(two, min(s + 1, s1 - 1)); // unconditional: a branch would have the products wait for these loads too
        add(one, s);
        load(one, min(s + 2, s1 - 1));
        if (s + 1 < s1)
          add(two, s + 1);
      }
    }
  } else { // two steps' operands would leave one wave to a SIMD
    for (int s = s0; s < s1; s++) {
      load(one, s);
      add(one, s);
    }
  }
  // the waves' sums: 2 and 3 to 0 and 1, then 1 to 0
#pragma unroll
  for (int half = 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int i = 0; i < NR; i++)
#pragma unroll
        for (int t = 0; t < RT; t++)
          *reinterpret_cast<v4f *>(red + (((wave - half) * NR + i) * RT + t) * 4 * kWave + 4 * lane) = acc[i][t];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int i = 0; i < NR; i++)
#pragma unroll
        for (int t = 0; t < RT; t++)
          acc[i][t] += *reinterpret_cast<const v4f *>(red + ((wave * NR + i) * RT + t) * 4 * kWave + 4 * lane);
    __syncthreads();
  }
  if (wave == 0) {
    float *dst = p.low + ((size_t)share * p.tiles + b) * kTileRows * p.width;
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
      for (int t = 0; t < RT; t++)
        if (t0 + i < all && 16 * t + lc < tile.rows)
          *reinterpret_cast<v4f *>(dst + (size_t)(16 * t + lc) * p.width + 16 * (t0 + i) + 4 * lq) = acc[i][t];
  }
}

template <class T, int NR> __global__ __launch_bounds__(kThreads) void lora_shrink(Tiled p) {
  __shared__ ShrinkLds sh;
  __shared__ __align__(16) float red[2 * NR * 2 * 4 * kWave];
  const int share = blockIdx.x, b = blockIdx.y, t0 = blockIdx.z * NR;
  bool bad = false;
  if (p.job.m <= kWave)
    find_tile_of_64(p, sh, b, bad);
  else
    find_tile(p, sh, b, bad);
  if (bad && share == 0 && b == 0 && t0 == 0)
    p.flags[5] = 1;
  __syncthreads();
  if (share == 0 && t0 == 0 && threadIdx.x < sizeof(Tiled::Tile) / sizeof(int)) // for the expansion
    reinterpret_cast<int *>(p.tile + b)[threadIdx.x] = reinterpret_cast<const int *>(&sh.tile)[threadIdx.x];
  if (sh.tile.rows == 0 || sh.tile.adapter < 0)
    return;
  if (sh.tile.rows > 16)
    shrink<T, NR, 2>(p, sh.tile, t0, share, b, red);
  else
    shrink<T, NR, 1>(p, sh.tile, t0, share, b, red);
}

__global__ __launch_bounds__(kThreads) void lora_join(Tiled p) {
  const Tiled::Tile &tile = p.tile[blockIdx.y];
  const int i = 4 * (blockIdx.x * kThreads + threadIdx.x);
  if (tile.adapter < 0 || i >= tile.rows * p.width)
    return;
  const size_t at = (size_t)blockIdx.y * kTileRows * p.width + i, next = (size_t)p.tiles * kTileRows * p.width;
  v4f sum = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int s = 0; s < p.shares; s++)
    sum += *reinterpret_cast<const v4f *>(p.low + s * next + at);
  *reinterpret_cast<v4f *>(p.joined + at) = sum;
}

// Block (p.columns of a segment, tile of rows). The tile's A x goes into LDS as its three parts; a wave takes 32 columns
// at a time, two 16-column tiles; the base rows are asked for before anything else.
template <class T, bool VEC, bool RANK8> __global__ __launch_bounds__(kThreads) void lora_expand(Tiled p) {
  extern __shared__ __align__(16) unsigned char lds[];
  const Tiled::Tile &tile = p.tile[blockIdx.y];
  const int rows = tile.rows, adapter = tile.adapter;
  if (rows == 0)
    return;
  int chunk = blockIdx.x, s = 0, first_matrix = 0;
  LoraSegmentDev seg = pick(p.job, 0);
  while (chunk >= (seg.n + p.columns - 1) / p.columns) { // the segment of this block's columns
    chunk -= (seg.n + p.columns - 1) / p.columns;
    first_matrix += seg.swiglu ? 2 : 1;
    seg = pick(p.job, ++s);
  }
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, lq = lane >> 4, lc = lane & 15;
  const int parts = seg.swiglu ? 2 : 1, pad = (seg.rank + 31) / 32 * 32, stride = pad + 8;
  uint16_t *low = reinterpret_cast<uint16_t *>(lds); // [matrix][part][32][stride]
  int row_of[2]; // the lane's rows; past the tile's last, that one
#pragma unroll
  for (int t = 0; t < 2; t++)
    row_of[t] = tile.row[min(16 * t + lc, rows - 1)];
  const float scale = adapter >= 0 && seg.scale ? seg.scale[adapter] : 1.0f;
  bool staged = false;
  if (adapter >= 0) {
    // sums of the shares, split: eight entries of a row an item, zeros past the rank
    for (int i = tid; i < parts * rows * (pad / 8); i += kThreads) {
      const int r = i % (pad / 8) * 8, row = i / (pad / 8) % rows, part = i / (pad / 8) / rows;
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (r < seg.rank) {
        const float *src = p.joined + ((size_t)blockIdx.y * kTileRows + row) * p.width +
                           16 * p.first_tile[first_matrix + part] + r;
        const size_t next = (size_t)p.tiles * kTileRows * p.width;
        const int shares = p.joined == p.low ? p.shares : 1;
#pragma unroll 4
        for (int k = 0; k < shares; k++) {
          const float4 a = *reinterpret_cast<const float4 *>(src + k * next), b = *reinterpret_cast<const float4 *>(src + k * next + 4);
          v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
          v[e] = r + e < seg.rank ? v[e] : 0.0f;
      }
      v4i h, m, l;
      parts_of(v, h, m, l);
      uint16_t *dst = low + (size_t)part * 3 * kTileRows * stride + (size_t)row * stride + r;
      *reinterpret_cast<v4i *>(dst) = h;
      *reinterpret_cast<v4i *>(dst + kTileRows * stride) = m;
      *reinterpret_cast<v4i *>(dst + 2 * kTileRows * stride) = l;
    }
  }
  const int end = min(seg.n, (chunk + 1) * p.columns);
  for (int n0 = chunk * p.columns + 32 * wave; n0 < end; n0 += 32 * (kThreads / kWave)) {
    // the base rows first: they come from far
    float4 y[2][2], z[2][2];
#pragma unroll
    for (int t = 0; t < 2; t++)
      if (16 * t < rows) // uniform
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int n = n0 + 16 * c + 4 * lq;
          const size_t at = (size_t)row_of[t] * seg.ldc + (VEC ? min(n, seg.n - 4) : 0);
          if (VEC) {
            y[t][c] = *reinterpret_cast<const float4 *>(seg.base + at);
            if (seg.swiglu)
              z[t][c] = *reinterpret_cast<const float4 *>(seg.base3 + at);
          } else {
            float u[4], v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              u[e] = seg.base[at + min(n + e, seg.n - 1)];
              v[e] = seg.swiglu ? seg.base3[at + min(n + e, seg.n - 1)] : 0.0f;
            }
            y[t][c] = float4{u[0], u[1], u[2], u[3]}, z[t][c] = float4{v[0], v[1], v[2], v[3]};
          }
        }
    v4f acc[2][2][2]; // [matrix][row tile][column tile]
#pragma unroll
    for (int part = 0; part < 2; part++)
#pragma unroll
      for (int t = 0; t < 2; t++)
        acc[part][t][0] = acc[part][t][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (adapter >= 0)
      for (int r0 = 0; r0 < seg.rank; r0 += 32) {
        const int r = r0 + 8 * lq;
        Operand<T> w[2][2];
#pragma unroll
        for (int part = 0; part < 2; part++)
          if (part < parts) {
            const T *b = (const T *)(part ? seg.b3 : seg.b) + (size_t)adapter * seg.n * seg.rank;
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const int n = min(n0 + 16 * c + lc, seg.n - 1);
              const T *src = b + (size_t)n * seg.rank;
              if constexpr (RANK8) {
                w[part][c].load(src + (r < seg.rank ? r : 0));
                w[part][c].keep(r < seg.rank);
              } else {
                w[part][c].load_some(src + (r < seg.rank ? r : 0), r < seg.rank ? seg.rank - r : 0);
              }
            }
          }
        if (!staged) { // the block's first products: the parts are whole behind this barrier
          __syncthreads();
          staged = true;
        }
#pragma unroll
        for (int part = 0; part < 2; part++)
          if (part < parts) {
            const uint16_t *src = low + (size_t)part * 3 * kTileRows * stride + r;
#pragma unroll
            for (int t = 0; t < 2; t++)
              if (16 * t < rows) {
                const uint16_t *at = src + (size_t)min(16 * t + lc, rows - 1) * stride;
                const v4i h = *reinterpret_cast<const v4i *>(at), m = *reinterpret_cast<const v4i *>(at + kTileRows * stride),
                          l = *reinterpret_cast<const v4i *>(at + 2 * kTileRows * stride);
#pragma unroll
                for (int c = 0; c < 2; c++)
                  acc[part][t][c] = w[part][c].times(h, m, l, acc[part][t][c]);
              }
          }
      }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (16 * t + lc >= rows)
        continue;
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int n = n0 + 16 * c + 4 * lq;
        float u[4] = {y[t][c].x, y[t][c].y, y[t][c].z, y[t][c].w};
        const float v[4] = {z[t][c].x, z[t][c].y, z[t][c].z, z[t][c].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          u[e] = fmaf(scale, acc[0][t][c][e], u[e]);
          if (seg.swiglu)
            u[e] = silu(u[e]) * fmaf(scale, acc[1][t][c][e], v[e]);
        }
        float *dst = seg.c + (size_t)row_of[t] * seg.ldc + n;
        if (VEC) {
          if (n < end)
            *reinterpret_cast<float4 *>(dst) = float4{u[0], u[1], u[2], u[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (n + e < end)
              dst[e] = u[e];
        }
      }
    }
  }
  if (adapter >= 0 && !staged)
    __syncthreads(); // a wave without columns of its own meets the others'
}

} // namespace

// The tiled form takes rows and adapters whose K is a multiple of 8, 16-byte aligned (its loads are of eight values), at most
// 4096 adapters (counted in LDS) and 2^20 rows.
bool lora_tiled(const LoraJob &job) {
  uintptr_t all = (uintptr_t)job.x;
  for (int s = 0; s < job.nseg; s++)
    all |= (uintptr_t)job.seg[s].a | (uintptr_t)job.seg[s].a3;
  return job.k % 8 == 0 && job.ldx % 4 == 0 && (all & 15) == 0 && job.adapters <= kMaxAdapters && job.m <= (1 << 20);
}

namespace {
struct LoraShape {
  int matrices, first_tile[7], tiles, shares, width;
  bool skip_plain, join;
};
LoraShape lora_shape(const LoraJob &job) {
  LoraShape f{};
  f.skip_plain = true;
  for (int s = 0; s < job.nseg; s++) {
    const LoraSegmentDev &g = job.seg[s];
    for (int part = 0; part < (g.swiglu ? 2 : 1); part++, f.matrices++)
      f.first_tile[f.matrices + 1] = f.first_tile[f.matrices] + (g.rank + 15) / 16;
    f.skip_plain &= !g.swiglu && g.base == g.c;
  }
  f.width = 16 * f.first_tile[f.matrices];
  const int groups = job.adapters + 1 < job.m ? job.adapters + 1 : job.m;
  f.tiles = job.m / kTileRows + groups;
  // shares of K: four blocks a CU (one: 82 us for 1100 rows beside W1 and W3, two 83, four 81), each wave at least two
  // steps of 32 values
  const int cus = device().cu_count > 0 ? device().cu_count : 256, steps = (job.k + 31) / 32;
  const int most = steps / (2 * kThreads / kWave) > 1 ? steps / (2 * kThreads / kWave) : 1;
  const int want = (4 * cus + f.tiles - 1) / f.tiles;
  f.shares = want < most ? want : most;
  // joined by a launch of their own where many rows' columns would each add them again (1100 rows: 80 us, 90 without it), and
  // by the columns' blocks where the launch takes longer (32 rows: 13.3 us, 15.6 with it; one row 10.3 and 13.7)
  f.join = job.m > 64 && f.shares > 1;
  return f;
}
} // namespace

size_t lora_workspace(const LoraJob &job) {
  if (!lora_tiled(job))
    return 0;
  const LoraShape f = lora_shape(job);
  const size_t sums = (size_t)(f.shares + (f.join ? 1 : 0)) * kTileRows * f.width * sizeof(float);
  return (size_t)f.tiles * (sizeof(Tiled::Tile) + sums) + 64;
}

namespace {
template <class T> bool launch_tiled(const LoraJob &job, void *workspace, hipStream_t stream) {
  const LoraShape f = lora_shape(job);
  Tiled p{};
  p.job = job;
  p.matrices = f.matrices;
  for (int i = 0; i <= f.matrices; i++)
    p.first_tile[i] = f.first_tile[i];
  p.shares = f.shares;
  p.steps = (job.k + 31) / 32;
  p.skip_plain = f.skip_plain;
  p.tiles = f.tiles;
  p.width = f.width;
  p.tile = (Tiled::Tile *)workspace;
  p.low = (float *)(((uintptr_t)(p.tile + f.tiles) + 15) & ~(uintptr_t)15);
  p.joined = f.join ? p.low + (size_t)f.shares * f.tiles * kTileRows * f.width : p.low;
  p.flags = device().error_flags;
  const int all = f.first_tile[f.matrices];
  const int nr = all <= 1 ? 1 : all <= 3 ? 3 : all <= 4 ? 4 : 8;
  const dim3 grid((unsigned)f.shares, (unsigned)f.tiles, (unsigned)((all + nr - 1) / nr));
  const auto shrink = nr == 1 ? lora_shrink<T, 1> : nr == 3 ? lora_shrink<T, 3> : nr == 4 ? lora_shrink<T, 4> : lora_shrink<T, 8>;
  hipLaunchKernelGGL(shrink, grid, dim3(kThreads), 0, stream, p);
  if (!launch_ok("lora_shrink"))
    return false;
  if (f.join) {
    hipLaunchKernelGGL(lora_join, dim3((unsigned)((kTileRows * f.width / 4 + kThreads - 1) / kThreads), (unsigned)f.tiles),
                       dim3(kThreads), 0, stream, p);
    if (!launch_ok("lora_join"))
      return false;
  }
  // Blocks of 128 columns where few rows leave the chip idle with 256 (10 instead of 11 us for one row, 13.0 instead of 13.6
  // for 32 beside QKV); of 256 else, which stage A x half as often (1100 rows beside W1 and W3: 86 us, 88 with 128, 89 with 512).
  long wide = 0;
  for (int s = 0; s < job.nseg; s++)
    wide += (long)((job.seg[s].n + 255) / 256) * f.tiles;
  p.columns = wide >= 1024 ? 256 : 128;
  bool vec = true, rank8 = true;
  int chunks = 0, pad = 0;
  for (int s = 0; s < job.nseg; s++) {
    const LoraSegmentDev &g = job.seg[s];
    vec &= g.n % 4 == 0 && g.ldc % 4 == 0 && (((uintptr_t)g.c | (uintptr_t)g.base | (uintptr_t)g.base3) & 15) == 0;
    rank8 &= g.rank % 8 == 0 && (((uintptr_t)g.b | (uintptr_t)g.b3) & 15) == 0;
    chunks += (g.n + p.columns - 1) / p.columns;
    const int mine = (g.swiglu ? 2 : 1) * ((g.rank + 31) / 32 * 32 + 8);
    pad = mine > pad ? mine : pad;
  }
  const size_t lds = (size_t)pad * 3 * kTileRows * sizeof(uint16_t);
  static const hipError_t allowed = [] {
    hipError_t e = hipSuccess;
    for (const void *k : {(const void *)lora_expand<T, true, true>, (const void *)lora_expand<T, true, false>,
                          (const void *)lora_expand<T, false, true>, (const void *)lora_expand<T, false, false>})
      if (e == hipSuccess)
        e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * (256 + 8) * 3 * kTileRows * 2);
    return e;
  }();
  if (allowed != hipSuccess)
    return raise("allowing the adapter kernel its LDS failed: %s", hipGetErrorString(allowed));
  const auto expand = vec ? (rank8 ? lora_expand<T, true, true> : lora_expand<T, true, false>)
                          : (rank8 ? lora_expand<T, false, true> : lora_expand<T, false, false>);
  hipLaunchKernelGGL(expand, dim3((unsigned)chunks, (unsigned)f.tiles), dim3(kThreads), lds, stream, p);
  return launch_ok("lora_expand");
}
} // namespace

bool launch_lora(const LoraJob &job, void *workspace, hipStream_t stream) {
  if (lora_tiled(job))
    return job.bf16 ? launch_tiled<uint16_t>(job, workspace, stream) : launch_tiled<float>(job, workspace, stream);
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
