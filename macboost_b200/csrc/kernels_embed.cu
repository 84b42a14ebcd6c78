// Kernels of the embeddings (embed.h).
//
// forward   a group of up to 32 lanes takes a row of out, or a slab of a wide one; a lane
//           one unit of 2 to 16 bytes (four of a wide row), the ids' rows of the table
//           eight at a time.  Sums in 32 bits, in the order of j, rounded once.
// gradient  The entries are sorted by row of the table (a stable radix sort: an entry's place
//           among its equals does not depend on timing), so that a row's dout lie in one
//           stretch of the sorted list.  Groups of lanes walk chunks of 16 to 128 sorted
//           entries: a stretch inside a chunk is done, the sums of one that crosses a border
//           are joined by a second launch, 64 chunks (and 64 x 64) at a time where it is
//           long.  Every sum is in 32 bits and in one order, all groups have the same work,
//           and a stretch of millions takes no longer than one of hundreds.
//
// Measured: 65,537 x 100 ids of 12,700 x 64 float32, forward 134 us (1.7 GB of gathers from the L2
// cache, 12.5 TB/s), gradient 295 (sort 172, its walk another 1.7 GB in 130 or less, joins 30); lookup
// of 16,384 x 2,048 bfloat16 16.5 us, its gradient 125, 87 of them for clearing 537 MB (6.2 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "embed.h"
#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int kThreads = 256;

template <int BYTES>
struct Unit;
template <>
struct Unit<16> { using T = uint4; };
template <>
struct Unit<8> { using T = uint2; };
template <>
struct Unit<4> { using T = unsigned; };
template <>
struct Unit<2> { using T = unsigned short; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// Two float32 sums in one instruction.
__device__ __forceinline__ void add2(float& x, float& y, float u, float v) {
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n"
      " mov.b64 {%0, %1}, a;\n}\n"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(v));
}

// `BYTES` of adjacent values of T.
template <class T, int BYTES>
struct Values {
  static constexpr int N = BYTES / int(sizeof(T));
  static constexpr int ROWS = N > 4 ? 2 : 4;  // of a group of lanes with many ids a row
  using U = typename Unit<BYTES>::T;
  U u;
  __device__ __forceinline__ void add_to(float (&acc)[N]) const {
    T v[N];
    memcpy(v, &u, BYTES);
    if constexpr (N == 1) {
      acc[0] += to_float(v[0]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) add2(acc[i], acc[i + 1], to_float(v[i]), to_float(v[i + 1]));
    }
  }
  __device__ __forceinline__ void set(const float (&acc)[N], float scale) {
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(acc[i] * scale);
    memcpy(&u, v, BYTES);
  }
};

// The row of the table that an id looks up, -1 for none.  An id is not negative, so the sum's
// low 32 bits are all of it for a start that is not negative either, and the sum itself for
// one that is: what lies outside the table does so as an unsigned number.
__device__ __forceinline__ int looked_up(int id, int start, int entries) {
  const unsigned e = unsigned(start) + unsigned(id);
  return id >= 0 && e < unsigned(entries) ? int(e) : -1;
}

// ---- forward --------------------------------------------------------------------

// A unit a lane.
template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    embed_kernel(const EmbedArgs a, int lanes, int units, int slabs) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  constexpr int STEP = 8;
  const int lane = threadIdx.x % lanes, entries = int(a.entries);
  const long long g = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const long long n = g / slabs;
  const int u = int(g - n * slabs) * lanes + lane;
  if (n >= a.rows || u >= units) return;
  const U* table = static_cast<const U*>(a.table) + u;
  const long long ld = a.ld / V::N;
  const int* ids = a.ids + n * a.k;
  float acc[V::N];
#pragma unroll
  for (int i = 0; i < V::N; ++i) acc[i] = 0.f;
  for (int j0 = 0; j0 < int(a.k); j0 += STEP) {
    int e[STEP];
#pragma unroll
    for (int j = 0; j < STEP; ++j)
      e[j] = j0 + j < int(a.k) ? looked_up(ids[j0 + j], a.starts ? a.starts[j0 + j] : 0, entries) : -1;
    V v[STEP];
#pragma unroll
    for (int j = 0; j < STEP; ++j)
      if (e[j] >= 0) v[j].u = __ldg(table + e[j] * ld);
#pragma unroll
    for (int j = 0; j < STEP; ++j)
      if (e[j] >= 0) v[j].add_to(acc);
  }
  V v;
  v.set(acc, a.scale);
  static_cast<U*>(a.out)[n * (a.ld_out / V::N) + u] = v.u;
}

// One id a row, Q units a lane: little but the loads and stores, so that eight blocks fit a
// multiprocessor.
template <class T, int BYTES, int Q>
__global__ void __launch_bounds__(kThreads, 8)
    embed_lookup_kernel(const EmbedArgs a, int lanes, int units, int slabs) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  const int lane = threadIdx.x % lanes;
  const long long g = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const long long n = g / slabs;
  if (n >= a.rows) return;
  const int u = int(g - n * slabs) * (Q * lanes) + lane;
  const int e = looked_up(a.ids[n], a.starts ? a.starts[0] : 0, int(a.entries));
  const U* row = static_cast<const U*>(a.table) + (long long)max(e, 0) * (a.ld / V::N) + u;
  V v[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (e >= 0 && u + q * lanes < units) v[q].u = __ldg(row + q * lanes);
  U* out = static_cast<U*>(a.out) + n * (a.ld_out / V::N) + u;
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (u + q * lanes < units) {
      float acc[V::N];
#pragma unroll
      for (int i = 0; i < V::N; ++i) acc[i] = 0.f;
      if (e >= 0) v[q].add_to(acc);
      v[q].set(acc, a.scale);
      __stcs(out + q * lanes, v[q].u);
    }
}

// Many ids a row.  Each lane of a group finds the rows of the table that one id of each of the
// group's R rows looks up, and hands them round.  The rows of a block (neighbours) meet the
// same columns of ids at the same time, so a column's few rows of the table are found in
// the L1 cache.
template <class T, int BYTES, int LANES>
__global__ void __launch_bounds__(kThreads, 4) embed_many_kernel(const EmbedArgs a, int units, int slabs) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  constexpr int R = V::ROWS, STEP = 2, GROUPS = kThreads / LANES;
  const int lane = threadIdx.x % LANES;
  const long long block = blockIdx.x / slabs;
  const int u = int(blockIdx.x - block * slabs) * LANES + lane;
  const long long n0 = block * (GROUPS * R) + threadIdx.x / LANES;
  const bool there = u < units;
  const U* table = static_cast<const U*>(a.table) + (there ? u : 0);
  const unsigned ld = unsigned(a.ld / V::N);
  const int k = int(a.k), entries = int(a.entries);
  float acc[R][V::N];
  const int* ids[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ids[r] = a.ids + min(n0 + r * GROUPS, a.rows - 1) * a.k;
#pragma unroll
    for (int i = 0; i < V::N; ++i) acc[r][i] = 0.f;
  }
  for (int j0 = 0; j0 < k; j0 += LANES) {
    int mine[R];
    {
      const int at = min(j0 + lane, k - 1), start = a.starts ? __ldg(a.starts + at) : 0;
#pragma unroll
      for (int r = 0; r < R; ++r)
        mine[r] = j0 + lane < k ? looked_up(__ldg(ids[r] + at), start, entries) : -1;
    }
#pragma unroll 2
    for (int t = 0; t < LANES; t += STEP) {
      if (j0 + t >= k) break;
      int e[STEP][R];
      V v[STEP][R];
#pragma unroll
      for (int j = 0; j < STEP; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          e[j][r] = __shfl_sync(~0u, mine[r], t + j, LANES);
          if (e[j][r] >= 0) v[j][r].u = __ldg(table + (unsigned long long)unsigned(e[j][r]) * ld);
        }
#pragma unroll
      for (int j = 0; j < STEP; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (e[j][r] >= 0) v[j][r].add_to(acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long n = n0 + r * GROUPS;
    if (n >= a.rows || !there) break;
    V v;
    v.set(acc[r], a.scale);
    static_cast<U*>(a.out)[n * (a.ld_out / V::N) + u] = v.u;
  }
}

// ---- the gradient's sort ----------------------------------------------------------

struct Sort {
  // the first digit's keys come from the ids, the others' from the digit before
  const int* ids;
  const int* starts;
  HeadDiv k;                 // an entry's row
  int entries;
  const int *keys_in, *order_in;
  int *keys, *order;         // rows of the table, and of dout
  long long n;
  int shift, bits, bins, tiles;
  int *counts, *totals;      // bins x tiles, bins
};

// Entry i's row of the table (`entries` for none) and of dout.
__device__ __forceinline__ int key_of(const Sort& a, int i, int& row) {
  if (a.keys_in) {
    row = a.order_in[i];
    return a.keys_in[i];
  }
  row = a.k(i);
  const int e = looked_up(a.ids[i], a.starts ? a.starts[i - row * int(a.k.d)] : 0, a.entries);
  return e >= 0 ? e : a.entries;
}

constexpr int kSortWarps = kThreads / 32;

template <int STEPS>
__global__ void __launch_bounds__(kThreads) embed_count_kernel(const Sort a) {
  extern __shared__ int cnt[];  // bins
  const long long first = (long long)blockIdx.x * (STEPS * kThreads);
  int key[STEPS];
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const long long i = first + t * kThreads + threadIdx.x;
    int row;
    key[t] = i < a.n ? key_of(a, int(i), row) : -1;
  }
  for (int b = threadIdx.x; b < a.bins; b += kThreads) cnt[b] = 0;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STEPS; ++t)
    if (key[t] >= 0) atomicAdd(cnt + ((key[t] >> a.shift) & (a.bins - 1)), 1);  // whole numbers: in any order
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += kThreads) a.counts[(long long)b * a.tiles + blockIdx.x] = cnt[b];
}

// Inclusive sum over the block's threads; `part` holds one value a warp.
template <int THREADS>
__device__ __forceinline__ int block_sum(int v, int* part, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int p = part[w];
    if (w < warp) before += p;
    all += p;
  }
  *total = all;
  return v + before;
}

// One block a bin: its tiles' counts become running sums, its total goes to totals.
__global__ void __launch_bounds__(kThreads) embed_scan_kernel(const Sort a) {
  constexpr int PER = 8;  // adjacent values a thread
  __shared__ int part[kSortWarps];
  int* c = a.counts + (long long)blockIdx.x * a.tiles;
  int run = 0;
  for (int t0 = 0; t0 < a.tiles; t0 += kThreads * PER) {
    const int t = t0 + int(threadIdx.x) * PER;
    int v[PER], sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      v[q] = t + q < a.tiles ? c[t + q] : 0;
      sum += v[q];
    }
    int all;
    int before = run + block_sum<kThreads>(sum, part, &all) - sum;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (t + q < a.tiles) c[t + q] = before;
      before += v[q];
    }
    run += all;
  }
  if (threadIdx.x == 0) a.totals[blockIdx.x] = run;
}

// Ranks of a warp's STEPS x 32 digits of `bits` bits among its equal ones (-1: none); its
// counts end up in cnt[1 << bits].  Equal digits find each other by a ballot a bit: with many
// different ones that is several times as fast as a match.
template <int STEPS, class C>
__device__ __forceinline__ void rank_warp(int bits, int lane, C* cnt, const int (&digit)[STEPS],
                                          int (&rank)[STEPS]) {
  for (int b = lane; b < (1 << bits); b += 32) cnt[b] = 0;
  unsigned same[STEPS];
#pragma unroll
  for (int t = 0; t < STEPS; ++t) same[t] = __ballot_sync(~0u, digit[t] >= 0);
  for (int b = 0; b < bits; ++b)
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      const bool one = digit[t] >> b & 1;
      const unsigned ones = __ballot_sync(~0u, one);
      same[t] &= one ? ones : ~ones;
    }
  __syncwarp();
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const int before = __popc(same[t] & ((1u << lane) - 1u));
    const int old = digit[t] >= 0 ? int(cnt[digit[t]]) : 0;
    __syncwarp();
    if (before == 0 && digit[t] >= 0) cnt[digit[t]] = C(old + __popc(same[t]));
    __syncwarp();
    rank[t] = old + before;
  }
}

// Places of a tile's entries; a warp has STEPS x 32 consecutive ones.  They are put in order
// in shared memory first, so that what goes to one bin is written side by side.
template <int STEPS>
__global__ void __launch_bounds__(kThreads, 4) embed_place_kernel(const Sort a) {
  extern __shared__ int shared[];
  int* cnt = shared;                          // kSortWarps x bins
  int* to = cnt + kSortWarps * a.bins;        // a bin's place in the output, less its place in the tile
  int* keys = to + a.bins;                    // the tile in order
  int* rows = keys + STEPS * kThreads;
  __shared__ int part[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long tile0 = (long long)blockIdx.x * (STEPS * kThreads);
  const long long first = tile0 + warp * (STEPS * 32);
  int key[STEPS], row[STEPS], digit[STEPS], rank[STEPS];
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const long long i = first + t * 32 + lane;
    key[t] = i < a.n ? key_of(a, int(i), row[t]) : 0;
    digit[t] = i < a.n ? (key[t] >> a.shift) & (a.bins - 1) : -1;
  }
  rank_warp(a.bits, lane, cnt + warp * a.bins, digit, rank);
  __syncthreads();
  int end = 0, mine = 0;
  for (int b0 = 0; b0 < a.bins; b0 += kThreads) {
    const int b = b0 + int(threadIdx.x);
    const int n = b < a.bins ? a.totals[b] : 0;
    int all, here = 0;
    if (b < a.bins)
      for (int w = 0; w < kSortWarps; ++w) here += cnt[w * a.bins + b];
    const int start = end + block_sum<kThreads>(n, part, &all) - n;
    end += all;
    int local = mine + block_sum<kThreads>(here, part, &all) - here;
    mine += all;
    if (b < a.bins) {
      to[b] = start + a.counts[(long long)b * a.tiles + blockIdx.x] - local;
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * a.bins + b];
        cnt[w * a.bins + b] = local;
        local += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STEPS; ++t)
    if (digit[t] >= 0) {
      const int at = cnt[warp * a.bins + digit[t]] + rank[t];
      keys[at] = key[t];
      rows[at] = row[t];
    }
  __syncthreads();
  const int here = int(a.n - tile0 < STEPS * kThreads ? a.n - tile0 : STEPS * kThreads);
  for (int i = threadIdx.x; i < here; i += kThreads) {
    const int k = keys[i], at = to[(k >> a.shift) & (a.bins - 1)] + i;
    a.keys[at] = k;
    a.order[at] = rows[i];
  }
}

// Lanes, units and slabs of the rows of a matrix: `lanes` lanes and their Q units each are a slab.
struct Shape {
  int lanes, units, slabs;
  // blocks for `items` rows in groups of lanes, 0 when they are too many
  unsigned blocks(long long items) const {
    const long long per = kThreads / lanes, n = (items * slabs + per - 1) / per;
    return n > INT_MAX ? 0u : unsigned(n);
  }
};
Shape shape(long long cols, int per, int q) {
  Shape s{1, int(cols / per), 0};
  while (s.lanes < 32 && s.lanes * q < s.units) s.lanes *= 2;
  s.slabs = (s.units + q * s.lanes - 1) / (q * s.lanes);
  return s;
}

// The whole sort of up to STEPS x 1,024 entries by the first block: digits of up to
// kEmbedOneBits bits, the entries in shared memory from digit to digit.  The other blocks
// clear the table's gradient meanwhile, U a unit of its rows.
constexpr int kOneThreads = 1024;
constexpr int kOneWarps = kOneThreads / 32;
template <int STEPS>
constexpr size_t one_smem(int bits) {
  return 2 * STEPS * kOneThreads * sizeof(int) + (size_t(kOneWarps) << bits) * sizeof(unsigned short);
}
template <int STEPS, class U>
__global__ void __launch_bounds__(kOneThreads)
    embed_sort_one_kernel(const Sort a, int digits, int bits, U* clear, long long ld, int units) {
  extern __shared__ int shared[];
  if (blockIdx.x > 0) {
    U zero;
    memset(&zero, 0, sizeof(U));
    const long long all = (long long)a.entries * units, step = (long long)(gridDim.x - 1) * kOneThreads;
    long long i = (long long)(blockIdx.x - 1) * kOneThreads + threadIdx.x;
    if (ld == units) {
      for (; i < all; i += step) clear[i] = zero;
    } else {
      for (; i < all; i += step) clear[i / units * ld + i % units] = zero;
    }
    return;
  }
  int *keys = shared, *rows = keys + STEPS * kOneThreads;
  unsigned short* cnt = reinterpret_cast<unsigned short*>(rows + STEPS * kOneThreads);
  __shared__ int part[kOneWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = int(a.n), bins = 1 << bits;
  const int first = warp * (STEPS * 32);
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const int i = first + t * 32 + lane;
    if (i < n) keys[i] = key_of(a, i, rows[i]);
  }
  for (int d = 0; d < digits; ++d) {
    __syncthreads();
    int key[STEPS], row[STEPS], rank[STEPS];
    {
      int digit[STEPS];
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        const int i = first + t * 32 + lane;
        key[t] = i < n ? keys[i] : 0;
        row[t] = i < n ? rows[i] : 0;
        digit[t] = i < n ? (key[t] >> (d * bits)) & (bins - 1) : -1;
      }
      rank_warp(bits, lane, cnt + warp * bins, digit, rank);
    }
    __syncthreads();
    const int b = threadIdx.x;
    int total = 0, all;
    if (b < bins)
      for (int w = 0; w < kOneWarps; ++w) total += cnt[w * bins + b];
    int run = block_sum<kOneThreads>(total, part, &all) - total;
    if (b < bins)
      for (int w = 0; w < kOneWarps; ++w) {
        const int c = cnt[w * bins + b];
        cnt[w * bins + b] = static_cast<unsigned short>(run);
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
      if (first + t * 32 + lane < n) {
        const int at = cnt[warp * bins + ((key[t] >> (d * bits)) & (bins - 1))] + rank[t];
        keys[at] = key[t];
        rows[at] = row[t];
      }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const int i = t * kOneThreads + int(threadIdx.x);
    if (i < n) {
      a.keys[i] = keys[i];
      a.order[i] = rows[i];
    }
  }
}

// ---- the gradient's sums ----------------------------------------------------------

struct Sums {
  const int* keys;           // sorted rows of the table, n of them
  const int* order;          // the row of dout of each
  long long n;
  int chunk;
  long long chunks;
  const void* dout;
  long long ld_out;
  void* dtable;
  long long ld, entries;
  int cols;
  float scale;
  // a chunk's sum of the stretch that it begins with, if that began before it, and of the one
  // that begins in it and goes on behind it
  float *heads, *tails;
  // the chunks where a row's stretch that crosses a border begins (null, or -1 for none) and ends
  int *begins, *ends;
  float* sums[kEmbedLevels]; // sums[l][g]: of the heads g 64^(l+1) ..., all of one stretch
};

// A chunk's entries in order, a unit a lane.  LONG: stretches are long, so a chunk has few of
// them: one after the other, with nothing to look at but the rows.  Else several entries at a
// time, whatever rows of the table they are of.  From an average of 16 entries a row on: 8,192 x 100
// of 12,700 x 64 (65 a row) 105 against 130 us; 32,768 of 32,000 x 2,048 (one a row) 177 against 154.
template <class T, int BYTES, bool LONG>
__global__ void __launch_bounds__(kThreads, 4) embed_walk_kernel(const Sums a, const Shape h) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  constexpr int N = V::N, STEP = !LONG && N > 4 ? 4 : 8;
  const int lane = threadIdx.x % h.lanes;
  const long long g = (long long)blockIdx.x * (kThreads / h.lanes) + threadIdx.x / h.lanes;
  const long long c = g / h.slabs;
  const int u = int(g - c * h.slabs) * h.lanes + lane, entries = int(a.entries);
  if (c >= a.chunks || u >= h.units) return;
  const long long lo = c * a.chunk;
  const int n = int(min((long long)a.chunk, a.n - lo));
  const int *keys = a.keys + lo, *order = a.order + lo;
  const U* d = static_cast<const U*>(a.dout) + u;
  const unsigned ld = unsigned(a.ld_out / N);
  int now = keys[0];
  bool begun = lo == 0 || keys[-1] != now;  // in this chunk
  float acc[N];
  auto clear = [&] {
#pragma unroll
    for (int x = 0; x < N; ++x) acc[x] = 0.f;
  };
  // the stretch `now` ends here (in this chunk), or goes on behind it
  auto flush = [&](bool ends) {
    if (now >= entries) return;
    if (begun && ends) {
      V v;
      v.set(acc, a.scale);
      static_cast<U*>(a.dtable)[now * (a.ld / N) + u] = v.u;
    } else {
      if (u == 0) {
        if (!begun && ends) a.ends[now] = int(c);
        if (begun && a.begins) a.begins[now] = int(c);
      }
      float* to = (begun ? a.tails : a.heads) + c * a.cols + u * N;
#pragma unroll
      for (int x = 0; x < N; ++x) to[x] = acc[x];
    }
  };
  clear();
  if constexpr (LONG) {
    for (int p = 0; p < n;) {
      // the stretch's end in this chunk: the first key that is larger
      int end = p + 1, high = n;
      if (keys[n - 1] == now)
        end = n;
      else
        while (end < high) {
          const int mid = (end + high) / 2;
          if (keys[mid] > now)
            high = mid;
          else
            end = mid + 1;
        }
      if (now >= entries) return;
#pragma unroll 1
      for (; p < end; p += STEP) {
        int row[STEP];
        V v[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) row[i] = __ldg(order + min(p + i, end - 1));
#pragma unroll
        for (int i = 0; i < STEP; ++i) v[i].u = __ldg(d + (unsigned long long)unsigned(row[i]) * ld);
#pragma unroll
        for (int i = 0; i < STEP; ++i)
          if (p + i < end) v[i].add_to(acc);
      }
      p = end;
      if (p < n) {
        flush(true);
        clear();
        now = keys[p];
        begun = true;
      }
    }
  } else {
    int key[STEP], row[STEP];
    auto look = [&](int p) {
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        key[i] = p + i < n ? __ldg(keys + p + i) : entries;
        row[i] = p + i < n ? __ldg(order + p + i) : 0;
      }
    };
    look(0);
    for (int p = 0; p < n; p += STEP) {
      V v[STEP];
#pragma unroll
      for (int i = 0; i < STEP; ++i)
        if (key[i] < entries) v[i].u = __ldg(d + (unsigned long long)unsigned(row[i]) * ld);
      int k[STEP];
#pragma unroll
      for (int i = 0; i < STEP; ++i) k[i] = key[i];
      if (p + STEP < n) look(p + STEP);
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        if (p + i >= n) break;
        if (k[i] != now) {
          flush(true);
          clear();
          now = k[i];
          begun = true;
        }
        if (now < entries) v[i].add_to(acc);
      }
    }
  }
  flush(lo + n == a.n || keys[n] != now);
}

// Sums of N adjacent floats, of items `cols` apart.
template <int N>
__device__ __forceinline__ void load_sum(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int x = 0; x < N; x += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + x);
      v[x] = f.x, v[x + 1] = f.y, v[x + 2] = f.z, v[x + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int x = 0; x < N; ++x) v[x] = p[x];
  }
}

// A level's sums: group g of 64 items, if all its chunks are of one stretch that began before.
template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    embed_groups_kernel(const Sums a, int level, long long groups, const Shape h) {
  constexpr int N = Values<T, BYTES>::N, STEP = 8;
  const int lane = threadIdx.x % h.lanes;
  const long long b = (long long)blockIdx.x * (kThreads / h.lanes) + threadIdx.x / h.lanes;
  const long long g = b / h.slabs;
  const int u = int(b - g * h.slabs) * h.lanes + lane;
  if (g == 0 || g >= groups || u >= h.units) return;
  const long long span = (level ? kEmbedGroup * kEmbedGroup : kEmbedGroup) * (long long)a.chunk;
  const int key = a.keys[g * span];
  if (key >= a.entries || a.keys[g * span - 1] != key || a.keys[(g + 1) * span - 1] != key) return;
  const float* s = (level ? a.sums[0] : a.heads) + g * kEmbedGroup * a.cols + u * N;
  float acc[N];
#pragma unroll
  for (int x = 0; x < N; ++x) acc[x] = 0.f;
  for (int i = 0; i < kEmbedGroup; i += STEP) {
    float v[STEP][N];
#pragma unroll
    for (int t = 0; t < STEP; ++t) load_sum(s + (long long)(i + t) * a.cols, v[t]);
#pragma unroll
    for (int t = 0; t < STEP; ++t)
#pragma unroll
      for (int x = 0; x < N; ++x) acc[x] += v[t][x];
  }
  float* to = (level ? a.sums[1] : a.sums[0]) + g * a.cols + u * N;
#pragma unroll
  for (int x = 0; x < N; ++x) to[x] = acc[x];
}

// A stretch that crosses a border: the tail of the chunk it begins in, the heads of the chunks
// behind, and sums of 64 of them from where those begin.  An item is a row of the table
// (a.begins) or a chunk, which may have a stretch begin in it and go on behind it.
template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads, 4)
    embed_join_kernel(const Sums a, long long items, const Shape h) {
  using V = Values<T, BYTES>;
  constexpr int N = V::N, STEP = N > 4 ? 4 : 8, SQUARE = kEmbedGroup * kEmbedGroup;
  const int lane = threadIdx.x % h.lanes;
  const long long b = (long long)blockIdx.x * (kThreads / h.lanes) + threadIdx.x / h.lanes;
  const long long item = b / h.slabs;
  const int u = int(b - item * h.slabs) * h.lanes + lane;
  if (item >= items || u >= h.units) return;
  int key = int(item), c = int(item);
  if (a.begins) {
    c = a.begins[key];
    if (c < 0) return;
  } else {
    const long long lo = item * a.chunk, hi = lo + a.chunk;
    if (hi >= a.n) return;
    key = a.keys[hi - 1];
    const int first = a.keys[lo], before = lo > 0 ? a.keys[lo - 1] : -1;
    if (a.keys[hi] != key || key >= a.entries || (first == key && before == key)) return;
  }
  const int end = a.ends[key];
  float acc[N];
  load_sum(a.tails + (long long)c * a.cols + u * N, acc);
  for (int m = c + 1; m <= end;) {
    // the largest sums that begin here and leave the last chunk out, up to where larger ones may begin
    int chunks = 1;
    const float* s = a.heads;
    if (m % kEmbedGroup == 0 && end - m >= kEmbedGroup) {
      chunks = kEmbedGroup;
      s = a.sums[0];
      if (m % SQUARE == 0 && end - m >= SQUARE) {
        chunks = SQUARE;
        s = a.sums[1];
      }
    }
    const int at = m / chunks;
    int n = chunks == 1 ? end - m + 1 : (end - m) / chunks;
    if (chunks < SQUARE) n = min(n, kEmbedGroup - at % kEmbedGroup);
    s += (long long)at * a.cols + u * N;
    for (int t0 = 0; t0 < n; t0 += STEP) {
      float v[STEP][N];
#pragma unroll
      for (int t = 0; t < STEP; ++t) load_sum(s + (long long)min(t0 + t, n - 1) * a.cols, v[t]);
#pragma unroll
      for (int t = 0; t < STEP; ++t)
        if (t0 + t < n)
#pragma unroll
          for (int x = 0; x < N; ++x) acc[x] += v[t][x];
    }
    m += n * chunks;
  }
  V v;
  v.set(acc, a.scale);
  static_cast<typename V::U*>(a.dtable)[key * (a.ld / N) + u] = v.u;
}

// ---- launches -----------------------------------------------------------------------

int unit_bytes(uintptr_t all) { return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2; }

template <class T, int BYTES>
cudaError_t forward(const EmbedArgs& a, cudaStream_t s) {
  constexpr int N = BYTES / int(sizeof(T));
  if (a.k == 1) {
    // Four units a lane where the GPU stays full: in us, against one, 65,536 rows of 512 bfloat16 16.3 and
    // 28.8, 262,144 of 64 float32 14.5 and 26.7, 16,384 of 2,048 bfloat16 16.5 and 28.9 (4.1 TB/s
    // stored); 4,096 of 256 float32 4.2 and 4.2.
    const bool wide = a.cols / N >= 8 && a.rows * (a.cols / N) >= 2ll * kThreads * device_sms();
    const Shape h = shape(a.cols, N, wide ? 4 : 1);
    const unsigned blocks = h.blocks(a.rows);
    if (!blocks) return cudaErrorInvalidValue;
    if (wide)
      embed_lookup_kernel<T, BYTES, 4><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
    else
      embed_lookup_kernel<T, BYTES, 1><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
    return cudaGetLastError();
  }
  const Shape h = shape(a.cols, N, 1);
  // Several rows a group where that leaves enough of them for the GPU: in us, against one, 65,536 x 4 of
  // 40,000 x 64 float32 12.5 and 22.7, 8,192 x 32 of 12,700 x 512 bfloat16 24.7 and 40.2, 65,537 x 100 of
  // 12,700 x 64 float32 134 and 170; 8,192 x 100 of these (128 blocks) 41 and 33.
  const long long tile = Values<T, BYTES>::ROWS * (kThreads / h.lanes), many = (a.rows + tile - 1) / tile * h.slabs;
  if (h.lanes >= 8 && many >= 4 * device_sms() && many <= INT_MAX) {
    const unsigned blocks = unsigned(many);
    if (h.lanes == 8)
      embed_many_kernel<T, BYTES, 8><<<blocks, kThreads, 0, s>>>(a, h.units, h.slabs);
    else if (h.lanes == 16)
      embed_many_kernel<T, BYTES, 16><<<blocks, kThreads, 0, s>>>(a, h.units, h.slabs);
    else
      embed_many_kernel<T, BYTES, 32><<<blocks, kThreads, 0, s>>>(a, h.units, h.slabs);
    return cudaGetLastError();
  }
  const unsigned blocks = h.blocks(a.rows);
  if (!blocks) return cudaErrorInvalidValue;
  embed_kernel<T, BYTES><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
  return cudaGetLastError();
}

template <class T, int BYTES>
cudaError_t walk(const Sums& a, bool stretches, cudaStream_t s) {
  const Shape h = shape(a.cols, BYTES / int(sizeof(T)), 1);
  const unsigned blocks = h.blocks(a.chunks);
  if (!blocks) return cudaErrorInvalidValue;
  if (stretches)
    embed_walk_kernel<T, BYTES, true><<<blocks, kThreads, 0, s>>>(a, h);
  else
    embed_walk_kernel<T, BYTES, false><<<blocks, kThreads, 0, s>>>(a, h);
  return cudaGetLastError();
}

template <int STEPS, class U>
cudaError_t sort_one(const Sort& t, const EmbedPlan& p, const EmbedArgs& a, int per, cudaStream_t s) {
  // the limit of the largest call: it is the kernel's, and other threads launch it too
  const auto k = embed_sort_one_kernel<STEPS, U>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             int(one_smem<STEPS>(kEmbedOneBits)));
  if (e != cudaSuccess) return e;
  const long long units = a.cols / per;
  // two blocks a multiprocessor keep the stores coming
  const long long fill = (a.entries * units + 4 * kOneThreads - 1) / (4 * kOneThreads);
  const int blocks = 1 + int(std::min<long long>(fill, 2 * device_sms() - 2));
  k<<<blocks, kOneThreads, one_smem<STEPS>(p.bits), s>>>(t, p.digits, p.bits, static_cast<U*>(a.dtable), a.ld / per,
                                                         int(units));
  return cudaGetLastError();
}

template <int STEPS>
cudaError_t sort_tiles(const Sort& t, cudaStream_t s) {
  const auto smem = [](int bins) { return ((kSortWarps + 1) * size_t(bins) + 2 * STEPS * kThreads) * sizeof(int); };
  const cudaError_t e = cudaFuncSetAttribute(embed_place_kernel<STEPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             int(smem(1024)));
  if (e != cudaSuccess) return e;
  embed_count_kernel<STEPS><<<t.tiles, kThreads, size_t(t.bins) * sizeof(int), s>>>(t);
  embed_scan_kernel<<<t.bins, kThreads, 0, s>>>(t);
  embed_place_kernel<STEPS><<<t.tiles, kThreads, smem(t.bins), s>>>(t);
  return cudaGetLastError();
}

template <class T, int BYTES>
cudaError_t gradient(const EmbedArgs& a, const EmbedPlan& p, int* launches, cudaStream_t s) {
  using U = typename Unit<BYTES>::T;
  constexpr int N = BYTES / int(sizeof(T));
  char* base = static_cast<char*>(a.workspace);
  auto ints = [&](long long at) { return reinterpret_cast<int*>(base + at); };
  Sort t{};
  t.ids = a.ids;
  t.starts = a.starts;
  t.k.set(a.k);
  t.entries = int(a.entries);
  t.n = p.n;
  t.bits = p.bits;
  t.bins = 1 << p.bits;
  t.tiles = p.tiles;
  t.counts = ints(p.counts);
  t.totals = ints(p.totals);
  cudaError_t e = cudaSuccess;
  // rows that no id leads to; the one-launch sort clears them itself
  if (!p.one)
    e = cudaMemset2DAsync(a.dtable, size_t(a.ld) * sizeof(T), 0, size_t(a.cols) * sizeof(T), size_t(a.entries), s);
  if (e != cudaSuccess) return e;
  int now = 0;
  if (p.one) {
    t.keys = ints(p.keys[0]);
    t.order = ints(p.order[0]);
    e = p.n <= kEmbedOne / 4 ? sort_one<kEmbedOne / 4 / kOneThreads, U>(t, p, a, N, s)
                             : sort_one<kEmbedOne / kOneThreads, U>(t, p, a, N, s);
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  for (int d = 0; d < p.digits && !p.one; ++d) {
    now = d % 2;
    t.keys_in = d ? ints(p.keys[now ^ 1]) : nullptr;
    t.order_in = d ? ints(p.order[now ^ 1]) : nullptr;
    t.keys = ints(p.keys[now]);
    t.order = ints(p.order[now]);
    t.shift = d * p.bits;
    e = sort_tiles<kEmbedTile / kThreads>(t, s);
    if (e != cudaSuccess) return e;
    *launches += 3;
  }
  Sums q{};
  q.keys = ints(p.keys[now]);
  q.order = ints(p.order[now]);
  q.n = p.n;
  q.chunk = p.chunk;
  q.chunks = p.chunks;
  q.dout = a.dout;
  q.ld_out = a.ld_out;
  q.dtable = a.dtable;
  q.ld = a.ld;
  q.entries = a.entries;
  q.cols = int(a.cols);
  q.scale = a.scale;
  q.heads = reinterpret_cast<float*>(base + p.heads);
  q.tails = reinterpret_cast<float*>(base + p.tails);
  q.begins = p.by_row ? ints(p.begins) : nullptr;
  q.ends = ints(p.ends);
  if (p.by_row) {
    e = cudaMemsetAsync(q.begins, 0xFF, size_t(a.entries) * 4, s);
    if (e != cudaSuccess) return e;
  }
  for (int l = 0; l < kEmbedLevels; ++l) q.sums[l] = reinterpret_cast<float*>(base + p.sums[l]);
  e = walk<T, BYTES>(q, p.stretches, s);
  if (e != cudaSuccess) return e;
  ++*launches;
  if (p.chunks < 2) return cudaSuccess;
  const Shape h = shape(a.cols, N, 1);
  for (int l = 0; l < kEmbedLevels && p.groups[l] > 1; ++l) {
    const unsigned blocks = h.blocks(p.groups[l]);
    if (!blocks) return cudaErrorInvalidValue;
    embed_groups_kernel<T, BYTES><<<blocks, kThreads, 0, s>>>(q, l, p.groups[l], h);
    ++*launches;
  }
  const long long items = p.by_row ? a.entries : p.chunks;
  const unsigned blocks = h.blocks(items);
  if (!blocks) return cudaErrorInvalidValue;
  embed_join_kernel<T, BYTES><<<blocks, kThreads, 0, s>>>(q, items, h);
  ++*launches;
  return cudaGetLastError();
}

template <class T>
cudaError_t forward_of(const EmbedArgs& a, int bytes, cudaStream_t s) {
  switch (bytes) {
    case 16: return forward<T, 16>(a, s);
    case 8: return forward<T, 8>(a, s);
    case 4: return forward<T, 4>(a, s);
    default: break;
  }
  if constexpr (sizeof(T) == 2) return forward<T, 2>(a, s);
  return cudaErrorInvalidValue;
}
template <class T>
cudaError_t gradient_of(const EmbedArgs& a, const EmbedPlan& p, int bytes, int* launches, cudaStream_t s) {
  switch (bytes) {
    case 16: return gradient<T, 16>(a, p, launches, s);
    case 8: return gradient<T, 8>(a, p, launches, s);
    case 4: return gradient<T, 4>(a, p, launches, s);
    default: break;
  }
  if constexpr (sizeof(T) == 2) return gradient<T, 2>(a, p, launches, s);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_embed(const EmbedArgs& a, cudaStream_t s) {
  const uintptr_t size = uintptr_t(dtype_bytes(a.dtype));
  const int bytes = unit_bytes(reinterpret_cast<uintptr_t>(a.table) | reinterpret_cast<uintptr_t>(a.out) |
                               uintptr_t(a.ld) * size | uintptr_t(a.ld_out) * size | uintptr_t(a.cols) * size);
  if (a.dtype == kF32) return forward_of<float>(a, bytes, s);
  if (a.dtype == kBF16) return forward_of<__nv_bfloat16>(a, bytes, s);
  return forward_of<__half>(a, bytes, s);
}

cudaError_t launch_embed_grad(const EmbedArgs& a, const EmbedPlan& p, int* launches, cudaStream_t s) {
  const uintptr_t size = uintptr_t(dtype_bytes(a.dtype));
  const int bytes = unit_bytes(reinterpret_cast<uintptr_t>(a.dout) | reinterpret_cast<uintptr_t>(a.dtable) |
                               uintptr_t(a.ld) * size | uintptr_t(a.ld_out) * size | uintptr_t(a.cols) * size);
  if (a.dtype == kF32) return gradient_of<float>(a, p, bytes, launches, s);
  if (a.dtype == kBF16) return gradient_of<__nv_bfloat16>(a, p, bytes, launches, s);
  return gradient_of<__half>(a, p, bytes, launches, s);
}

}  // namespace mb
