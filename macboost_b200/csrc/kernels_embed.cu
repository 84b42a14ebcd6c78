// Kernels of the embeddings (embed.h).
//
// forward   a group of up to 32 lanes takes a row of out, or a slab of a wide one; a lane
//           one unit of 2 to 16 bytes (four of a wide row), the ids' rows of the table
//           eight at a time.  Sums in 32 bits, in the order of j, rounded once.
// gradient  The entries are sorted by row of the table (a stable radix sort: an entry's place
//           among its equals does not depend on timing), so that a row's dout lie in one
//           stretch of the sorted list.  Parts of 64 positions that lie within one stretch
//           are added up first, then 64 of these sums, then 64 of those; a row adds what
//           its stretch begins and ends with and the sums between.  Every sum is in 32 bits
//           and in one order, and a stretch of millions is no longer than one of hundreds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "embed.h"
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

// `BYTES` of adjacent values of T.
template <class T, int BYTES>
struct Values {
  static constexpr int N = BYTES / int(sizeof(T));
  using U = typename Unit<BYTES>::T;
  U u;
  __device__ __forceinline__ void add_to(float (&acc)[N]) const {
    T v[N];
    memcpy(v, &u, BYTES);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += to_float(v[i]);
  }
  __device__ __forceinline__ void set(const float (&acc)[N], float scale) {
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(acc[i] * scale);
    memcpy(&u, v, BYTES);
  }
};

// The row of the table that id j of a row looks up, -1 for none.
__device__ __forceinline__ long long looked_up(int id, int start, long long entries) {
  const long long e = (long long)start + id;
  return id >= 0 && e >= 0 && e < entries ? e : -1;
}

// ---- forward --------------------------------------------------------------------

// Q units a lane, `lanes` apart; slabs of Q * lanes units.
template <class T, int BYTES, int Q>
__global__ void __launch_bounds__(kThreads)
    embed_kernel(const EmbedArgs a, int lanes, int units, int slabs) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  constexpr int STEP = Q > 1 ? 2 : 8;
  const int lane = threadIdx.x % lanes;
  const long long g = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const long long n = g / slabs;
  if (n >= a.rows) return;
  const int u0 = int(g - n * slabs) * (Q * lanes) + lane;
  const U* table = static_cast<const U*>(a.table);
  const long long ld = a.ld / V::N;
  const int* ids = a.ids + n * a.k;
  float acc[Q][V::N];
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int i = 0; i < V::N; ++i) acc[q][i] = 0.f;
  for (int j0 = 0; j0 < int(a.k); j0 += STEP) {
    long long e[STEP];
#pragma unroll
    for (int j = 0; j < STEP; ++j)
      e[j] = j0 + j < int(a.k) ? looked_up(ids[j0 + j], a.starts ? a.starts[j0 + j] : 0, a.entries) : -1;
    V v[STEP][Q];
#pragma unroll
    for (int j = 0; j < STEP; ++j)
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (e[j] >= 0 && u0 + q * lanes < units) v[j][q].u = __ldg(table + e[j] * ld + u0 + q * lanes);
#pragma unroll
    for (int j = 0; j < STEP; ++j)
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (e[j] >= 0 && u0 + q * lanes < units) v[j][q].add_to(acc[q]);
  }
  U* out = static_cast<U*>(a.out) + n * (a.ld_out / V::N);
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (u0 + q * lanes < units) {
      V v;
      v.set(acc[q], a.scale);
      out[u0 + q * lanes] = v.u;
    }
}

// ---- the gradient's sort ----------------------------------------------------------

struct Sort {
  // the first digit's keys come from the ids, the others' from the digit before
  const int* ids;
  const int* starts;
  int k, entries;
  const int *keys_in, *order_in;
  int *keys, *order;
  long long n;
  int shift, bins, tiles;
  int *counts, *totals;      // bins x tiles, bins
  int last;                  // order gets the row of dout in place of the entry
};

__device__ __forceinline__ int key_of(const Sort& a, long long i) {
  if (a.keys_in) return a.keys_in[i];
  const int start = a.starts ? a.starts[unsigned(i) % unsigned(a.k)] : 0;
  const long long e = looked_up(a.ids[i], start, a.entries);
  return e >= 0 ? int(e) : a.entries;
}

constexpr int kSortWarps = kThreads / 32;
constexpr int kSortSteps = kEmbedTile / kThreads;

__global__ void __launch_bounds__(kThreads) embed_count_kernel(const Sort a) {
  extern __shared__ int cnt[];  // bins
  for (int b = threadIdx.x; b < a.bins; b += kThreads) cnt[b] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * kEmbedTile;
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const long long i = first + t * kThreads + threadIdx.x;
    if (i < a.n) atomicAdd(cnt + ((key_of(a, i) >> a.shift) & (a.bins - 1)), 1);  // whole numbers: in any order
  }
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

// Ranks of a warp's STEPS x 32 digits among its equal ones (-1: none); its counts end up
// in cnt[bins].
template <int STEPS>
__device__ __forceinline__ void rank_warp(int bins, int lane, int* cnt, const int (&digit)[STEPS],
                                          int (&rank)[STEPS]) {
  for (int b = lane; b < bins; b += 32) cnt[b] = 0;
  __syncwarp();
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const unsigned same = __match_any_sync(~0u, digit[t]);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int old = digit[t] >= 0 ? cnt[digit[t]] : 0;
    __syncwarp();
    if (before == 0 && digit[t] >= 0) cnt[digit[t]] = old + __popc(same);
    __syncwarp();
    rank[t] = old + before;
  }
}

// Places of a tile's entries.  A warp has kSortSteps x 32 consecutive ones.
__global__ void __launch_bounds__(kThreads) embed_place_kernel(const Sort a) {
  extern __shared__ int cnt[];  // kSortWarps x bins
  __shared__ int part[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long first = (long long)blockIdx.x * kEmbedTile + warp * (kSortSteps * 32);
  int key[kSortSteps], digit[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const long long i = first + t * 32 + lane;
    key[t] = i < a.n ? key_of(a, i) : 0;
    digit[t] = i < a.n ? (key[t] >> a.shift) & (a.bins - 1) : -1;
  }
  rank_warp(a.bins, lane, cnt + warp * a.bins, digit, rank);
  __syncthreads();
  int end = 0;
  for (int b0 = 0; b0 < a.bins; b0 += kThreads) {
    const int b = b0 + int(threadIdx.x);
    const int n = b < a.bins ? a.totals[b] : 0;
    int all;
    int run = end + block_sum<kThreads>(n, part, &all) - n;
    end += all;
    if (b < a.bins) {
      run += a.counts[(long long)b * a.tiles + blockIdx.x];
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * a.bins + b];
        cnt[w * a.bins + b] = run;
        run += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const long long i = first + t * 32 + lane;
    if (i < a.n) {
      const int at = cnt[warp * a.bins + digit[t]] + rank[t];
      const int e = a.order_in ? a.order_in[i] : int(i);
      a.keys[at] = key[t];
      a.order[at] = a.last ? int(unsigned(e) / unsigned(a.k)) : e;
    }
  }
}

// The whole sort of up to kEmbedOne entries: digits of at most 8 bits, the entries in
// shared memory from digit to digit.
constexpr int kOneThreads = 512;
constexpr int kOneWarps = kOneThreads / 32;
constexpr int kOneSteps = kEmbedOne / kOneThreads;
constexpr size_t kOneSmem = (2 * kEmbedOne + kOneWarps * 256) * sizeof(int);
__global__ void __launch_bounds__(kOneThreads) embed_sort_one_kernel(const Sort a, int digits, int bits) {
  extern __shared__ int shared[];
  int *keys = shared, *order = keys + kEmbedOne, *cnt = order + kEmbedOne;
  __shared__ int part[kOneWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = int(a.n), bins = 1 << bits;
  const int first = warp * (kOneSteps * 32);
  int key[kOneSteps], entry[kOneSteps];
#pragma unroll
  for (int t = 0; t < kOneSteps; ++t) {
    const int i = first + t * 32 + lane;
    key[t] = i < n ? key_of(a, i) : 0;
    entry[t] = i;
  }
  for (int d = 0; d < digits; ++d) {
    int digit[kOneSteps], rank[kOneSteps];
#pragma unroll
    for (int t = 0; t < kOneSteps; ++t)
      digit[t] = first + t * 32 + lane < n ? (key[t] >> (d * bits)) & (bins - 1) : -1;
    rank_warp(bins, lane, cnt + warp * bins, digit, rank);
    __syncthreads();
    const int b = threadIdx.x;
    int total = 0;
    if (b < bins)
      for (int w = 0; w < kOneWarps; ++w) total += cnt[w * bins + b];
    int all;
    int run = block_sum<kOneThreads>(total, part, &all) - total;
    if (b < bins)
      for (int w = 0; w < kOneWarps; ++w) {
        const int c = cnt[w * bins + b];
        cnt[w * bins + b] = run;
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kOneSteps; ++t)
      if (digit[t] >= 0) {
        const int at = cnt[warp * bins + digit[t]] + rank[t];
        keys[at] = key[t];
        order[at] = entry[t];
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kOneSteps; ++t) {
      const int i = first + t * 32 + lane;
      if (i < n) {
        key[t] = keys[i];
        entry[t] = order[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < kOneSteps; ++t) {
    const int i = first + t * 32 + lane;
    if (i < n) {
      a.keys[i] = key[t];
      a.order[i] = entry[t] / a.k;
    }
  }
}

// ---- the gradient's sums ----------------------------------------------------------

struct Sums {
  const int* keys;           // sorted rows of the table, n of them
  const int* order;          // the row of dout of each
  long long n;
  const void* dout;
  long long ld_out;
  void* dtable;
  long long ld, entries;
  int cols;
  float scale;
  int *first, *last;         // a row's stretch: first is -1 for none
  float* part[kEmbedLevels]; // part[l][c]: the sum of positions c 64^(l+1) ... of one row
};

// acc += the items lo ... hi - 1 of a level: rows of dout (level 0), or sums below.
template <class T, int BYTES>
__device__ __forceinline__ void add_items(const Sums& a, int level, long long lo, long long hi, int u,
                                          float (&acc)[Values<T, BYTES>::N]) {
  using V = Values<T, BYTES>;
  using U = typename V::U;
  constexpr int STEP = 8;
  if (level == 0) {
    const U* d = static_cast<const U*>(a.dout) + u;
    const long long ld = a.ld_out / V::N;
    for (; lo + STEP <= hi; lo += STEP) {
      int r[STEP];
      V v[STEP];
#pragma unroll
      for (int i = 0; i < STEP; ++i) r[i] = __ldg(a.order + lo + i);
#pragma unroll
      for (int i = 0; i < STEP; ++i) v[i].u = __ldg(d + r[i] * ld);
#pragma unroll
      for (int i = 0; i < STEP; ++i) v[i].add_to(acc);
    }
    for (; lo < hi; ++lo) {
      V v;
      v.u = __ldg(d + __ldg(a.order + lo) * ld);
      v.add_to(acc);
    }
    return;
  }
  const float* s = a.part[level - 1] + u * V::N;
  for (; lo + STEP <= hi; lo += STEP) {
    float v[STEP][V::N];
#pragma unroll
    for (int i = 0; i < STEP; ++i)
#pragma unroll
      for (int q = 0; q < V::N; ++q) v[i][q] = s[(lo + i) * a.cols + q];
#pragma unroll
    for (int i = 0; i < STEP; ++i)
#pragma unroll
      for (int q = 0; q < V::N; ++q) acc[q] += v[i][q];
  }
  for (; lo < hi; ++lo)
#pragma unroll
    for (int q = 0; q < V::N; ++q) acc[q] += s[lo * a.cols + q];
}

// A level's sums: part c of 64 items, if all 64^(level+1) positions are of one row.
template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    embed_parts_kernel(const Sums a, int level, long long parts, int lanes, int units, int slabs) {
  constexpr int N = Values<T, BYTES>::N;
  const int lane = threadIdx.x % lanes;
  const long long g = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const long long c = g / slabs;
  if (c >= parts) return;
  const int u = int(g - c * slabs) * lanes + lane;
  long long span = kEmbedPart;
  for (int l = 0; l < level; ++l) span *= kEmbedPart;
  const int key = a.keys[c * span];
  if (u >= units || key >= a.entries || key != a.keys[(c + 1) * span - 1]) return;
  float acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = 0.f;
  add_items<T, BYTES>(a, level, c * kEmbedPart, (c + 1) * kEmbedPart, u, acc);
  float* to = a.part[level] + c * a.cols + u * N;
#pragma unroll
  for (int q = 0; q < N; ++q) to[q] = acc[q];
}

// Where each row's stretch begins and ends.
__global__ void __launch_bounds__(kThreads) embed_stretch_kernel(const Sums a) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n) return;
  const int key = a.keys[i];
  if (key >= a.entries) return;
  if (i == 0 || a.keys[i - 1] != key) a.first[key] = int(i);
  if (i + 1 == a.n || a.keys[i + 1] != key) a.last[key] = int(i + 1);
}

template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    embed_rows_kernel(const Sums a, int lanes, int units, int slabs) {
  using V = Values<T, BYTES>;
  const int lane = threadIdx.x % lanes;
  const long long g = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const long long e = g / slabs;
  if (e >= a.entries) return;
  const int u = int(g - e * slabs) * lanes + lane;
  if (u >= units) return;
  float acc[V::N];
#pragma unroll
  for (int q = 0; q < V::N; ++q) acc[q] = 0.f;
  const int first = a.first[e];
  if (first >= 0) {
    long long lo = first, hi = a.last[e];
    for (int level = 0;; ++level) {
      const long long b = (lo + kEmbedPart - 1) / kEmbedPart, c = hi / kEmbedPart;
      if (level == kEmbedLevels || b >= c) {
        add_items<T, BYTES>(a, level, lo, hi, u, acc);
        break;
      }
      add_items<T, BYTES>(a, level, lo, b * kEmbedPart, u, acc);
      add_items<T, BYTES>(a, level, c * kEmbedPart, hi, u, acc);
      lo = b;
      hi = c;
    }
  }
  V v;
  v.set(acc, a.scale);
  static_cast<typename V::U*>(a.dtable)[e * (a.ld / V::N) + u] = v.u;
}

// ---- launches -----------------------------------------------------------------------

struct Shape {
  int lanes, units, slabs;
  // blocks for `items` groups of slabs, 0 when they are too many
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

int unit_bytes(uintptr_t all) { return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2; }

template <class T, int BYTES>
cudaError_t forward(const EmbedArgs& a, cudaStream_t s) {
  constexpr int N = BYTES / int(sizeof(T));
  // four units a lane where a row has that many for every lane and few rows are added up
  const bool wide = a.k < 4 && a.cols / N >= 128 && a.rows * (a.cols / N) >= 4ll * kThreads * device_sms();
  const Shape h = shape(a.cols, N, wide ? 4 : 1);
  const unsigned blocks = h.blocks(a.rows);
  if (!blocks) return cudaErrorInvalidValue;
  if (wide)
    embed_kernel<T, BYTES, 4><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
  else
    embed_kernel<T, BYTES, 1><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
  return cudaGetLastError();
}

template <class T, int BYTES>
cudaError_t sums(const Sums& a, const EmbedPlan& p, int* launches, cudaStream_t s) {
  const Shape h = shape(a.cols, BYTES / int(sizeof(T)), 1);
  for (int l = 0; l < kEmbedLevels && p.parts[l] > 0; ++l) {
    const unsigned blocks = h.blocks(p.parts[l]);
    if (!blocks) return cudaErrorInvalidValue;
    embed_parts_kernel<T, BYTES><<<blocks, kThreads, 0, s>>>(a, l, p.parts[l], h.lanes, h.units, h.slabs);
    ++*launches;
  }
  const unsigned blocks = h.blocks(a.entries);
  if (!blocks) return cudaErrorInvalidValue;
  embed_rows_kernel<T, BYTES><<<blocks, kThreads, 0, s>>>(a, h.lanes, h.units, h.slabs);
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
cudaError_t sums_of(const Sums& a, const EmbedPlan& p, int bytes, int* launches, cudaStream_t s) {
  switch (bytes) {
    case 16: return sums<T, 16>(a, p, launches, s);
    case 8: return sums<T, 8>(a, p, launches, s);
    case 4: return sums<T, 4>(a, p, launches, s);
    default: break;
  }
  if constexpr (sizeof(T) == 2) return sums<T, 2>(a, p, launches, s);
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
  char* base = static_cast<char*>(a.workspace);
  auto ints = [&](long long at) { return reinterpret_cast<int*>(base + at); };
  cudaError_t e = cudaMemsetAsync(base + p.first, 0xFF, size_t(a.entries) * 4, s);
  if (e != cudaSuccess) return e;
  Sort t{};
  t.ids = a.ids;
  t.starts = a.starts;
  t.k = int(a.k);
  t.entries = int(a.entries);
  t.n = p.n;
  t.bins = 1 << p.bits;
  t.tiles = p.tiles;
  t.counts = ints(p.counts);
  t.totals = ints(p.totals);
  int now = 0;
  if (p.n <= kEmbedOne) {
    t.keys = ints(p.keys[0]);
    t.order = ints(p.order[0]);
    e = cudaFuncSetAttribute(embed_sort_one_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kOneSmem));
    if (e != cudaSuccess) return e;
    embed_sort_one_kernel<<<1, kOneThreads, kOneSmem, s>>>(t, p.digits, p.bits);
    ++*launches;
  } else {
    for (int d = 0; d < p.digits; ++d) {
      now = d % 2;
      t.keys_in = d ? ints(p.keys[now ^ 1]) : nullptr;
      t.order_in = d ? ints(p.order[now ^ 1]) : nullptr;
      t.keys = ints(p.keys[now]);
      t.order = ints(p.order[now]);
      t.shift = d * p.bits;
      t.last = d + 1 == p.digits;
      const size_t bins = size_t(t.bins) * sizeof(int);
      embed_count_kernel<<<p.tiles, kThreads, bins, s>>>(t);
      embed_scan_kernel<<<t.bins, kThreads, 0, s>>>(t);
      embed_place_kernel<<<p.tiles, kThreads, kSortWarps * bins, s>>>(t);  // at most 32 KB
      *launches += 3;
    }
  }
  Sums q{};
  q.keys = ints(p.keys[now]);
  q.order = ints(p.order[now]);
  q.n = p.n;
  q.dout = a.dout;
  q.ld_out = a.ld_out;
  q.dtable = a.dtable;
  q.ld = a.ld;
  q.entries = a.entries;
  q.cols = int(a.cols);
  q.scale = a.scale;
  q.first = ints(p.first);
  q.last = ints(p.last);
  for (int l = 0; l < kEmbedLevels; ++l) q.part[l] = reinterpret_cast<float*>(base + p.sums[l]);
  embed_stretch_kernel<<<unsigned((p.n + kThreads - 1) / kThreads), kThreads, 0, s>>>(q);
  ++*launches;
  const uintptr_t size = uintptr_t(dtype_bytes(a.dtype));
  const int bytes = unit_bytes(reinterpret_cast<uintptr_t>(a.dout) | reinterpret_cast<uintptr_t>(a.dtable) |
                               uintptr_t(a.ld) * size | uintptr_t(a.ld_out) * size | uintptr_t(a.cols) * size);
  if (a.dtype == kF32) return sums_of<float>(q, p, bytes, launches, s);
  if (a.dtype == kBF16) return sums_of<__nv_bfloat16>(q, p, bytes, launches, s);
  return sums_of<__half>(q, p, bytes, launches, s);
}

}  // namespace mb
