// Rows sorted by model, gathered into each model's segment, and the models'
// outputs combined again, with the gradient (mixture.h).
//
// sort     A stable counting sort.  A tile of 4,096 entries belongs to a block, 512
//          consecutive ones to a warp; lanes with equal ids find each other with a
//          match and rank themselves by lane, so an entry's place among its
//          warp's equals is known without an atomic and the result is the same
//          every time.  Up to one tile: one launch.  More: counts of each (expert,
//          tile), their running sums per expert, then the places.
// gather   out[slot] = x[row of the entry in slot], zeros in a slot without entry.
//          Row-major to row-major reads every row once and writes it to its k
//          slots; the forms with a feature-major side go through a tile in shared
//          memory, or column by column.
// combine  out[n] = sum_j w[n, j] y[slot[n, j]], summed in 32 bits in the order of j.
// gradient dy[slot[n, j]] = w[n, j] dout[n], dw[n, j] = <dout[n], y[slot[n, j]]>, and
//          zeros in the rows of dy that hold no entry.
//
// All of it moves bytes and is bound by them: the unit of a copy is the largest of
// 16, 8, 4 and 2 bytes that the addresses, strides and row lengths share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>

#include "mixture.h"

namespace mb {

namespace {

// ---- sort -------------------------------------------------------------------

constexpr int kSortWarps = 8;
constexpr int kSortSteps = 16;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kSortTile = kSortThreads * kSortSteps;  // entries a block

// Ranks of a warp's 512 entries among its equal ids; its counts end up in cnt[E].
__device__ __forceinline__ void rank_warp(const SortArgs& a, long long first, int lane, int* cnt,
                                          int (&id)[kSortSteps], int (&rank)[kSortSteps]) {
  for (int e = lane; e < a.experts; e += 32) cnt[e] = 0;
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const long long i = first + t * 32 + lane;
    const int v = i < a.entries ? a.ids[i] : -1;
    id[t] = unsigned(v) < unsigned(a.experts) ? v : -1;
  }
  __syncwarp();
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const unsigned same = __match_any_sync(~0u, id[t]);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int old = id[t] >= 0 ? cnt[id[t]] : 0;
    __syncwarp();
    if (before == 0 && id[t] >= 0) cnt[id[t]] = old + __popc(same);
    __syncwarp();
    rank[t] = old + before;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a, int tiles) {
  extern __shared__ int cnt[];  // kSortWarps x experts
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int id[kSortSteps], rank[kSortSteps];
  rank_warp(a, (long long)blockIdx.x * kSortTile + warp * (32 * kSortSteps), lane,
            cnt + warp * a.experts, id, rank);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kSortThreads) {
    int n = 0;
    for (int w = 0; w < kSortWarps; ++w) n += cnt[w * a.experts + e];
    a.tile_counts[(long long)e * tiles + blockIdx.x] = n;
  }
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

// One block an expert: its tiles' counts become running sums, its total goes to counts.
__global__ void __launch_bounds__(256) sort_scan_kernel(const SortArgs a, int tiles) {
  __shared__ int part[8];
  int* c = a.tile_counts + (long long)blockIdx.x * tiles;
  int run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + int(threadIdx.x);
    const int v = t < tiles ? c[t] : 0;
    int all;
    const int upto = block_sum<256>(v, part, &all);
    if (t < tiles) c[t] = run + upto - v;
    run += all;
  }
  if (threadIdx.x == 0) a.counts[blockIdx.x] = run;
}

// ONE: the whole sort of up to one tile.
template <bool ONE>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortArgs a, int tiles) {
  extern __shared__ int cnt[];  // kSortWarps x experts
  __shared__ int part[kSortWarps];
  constexpr int PER = kMaxExperts / kSortThreads;  // experts a thread
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, E = a.experts;
  int id[kSortSteps], rank[kSortSteps];
  const long long first = (long long)blockIdx.x * kSortTile + warp * (32 * kSortSteps);
  rank_warp(a, first, lane, cnt + warp * E, id, rank);
  __syncthreads();
  int n[PER], room = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = int(threadIdx.x) * PER + q;
    n[q] = 0;
    if (e < E) {
      if (ONE)
        for (int w = 0; w < kSortWarps; ++w) n[q] += cnt[w * E + e];
      else
        n[q] = a.counts[e];
    }
    room += (n[q] + a.align - 1) / a.align * a.align;
  }
  int end;
  int start = block_sum<kSortThreads>(room, part, &end) - room;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = int(threadIdx.x) * PER + q;
    if (e < E) {
      const int next = start + (n[q] + a.align - 1) / a.align * a.align;
      if (blockIdx.x == 0) {
        a.offsets[e] = start;
        if (ONE) a.counts[e] = n[q];
        for (int s = start + n[q]; s < next; ++s) a.order[s] = -1;
      }
      int run = start + (ONE ? 0 : a.tile_counts[(long long)e * tiles + blockIdx.x]);
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * E + e];
        cnt[w * E + e] = run;
        run += c;
      }
      start = next;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[E] = end;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kSortSteps; ++t) {
    const long long i = first + t * 32 + lane;
    if (i < a.entries) {
      const int slot = id[t] >= 0 ? cnt[warp * E + id[t]] + rank[t] : -1;
      a.slots[i] = slot;
      if (slot >= 0) a.order[slot] = int(i);
    }
  }
  for (long long s = end + (long long)blockIdx.x * kSortThreads + threadIdx.x; s < a.capacity;
       s += (long long)gridDim.x * kSortThreads)
    a.order[s] = -1;
}

// ---- units of a copy --------------------------------------------------------

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

template <class U>
__device__ __forceinline__ U zero() {
  U u;
  memset(&u, 0, sizeof(U));
  return u;
}

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

constexpr int kThreads = 256;

// Slots first .. first + 31 without an entry: the warp writes zeros to their rows.
template <class U>
__device__ __forceinline__ void zero_empty(const int* order, long long first, long long capacity,
                                           U* out, long long ld, long long units, int lane) {
  const long long s = first + lane;
  unsigned empty = __ballot_sync(~0u, s < capacity && order[s < capacity ? s : 0] < 0);
  while (empty) {
    const int q = __ffs(int(empty)) - 1;
    empty &= empty - 1;
    for (long long u = lane; u < units; u += 32) out[(first + q) * ld + u] = zero<U>();
  }
}

// ---- gather -----------------------------------------------------------------

// Row-major to row-major.  `lanes` lanes a row (a power of two); the blocks from
// `row_blocks` on clear the empty slots.  Units and strides in units.
template <class U>
__global__ void __launch_bounds__(kThreads)
    gather_rows_kernel(const U* x, long long rows, long long units, long long ld, int k,
                       const int* order, const int* slots, long long capacity, U* out,
                       long long ld_out, int lanes, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) {
    const long long warp = (long long)(blockIdx.x - row_blocks) * (kThreads / 32) + threadIdx.x / 32;
    if (warp * 32 < capacity)
      zero_empty(order, warp * 32, capacity, out, ld_out, units, threadIdx.x % 32);
    return;
  }
  const int lane = threadIdx.x % lanes;
  const long long n = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (n >= rows) return;
  const U* row = x + n * ld;
  const int* mine = slots + n * k;
  for (long long u = lane; u < units; u += 4 * lanes) {
    U v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = u + q * lanes < units ? row[u + q * lanes] : zero<U>();
    for (int j = 0; j < k; ++j) {
      const unsigned s = unsigned(mine[j]);
      if (s >= (unsigned long long)capacity) continue;
      U* to = out + s * ld_out;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (u + q * lanes < units) to[u + q * lanes] = v[q];
    }
  }
}

// Forms with a feature-major side: a tile of 64 slots x 128 columns in shared memory.
constexpr int kTileSlots = 64, kTileCols = 128;

template <class T, bool IN_ROW, bool OUT_ROW>
__global__ void __launch_bounds__(kThreads)
    gather_tile_kernel(const T* x, long long entries, long long cols, long long ld, int k,
                       const int* order, long long capacity, T* out, long long ld_out) {
  __shared__ T tile[kTileSlots][kTileCols + (sizeof(T) == 4 ? 1 : 2)];
  __shared__ int from[kTileSlots];
  const long long s0 = (long long)blockIdx.x * kTileSlots;
  const long long c0 = (long long)blockIdx.y * kTileCols;
  const int ns = int(capacity - s0 < kTileSlots ? capacity - s0 : kTileSlots);
  const int nc = int(cols - c0 < kTileCols ? cols - c0 : kTileCols);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x < kTileSlots) {
    const int e = int(threadIdx.x) < ns ? order[s0 + threadIdx.x] : -1;
    from[threadIdx.x] = e >= 0 && e < entries ? e / k : -1;
  }
  __syncthreads();
  if (IN_ROW) {
#pragma unroll
    for (int q = 0; q < kTileSlots / 8; ++q) {
      const int s = warp + q * 8;
      const int n = from[s];
      const T* row = x + (long long)(n < 0 ? 0 : n) * ld + c0;
#pragma unroll
      for (int p = 0; p < kTileCols / 32; ++p) {
        const int c = lane + p * 32;
        if (c < nc) tile[s][c] = n >= 0 ? row[c] : from_float<T>(0.f);
      }
    }
  } else {
    for (int i = threadIdx.x; i < kTileSlots * nc; i += kThreads) {
      const int c = i / kTileSlots, s = i % kTileSlots, n = from[s];
      tile[s][c] = n >= 0 ? x[(c0 + c) * ld + n] : from_float<T>(0.f);
    }
  }
  __syncthreads();
  if (OUT_ROW) {
    for (int s = warp; s < ns; s += 8)
      for (int c = lane; c < nc; c += 32) out[(s0 + s) * ld_out + c0 + c] = tile[s][c];
  } else {
    for (int i = threadIdx.x; i < kTileSlots * nc; i += kThreads) {
      const int c = i / kTileSlots, s = i % kTileSlots;
      if (s < ns) out[(c0 + c) * ld_out + s0 + s] = tile[s][c];
    }
  }
}

// Feature-major to feature-major: a thread a slot, down 8 columns.
constexpr int kColumns = 8;
template <class T>
__global__ void __launch_bounds__(kThreads)
    gather_columns_kernel(const T* x, long long entries, long long cols, long long ld, int k,
                          const int* order, long long capacity, T* out, long long ld_out) {
  const long long s = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (s >= capacity) return;
  const int e = order[s];
  const long long n = e >= 0 && e < entries ? e / k : -1;
  const long long c0 = (long long)blockIdx.y * kColumns;
  T v[kColumns];
#pragma unroll
  for (int q = 0; q < kColumns; ++q)
    v[q] = n >= 0 && c0 + q < cols ? x[(c0 + q) * ld + n] : from_float<T>(0.f);
#pragma unroll
  for (int q = 0; q < kColumns; ++q)
    if (c0 + q < cols) out[(c0 + q) * ld_out + s] = v[q];
}

// ---- combine ----------------------------------------------------------------

template <class T, int BYTES>
struct Values {
  static constexpr int N = BYTES / int(sizeof(T));
  union {
    typename Unit<BYTES>::T u;
    T t[N];
  };
  __device__ Values() {}
};

template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads) combine_kernel(const CombineArgs a, int lanes) {
  using U = typename Unit<BYTES>::T;
  using W = Values<T, BYTES>;
  const int lane = threadIdx.x % lanes;
  const long long n = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (n >= a.rows) return;
  const int units = int(a.cols * (long long)sizeof(T) / BYTES);
  const int* slots = a.slots + n * a.k;
  const float* weights = a.weights ? a.weights + n * a.k : nullptr;
  for (int u = lane; u < units; u += lanes) {
    float acc[W::N] = {};
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
      const unsigned s = unsigned(slots[j]);
      if (s < (unsigned long long)a.capacity) {
        const float w = weights ? weights[j] : 1.f;
        W v;
        v.u = reinterpret_cast<const U*>(static_cast<const T*>(a.y) + s * a.ld)[u];
#pragma unroll
        for (int i = 0; i < W::N; ++i) acc[i] = fmaf(w, to_float(v.t[i]), acc[i]);
      }
    }
    W o;
#pragma unroll
    for (int i = 0; i < W::N; ++i) o.t[i] = from_float<T>(acc[i]);
    reinterpret_cast<U*>(static_cast<T*>(a.out) + n * a.ld_out)[u] = o.u;
  }
}

template <class T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    combine_grad_kernel(const CombineArgs a, int lanes, unsigned row_blocks) {
  using U = typename Unit<BYTES>::T;
  using W = Values<T, BYTES>;
  const int units = int(a.cols * (long long)sizeof(T) / BYTES);
  if (blockIdx.x >= row_blocks) {
    const long long warp = (long long)(blockIdx.x - row_blocks) * (kThreads / 32) + threadIdx.x / 32;
    if (warp * 32 < a.capacity)
      zero_empty(a.order, warp * 32, a.capacity, static_cast<U*>(a.dy),
                 a.ld_dy * (long long)sizeof(T) / BYTES, units, threadIdx.x % 32);
    return;
  }
  const int lane = threadIdx.x % lanes;
  const long long n = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const bool there = n < a.rows;  // whole groups stay for the shuffles
  const long long row = there ? n : 0;
  const U* dout = reinterpret_cast<const U*>(static_cast<const T*>(a.dout) + row * a.ld_dout);
  for (int j = 0; j < a.k; ++j) {
    const unsigned s = there ? unsigned(a.slots[row * a.k + j]) : ~0u;
    const bool ok = s < (unsigned long long)a.capacity;
    float dot = 0.f;
    if (ok) {
      const float w = a.weights ? a.weights[row * a.k + j] : 1.f;
      const U* y = reinterpret_cast<const U*>(static_cast<const T*>(a.y) + s * a.ld);
      U* dy = reinterpret_cast<U*>(static_cast<T*>(a.dy) + s * a.ld_dy);
#pragma unroll 4
      for (int u = lane; u < units; u += lanes) {
        W g, v, o;
        g.u = dout[u];
        v.u = y[u];
#pragma unroll
        for (int i = 0; i < W::N; ++i) {
          const float up = to_float(g.t[i]);
          dot = fmaf(up, to_float(v.t[i]), dot);
          o.t[i] = from_float<T>(w * up);
        }
        dy[u] = o.u;
      }
    }
    for (int o = lanes / 2; o > 0; o /= 2) dot += __shfl_xor_sync(~0u, dot, o);
    if (there && lane == 0 && a.dweights) a.dweights[row * a.k + j] = dot;
  }
}

// The largest unit that divides all of these.
int unit_bytes(uintptr_t all) {
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Lanes a row: the smallest power of two that covers its units, at most a warp.
int lanes_for(long long units) {
  int l = 1;
  while (l < 32 && l < units) l *= 2;
  return l;
}

template <class U>
cudaError_t gather_rows(const GatherArgs& a, cudaStream_t s) {
  const long long size = dtype_bytes(a.dtype), per = (long long)sizeof(U) / size;
  const long long units = a.cols / per;
  const int lanes = lanes_for(units);
  const long long row_blocks = (a.rows + kThreads / lanes - 1) / (kThreads / lanes);
  const long long blocks = row_blocks + (a.capacity + kThreads - 1) / kThreads;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  gather_rows_kernel<U><<<unsigned(blocks), kThreads, 0, s>>>(
      static_cast<const U*>(a.x), a.rows, units, a.ld / per, a.k, a.order, a.slots, a.capacity,
      static_cast<U*>(a.out), a.ld_out / per, lanes, unsigned(row_blocks));
  return cudaGetLastError();
}

template <class T>
cudaError_t gather_tiles(const GatherArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  T* out = static_cast<T*>(a.out);
  const long long entries = a.rows * a.k;
  if (a.layout == 0 && a.layout_out == 0) {
    const long long parts = (a.cols + kColumns - 1) / kColumns;
    if (parts > 65535) return cudaErrorInvalidValue;
    const dim3 grid(unsigned((a.capacity + kThreads - 1) / kThreads), unsigned(parts));
    gather_columns_kernel<T><<<grid, kThreads, 0, s>>>(x, entries, a.cols, a.ld, a.k, a.order,
                                                       a.capacity, out, a.ld_out);
    return cudaGetLastError();
  }
  const long long parts = (a.cols + kTileCols - 1) / kTileCols;
  if (parts > 65535) return cudaErrorInvalidValue;
  const dim3 grid(unsigned((a.capacity + kTileSlots - 1) / kTileSlots), unsigned(parts));
  if (a.layout == 1)
    gather_tile_kernel<T, true, false><<<grid, kThreads, 0, s>>>(
        x, entries, a.cols, a.ld, a.k, a.order, a.capacity, out, a.ld_out);
  else
    gather_tile_kernel<T, false, true><<<grid, kThreads, 0, s>>>(
        x, entries, a.cols, a.ld, a.k, a.order, a.capacity, out, a.ld_out);
  return cudaGetLastError();
}

template <class T, int BYTES>
cudaError_t combine(const CombineArgs& a, bool grad, cudaStream_t s) {
  const int lanes = lanes_for(a.cols * (long long)sizeof(T) / BYTES);
  const long long row_blocks = (a.rows + kThreads / lanes - 1) / (kThreads / lanes);
  const long long blocks = row_blocks + (grad ? (a.capacity + kThreads - 1) / kThreads : 0);
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (grad)
    combine_grad_kernel<T, BYTES><<<unsigned(blocks), kThreads, 0, s>>>(a, lanes, unsigned(row_blocks));
  else
    combine_kernel<T, BYTES><<<unsigned(blocks), kThreads, 0, s>>>(a, lanes);
  return cudaGetLastError();
}

template <class T>
cudaError_t combine_of(const CombineArgs& a, bool grad, cudaStream_t s) {
  const uintptr_t size = sizeof(T);
  uintptr_t all = reinterpret_cast<uintptr_t>(a.y) | uintptr_t(a.ld) * size | uintptr_t(a.cols) * size;
  if (grad)
    all |= reinterpret_cast<uintptr_t>(a.dout) | uintptr_t(a.ld_dout) * size |
           reinterpret_cast<uintptr_t>(a.dy) | uintptr_t(a.ld_dy) * size;
  else
    all |= reinterpret_cast<uintptr_t>(a.out) | uintptr_t(a.ld_out) * size;
  switch (unit_bytes(all)) {
    case 16: return combine<T, 16>(a, grad, s);
    case 8: return combine<T, 8>(a, grad, s);
    case 4: return combine<T, 4>(a, grad, s);
    default: break;
  }
  if constexpr (sizeof(T) == 2) return combine<T, 2>(a, grad, s);
  return cudaErrorInvalidValue;
}

cudaError_t combine_any(const CombineArgs& a, bool grad, cudaStream_t s) {
  return a.dtype == kF32    ? combine_of<float>(a, grad, s)
         : a.dtype == kBF16 ? combine_of<__nv_bfloat16>(a, grad, s)
                            : combine_of<__half>(a, grad, s);
}

int sort_tiles(long long entries) { return int((entries + kSortTile - 1) / kSortTile); }

}  // namespace

long long sort_workspace_ints(long long entries, int experts) {
  const int tiles = sort_tiles(entries);
  return tiles <= 1 ? 0 : (long long)tiles * experts;
}

cudaError_t launch_sort(const SortArgs& a, int* launches, cudaStream_t s) {
  const int tiles = sort_tiles(a.entries);
  const size_t smem = size_t(kSortWarps) * size_t(a.experts) * sizeof(int);  // at most 32 KB
  if (tiles <= 1) {
    sort_place_kernel<true><<<1, kSortThreads, smem, s>>>(a, 1);
    *launches = 1;
    return cudaGetLastError();
  }
  sort_count_kernel<<<tiles, kSortThreads, smem, s>>>(a, tiles);
  sort_scan_kernel<<<a.experts, 256, 0, s>>>(a, tiles);
  sort_place_kernel<false><<<tiles, kSortThreads, smem, s>>>(a, tiles);
  *launches = 3;
  return cudaGetLastError();
}

cudaError_t launch_gather(const GatherArgs& a, cudaStream_t s) {
  const uintptr_t size = uintptr_t(dtype_bytes(a.dtype));
  if (a.layout == 1 && a.layout_out == 1) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out) |
                          uintptr_t(a.ld) * size | uintptr_t(a.ld_out) * size |
                          uintptr_t(a.cols) * size;
    switch (unit_bytes(all)) {
      case 16: return gather_rows<uint4>(a, s);
      case 8: return gather_rows<uint2>(a, s);
      case 4: return gather_rows<unsigned>(a, s);
      default: return gather_rows<unsigned short>(a, s);
    }
  }
  // only moved, never computed with: any two-byte type serves for both
  return size == 4 ? gather_tiles<float>(a, s) : gather_tiles<__half>(a, s);
}

cudaError_t launch_combine(const CombineArgs& a, cudaStream_t s) { return combine_any(a, false, s); }

cudaError_t launch_combine_grad(const CombineArgs& a, cudaStream_t s) {
  return combine_any(a, true, s);
}

}  // namespace mb
