// Rows sorted by model, gathered into each model's segment, and the models'
// outputs combined again, with the gradient (mixture.h).
//
// sort     A stable counting sort.  A tile of entries belongs to a block, an eighth of it,
//          consecutive ones, to a warp; lanes with equal ids find each other with a
//          match and rank themselves by lane, so an entry's place among its
//          warp's equals is known without an atomic and the result is the same
//          every time.  Up to 4,096 entries are one tile and one launch.  More, in
//          tiles of 1,024 or 2,048: counts of each (expert, tile), their running sums
//          per expert, then the places.
// gather   out[slot] = x[row of the entry in slot], zeros in a slot without entry.
//          Row-major to row-major reads every row once and writes it to its k
//          slots; the forms with a feature-major side go through a tile in shared
//          memory, or column by column.
// combine  out[n] = sum_j w[n, j] y[slot[n, j]], summed in 32 bits in the order of j.
// gradient dy[slot[n, j]] = w[n, j] dout[n], dw[n, j] = <dout[n], y[slot[n, j]]>, and
//          zeros in the rows of dy that hold no entry.
//
// Measured: sorting 10M entries among 8 models 59 us (11 counts, 7 sums, 41 places); 8,191 x
// 2,048 bfloat16 rows to eight slots each 52 us (302 MB, 5.8 TB/s), combined 51 us and
// their gradient 92 us (570 MB, 6.2 TB/s); 1M x 10 float32 of two models combined 24 us,
// the gradient 50 us (40-byte rows: latency and partly used sectors).
//
// All of it moves bytes and is bound by them: the unit of a copy is the largest of
// 16, 8, 4 and 2 bytes that the addresses, strides and row lengths share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "mixture.h"

namespace mb {

namespace {

// ---- sort -------------------------------------------------------------------

constexpr int kSortWarps = 8;
constexpr int kSortThreads = kSortWarps * 32;
// Steps of 32 entries a warp: 8 (tiles of 2,048) fill the GPU from some 300,000 entries
// on, with registers for five blocks a multiprocessor (the launches wait for memory and
// for the chain of steps, not for bandwidth); below that 4 give twice the blocks and half
// the chain.
constexpr int kSteps = 8, kFewSteps = 4, kOneSteps = 16;  // kOneSteps: the most of one launch
constexpr long long kFewEntries = 300000;
constexpr int kRunSteps = 16;  // of gather_runs_kernel

// Ranks of a warp's STEPS x 32 entries among its equal ids (-1: none); its counts end up
// in cnt[experts].
template <int STEPS>
__device__ __forceinline__ void rank_warp(int experts, int lane, int* cnt, const int (&id)[STEPS],
                                          int (&rank)[STEPS]) {
  for (int e = lane; e < experts; e += 32) cnt[e] = 0;
  __syncwarp();
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const unsigned same = __match_any_sync(~0u, id[t]);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int old = id[t] >= 0 ? cnt[id[t]] : 0;
    __syncwarp();
    if (before == 0 && id[t] >= 0) cnt[id[t]] = old + __popc(same);
    __syncwarp();
    rank[t] = old + before;
  }
}

// A lane's ids of its warp's STEPS x 32 entries from `first` on.
template <int STEPS>
__device__ __forceinline__ void load_ids(const SortArgs& a, long long first, int lane, int (&id)[STEPS]) {
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    const long long i = first + t * 32 + lane;
    const int v = i < a.entries ? a.ids[i] : -1;
    id[t] = unsigned(v) < unsigned(a.experts) ? v : -1;
  }
}

template <int STEPS>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a, int tiles) {
  extern __shared__ int cnt[];  // experts
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int id[STEPS];
  load_ids(a, ((long long)blockIdx.x * kSortWarps + warp) * (32 * STEPS), lane, id);
  for (int e = threadIdx.x; e < a.experts; e += kSortThreads) cnt[e] = 0;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STEPS; ++t)
    if (id[t] >= 0) atomicAdd(cnt + id[t], 1);  // whole numbers: in any order
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kSortThreads)
    a.tile_counts[(long long)e * tiles + blockIdx.x] = cnt[e];
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
  constexpr int PER = 8;  // adjacent values a thread
  __shared__ int part[8];
  int* c = a.tile_counts + (long long)blockIdx.x * tiles;
  int run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256 * PER) {
    const int t = t0 + int(threadIdx.x) * PER;
    int v[PER], sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      v[q] = t + q < tiles ? c[t + q] : 0;
      sum += v[q];
    }
    int all;
    int before = run + block_sum<256>(sum, part, &all) - sum;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (t + q < tiles) c[t + q] = before;
      before += v[q];
    }
    run += all;
  }
  if (threadIdx.x == 0) a.counts[blockIdx.x] = run;
}

// ONE: the whole sort of up to one tile.
template <bool ONE, int STEPS>
__global__ void __launch_bounds__(kSortThreads, ONE ? 1 : 5) sort_place_kernel(const SortArgs a, int tiles) {
  extern __shared__ int cnt[];  // kSortWarps x experts
  __shared__ int part[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, E = a.experts;
  int id[STEPS], rank[STEPS];
  const long long first = ((long long)blockIdx.x * kSortWarps + warp) * (32 * STEPS);
  load_ids(a, first, lane, id);
  rank_warp(E, lane, cnt + warp * E, id, rank);
  __syncthreads();
  int end = 0;
  for (int e0 = 0; e0 < E; e0 += kSortThreads) {
    const int e = e0 + int(threadIdx.x);
    int n = 0, before = 0;
    if (e < E) {
      if (ONE) {
        for (int w = 0; w < kSortWarps; ++w) n += cnt[w * E + e];
      } else {
        n = a.counts[e];
        before = a.tile_counts[(long long)e * tiles + blockIdx.x];
      }
    }
    const int room = (n + a.align - 1) / a.align * a.align;
    int all;
    const int start = end + block_sum<kSortThreads>(room, part, &all) - room;
    end += all;
    if (e < E) {
      if (blockIdx.x == 0) {
        a.offsets[e] = start;
        if (ONE) a.counts[e] = n;
        for (int s = start + n; s < start + room; ++s) a.order[s] = -1;
      }
      int run = start + before;
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * E + e];
        cnt[w * E + e] = run;
        run += c;
      }
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[E] = end;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
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

// Slots without an entry get rows of zeros.  They lie together, behind the last segment
// above all, so a warp looks at few slots when rows are wide: about 2,048 units, at most
// 256 slots.
__host__ __device__ inline int clear_slots(long long units) {
  const long long n = 2048 / units;
  return n < 1 ? 1 : n > 256 ? 256 : int(n);
}
template <class U>
__device__ __forceinline__ void zero_empty(const int* order, long long warp, long long capacity,
                                           U* out, long long ld, long long units, int lane) {
  const int slots = clear_slots(units);
  const long long first = warp * slots;
  if (units <= 32) {  // a lane a slot
    for (int t = lane; t < slots; t += 32)
      if (first + t < capacity && order[first + t] < 0)
        for (long long u = 0; u < units; ++u) out[(first + t) * ld + u] = zero<U>();
    return;
  }
  for (int t = 0; t < slots; t += 32) {
    const long long s = first + t + lane;
    unsigned empty = __ballot_sync(~0u, t + lane < slots && s < capacity && order[s] < 0);
    while (empty) {
      const int q = __ffs(int(empty)) - 1;
      empty &= empty - 1;
      for (long long u = lane; u < units; u += 32) out[(first + t + q) * ld + u] = zero<U>();
    }
  }
}
// Blocks of 8 warps that clear `capacity` slots.
long long clear_blocks(long long capacity, long long units) {
  const long long per = 8ll * clear_slots(units);
  return (capacity + per - 1) / per;
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
    zero_empty(order, warp, capacity, out, ld_out, units, threadIdx.x % 32);
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

// Row-major to feature-major with rows of whole 16-byte units: 64 slots x `quads` units
// a tile, fetched by asynchronous copies (a warp a row) that need no registers, so that
// several tiles a multiprocessor are in flight; then a lane a slot takes 16 bytes and
// writes its values to their columns, 64 consecutive slots each.  Rows of the tile are an
// odd number of units apart, which makes the 16-byte reads of 8 slots free of bank
// conflicts.  Rows with k choices are read k times.  Walking the segments side by side, to
// find the second reading in the L2 cache, cost more than it saved (500,000 x 100 rows to
// two of 64: 131 us here; 250 with a block walking a window of all segments, 166 with
// blocks in the order of their tiles' place in the segments): the writes then go to 64
// places at once.
constexpr int kUnitSlots = 64, kMaxQuads = 32;
template <class T>
__global__ void __launch_bounds__(kThreads)
    gather_units_kernel(const T* x, long long entries, int units, long long ld, int k,
                        const int* order, long long capacity, T* out, long long ld_out, int quads) {
  constexpr int PER = 16 / int(sizeof(T));
  extern __shared__ uint4 tile[];  // kUnitSlots rows of `pitch`
  const long long s0 = (long long)blockIdx.x * kUnitSlots;
  const int q0 = int(blockIdx.y) * quads;
  const int nq = min(quads, units - q0), pitch = nq | 1;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  // a warp fetches 8 adjacent slots' rows
  const long long mine = s0 + warp * 8 + lane % 8;
  const int e = mine < capacity ? order[mine] : -1;
  const int n = e >= 0 && e < entries ? e / k : -1;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int row = __shfl_sync(~0u, n, q);
    uint4* to = tile + (warp * 8 + q) * pitch + lane;
    if (lane < nq) {
      if (row >= 0) {
        const T* from = x + row * ld + (long long)(q0 + lane) * PER;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         static_cast<unsigned>(__cvta_generic_to_shared(to))),
                     "l"(from)
                     : "memory");
      } else {
        *to = make_uint4(0, 0, 0, 0);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  for (int i = warp; i < 2 * nq; i += kThreads / 32) {
    const int s = (i & 1) * 32 + lane, q = i >> 1;
    if (s0 + s >= capacity) continue;
    union {
      uint4 u;
      T t[PER];
    } v;
    v.u = tile[s * pitch + q];
    T* to = out + (long long)(q0 + q) * PER * ld_out + s0 + s;
#pragma unroll
    for (int p = 0; p < PER; ++p) to[p * ld_out] = v.t[p];
  }
}

// Feature-major to feature-major, few rows: a thread a slot, down 8 columns.
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

constexpr long long kRunEntries = 65536;

// Feature-major to feature-major, many rows: a block takes 4,096 / k adjacent rows,
// groups their entries by model once -- as the sort does, the model of a slot found by
// bisection of the offsets -- and keeps the list (16 entries a thread) for `per` columns:
// each column's values come in with adjacent loads, and leave in runs of adjacent slots.
// A thread a slot would read a 32-byte sector of x for each 4-byte value (10M x 28 among
// 8: 1,392 us, here 457, 77% of copy speed; tiles of 2,048 took 555 and of 8,192, with
// twice the threads, 510).  Blocks from `tiles` on clear the empty slots.
template <class T>
__global__ void __launch_bounds__(kSortThreads, 3)
    gather_runs_kernel(const GatherArgs a, int tile_rows, long long tiles, long long per) {
  constexpr int N = kSortThreads * kRunSteps;  // entries
  extern __shared__ int shared[];
  const T* x = static_cast<const T*>(a.x);
  T* out = static_cast<T*>(a.out);
  const long long c0 = (long long)blockIdx.y * per;
  const long long c1 = c0 + per < a.cols ? c0 + per : a.cols;
  if (blockIdx.x >= tiles) {
    const long long s = (blockIdx.x - tiles) * kSortThreads + threadIdx.x;
    if (s < a.capacity && a.order[s] < 0)
      for (long long c = c0; c < c1; ++c) out[c * a.ld_out + s] = from_float<T>(0.f);
    return;
  }
  const int E = a.experts;
  // the list, later two columns of the tile; then the counts; then the offsets
  int* list_slot = shared;
  unsigned short* list_row = reinterpret_cast<unsigned short*>(shared + N);
  T* column = reinterpret_cast<T*>(shared);
  int* cnt = shared + 2 * N;
  int* offs = cnt + kSortWarps * E;
  __shared__ int part[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long row0 = (long long)blockIdx.x * tile_rows;
  const int nr = int(a.rows - row0 < tile_rows ? a.rows - row0 : tile_rows);
  const int ne = nr * a.k;
  for (int e = threadIdx.x; e < E; e += kSortThreads) offs[e] = int(a.offsets[e]);
  __syncthreads();
  int id[kRunSteps], rank[kRunSteps], slot[kRunSteps];
#pragma unroll
  for (int t = 0; t < kRunSteps; ++t) {
    const int i = warp * (32 * kRunSteps) + t * 32 + lane;
    slot[t] = i < ne ? a.slots[row0 * a.k + i] : -1;
    if (slot[t] >= a.capacity) slot[t] = -1;
    int low = 0, n = E;  // the last expert that starts at or before the slot
    while (n > 1) {
      const int half = n / 2;
      if (offs[low + half] <= slot[t]) low += half;
      n -= half;
    }
    id[t] = slot[t] >= 0 ? low : -1;
  }
  rank_warp(E, lane, cnt + warp * E, id, rank);
  __syncthreads();
  constexpr int PER = kMaxExperts / kSortThreads;
  int n = 0, all;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = int(threadIdx.x) * PER + q;
    if (e < E)
      for (int w = 0; w < kSortWarps; ++w) n += cnt[w * E + e];
  }
  int run = block_sum<kSortThreads>(n, part, &all) - n;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = int(threadIdx.x) * PER + q;
    if (e < E)
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * E + e];
        cnt[w * E + e] = run;
        run += c;
      }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kRunSteps; ++t)
    if (id[t] >= 0) {
      const int at = cnt[warp * E + id[t]] + rank[t];
      list_slot[at] = slot[t];
      list_row[at] = static_cast<unsigned short>((warp * (32 * kRunSteps) + t * 32 + lane) / a.k);
    }
  __syncthreads();
  int row[kRunSteps];
#pragma unroll
  for (int t = 0; t < kRunSteps; ++t) {
    const int i = t * kSortThreads + int(threadIdx.x);
    slot[t] = i < all ? list_slot[i] : -1;
    row[t] = i < all ? list_row[i] : 0;
  }
  T v[kRunSteps];
  auto fetch = [&](long long c) {
#pragma unroll
    for (int t = 0; t < kRunSteps; ++t) {
      const int i = t * kSortThreads + int(threadIdx.x);
      if (i < nr) v[t] = x[c * a.ld + row0 + i];
    }
  };
  fetch(c0);
  __syncthreads();  // the list has been read
  for (long long c = c0; c < c1; ++c) {
    T* buf = column + ((c - c0) & 1) * N;
#pragma unroll
    for (int t = 0; t < kRunSteps; ++t) {
      const int i = t * kSortThreads + int(threadIdx.x);
      if (i < nr) buf[i] = v[t];
    }
    if (c + 1 < c1) fetch(c + 1);
    __syncthreads();
    T* to = out + c * a.ld_out;
#pragma unroll
    for (int t = 0; t < kRunSteps; ++t)
      if (slot[t] >= 0) to[slot[t]] = buf[row[t]];
  }
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

// How a warp or a block is laid over rows of `units` units.  Up to 32 units: a warp has
// 32 / units rows (no division: (lane * inv) >> 16 is lane / units for lane < 32).  More:
// `warps` warps (1, 2, 4 or 8) have a row.  Strides in bytes, below 2^32, so that the
// address of a row is one multiply-add.
struct Lay {
  int units, rows, inv, warps;
  unsigned ld_y, ld_out, ld_dout, ld_dy, capacity;
};

// Rows n[f] of this thread (-1: none), its first unit and the step to the next.
template <int FLIGHT>
__device__ __forceinline__ void lay_rows(const Lay& l, long long rows, long long (&n)[FLIGHT], int* u0,
                                         int* step) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (l.units <= 32) {
    const int r = (lane * l.inv) >> 16;
    *u0 = lane - r * l.units;
    *step = 32;  // once
    const long long first = ((long long)blockIdx.x * (kThreads / 32) + warp) * l.rows * FLIGHT + r;
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      n[f] = first + f * l.rows;
      if (r >= l.rows || n[f] >= rows) n[f] = -1;
    }
  } else {
    *u0 = (warp % l.warps) * 32 + lane;
    *step = l.warps * 32;
    const int per = kThreads / 32 / l.warps;
    const long long first = ((long long)blockIdx.x * per + warp / l.warps) * FLIGHT;
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) n[f] = first + f < rows ? first + f : -1;
  }
}

// J choices of row n from j0 on: their slots (~0: none) and weights (0: none).  K > 0:
// all of the row's, with the widest loads.
template <int K, int J>
__device__ __forceinline__ void load_choices(const CombineArgs& a, const Lay& l, long long n, int j0,
                                             unsigned (&s)[J], float (&w)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    s[j] = ~0u;
    w[j] = 1.f;
  }
  if (n >= 0) {
    const int* ps = a.slots + n * (K ? K : a.k) + j0;
    const float* pw = a.weights ? a.weights + n * (K ? K : a.k) + j0 : nullptr;
    if constexpr (K >= 4) {
#pragma unroll
      for (int j = 0; j < J; j += 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(ps + j);
        s[j] = q.x, s[j + 1] = q.y, s[j + 2] = q.z, s[j + 3] = q.w;
        if (pw) {
          const float4 x = *reinterpret_cast<const float4*>(pw + j);
          w[j] = x.x, w[j + 1] = x.y, w[j + 2] = x.z, w[j + 3] = x.w;
        }
      }
    } else if constexpr (K == 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(ps);
      s[0] = q.x, s[1] = q.y;
      if (pw) {
        const float2 x = *reinterpret_cast<const float2*>(pw);
        w[0] = x.x, w[1] = x.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (K || j0 + j < a.k) {
          s[j] = unsigned(ps[j]);
          if (pw) w[j] = pw[j];
        }
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (s[j] >= l.capacity) {
      s[j] = ~0u;
      w[j] = 0.f;
    }
}

// K choices a row, or any number (K = 0).  FLIGHT groups of rows a warp at once.  Narrow
// rows wait for memory: 1M x 10 of two models took 89 us, with the gradient, at 4 blocks a
// multiprocessor and 82 at 8 and 6 (the gradient); four groups a warp, 96.
template <class T, int BYTES, int K>
__global__ void __launch_bounds__(kThreads, K == 1 || K == 2 ? 8 : 4)
    combine_kernel(const CombineArgs a, const Lay l) {
  using U = typename Unit<BYTES>::T;
  using W = Values<T, BYTES>;
  constexpr int FLIGHT = K == 1 ? 4 : K == 2 ? 2 : 1;
  constexpr int J = K ? K : 4;          // loads a thread has in flight for a row
  long long n[FLIGHT];
  int u0, step;
  lay_rows(l, a.rows, n, &u0, &step);
  for (int u = u0; u < l.units; u += step) {
    const char* y = static_cast<const char*>(a.y) + u * BYTES;
    char* out = static_cast<char*>(a.out) + u * BYTES;
    float acc[FLIGHT][W::N] = {};
    for (int j0 = 0; j0 < (K ? K : a.k); j0 += J) {
      W v[FLIGHT][J];
      unsigned s[FLIGHT][J];
      float w[FLIGHT][J];
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) load_choices<K, J>(a, l, n[f], j0, s[f], w[f]);
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
        for (int j = 0; j < J; ++j)
          v[f][j].u = s[f][j] != ~0u
                          ? *reinterpret_cast<const U*>(y + (unsigned long long)s[f][j] * l.ld_y)
                          : zero<U>();
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < W::N; ++i)
            acc[f][i] = fmaf(w[f][j], to_float(v[f][j].t[i]), acc[f][i]);
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f)
      if (n[f] >= 0) {
        W o;
#pragma unroll
        for (int i = 0; i < W::N; ++i) o.t[i] = from_float<T>(acc[f][i]);
        *reinterpret_cast<U*>(out + n[f] * l.ld_out) = o.u;
      }
  }
}

template <class T, int BYTES, int K>
__global__ void __launch_bounds__(kThreads, K == 8 ? 2 : 6)
    combine_grad_kernel(const CombineArgs a, const Lay l, unsigned row_blocks) {
  using U = typename Unit<BYTES>::T;
  using W = Values<T, BYTES>;
  constexpr int FLIGHT = K == 1 ? 4 : K == 2 ? 2 : 1;
  constexpr int J = K ? K : 4;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int k = K ? K : a.k;
  __shared__ float dots[kThreads / 32][J];
  if (blockIdx.x >= row_blocks) {
    const long long w = (long long)(blockIdx.x - row_blocks) * (kThreads / 32) + warp;
    zero_empty(a.order, w, a.capacity, static_cast<U*>(a.dy), l.ld_dy / BYTES, l.units, lane);
    return;
  }
  const bool narrow = l.units <= 32;
  long long n[FLIGHT];
  int u0, step;
  lay_rows(l, a.rows, n, &u0, &step);
  for (int j0 = 0; j0 < k; j0 += J) {
    unsigned s[FLIGHT][J];
    float w[FLIGHT][J], dot[FLIGHT][J] = {};
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) load_choices<K, J>(a, l, n[f], j0, s[f], w[f]);
    for (int u = u0; u < l.units; u += step) {
      const char* y = static_cast<const char*>(a.y) + u * BYTES;
      const char* dout = static_cast<const char*>(a.dout) + u * BYTES;
      char* dy = static_cast<char*>(a.dy) + u * BYTES;
      W g[FLIGHT], v[FLIGHT][J];
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        g[f].u = n[f] >= 0 ? *reinterpret_cast<const U*>(dout + n[f] * l.ld_dout) : zero<U>();
#pragma unroll
        for (int j = 0; j < J; ++j)
          v[f][j].u = s[f][j] != ~0u
                          ? *reinterpret_cast<const U*>(y + (unsigned long long)s[f][j] * l.ld_y)
                          : zero<U>();
      }
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (s[f][j] != ~0u) {
            W o;
#pragma unroll
            for (int i = 0; i < W::N; ++i) {
              const float up = to_float(g[f].t[i]);
              dot[f][j] = fmaf(up, to_float(v[f][j].t[i]), dot[f][j]);
              o.t[i] = from_float<T>(w[f][j] * up);
            }
            *reinterpret_cast<U*>(dy + (unsigned long long)s[f][j] * l.ld_dy) = o.u;
          }
    }
    if (!a.dweights) continue;
    if (narrow) {
      // sums over a row's adjacent lanes, halves first
      for (int o = 16; o > 0; o /= 2) {
        if (o >= l.units) continue;
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const float other = __shfl_down_sync(~0u, dot[f][j], o);
            if (u0 < o && u0 + o < l.units) dot[f][j] += other;
          }
      }
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (u0 == 0 && n[f] >= 0 && (K || j0 + j < k)) a.dweights[n[f] * k + j0 + j] = dot[f][j];
    } else {
      // J sums over a warp: each step hands half of the sums that are left to the other
      // half of the lanes, so it takes J - 1 + 5 - log2 J shuffles, and lane (32 / J) j
      // ends with sum j
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        int o = 16;
#pragma unroll
        for (int m = J / 2; m > 0; m /= 2) {
          const bool high = lane & o;
#pragma unroll
          for (int i = 0; i < m; ++i) {
            const float give = high ? dot[f][i] : dot[f][i + m];
            const float keep = high ? dot[f][i + m] : dot[f][i];
            dot[f][i] = keep + __shfl_xor_sync(~0u, give, o);
          }
          o /= 2;
        }
        float sum = dot[f][0];
        for (; o > 0; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        const int j = lane / (32 / J);
        const bool leader = lane % (32 / J) == 0;
        if (l.warps > 1) {
          __syncthreads();
          if (leader) dots[warp][j] = sum;
          __syncthreads();
          if (leader && warp % l.warps == 0) {
            sum = 0.f;
            for (int q = 0; q < l.warps; ++q) sum += dots[warp + q][j];
          }
        }
        if (leader && warp % l.warps == 0 && n[f] >= 0 && (K || j0 + j < k))
          a.dweights[n[f] * k + j0 + j] = sum;
      }
    }
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
  const long long blocks = row_blocks + clear_blocks(a.capacity, units);
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
    if (entries >= kRunEntries) {
      const int tile_rows = kSortThreads * kRunSteps / a.k;
      const long long tiles = (a.rows + tile_rows - 1) / tile_rows;
      const long long clear = (a.capacity + kSortThreads - 1) / kSortThreads;
      // few tiles: fewer columns each, so that there are blocks for the whole GPU
      const long long want = (4 * device_sms() + tiles - 1) / tiles;
      const long long parts = std::min<long long>(std::min<long long>(want, a.cols), 65535);
      const long long per = (a.cols + parts - 1) / parts;
      const dim3 grid(unsigned(tiles + clear), unsigned((a.cols + per - 1) / per));
      const size_t smem = (2 * kSortThreads * kRunSteps + size_t(kSortWarps + 1) * a.experts) * sizeof(int);
      // the limit of the largest call, not this one's: it is the kernel's, and another
      // thread may launch between this thread's two calls
      constexpr int most = (2 * kSortThreads * kRunSteps + (kSortWarps + 1) * kMaxExperts) * int(sizeof(int));
      const cudaError_t e = cudaFuncSetAttribute(gather_runs_kernel<T>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e != cudaSuccess) return e;
      gather_runs_kernel<T><<<grid, kSortThreads, smem, s>>>(a, tile_rows, tiles, per);
      return cudaGetLastError();
    }
    const long long parts = (a.cols + kColumns - 1) / kColumns;
    if (parts > 65535) return cudaErrorInvalidValue;
    const dim3 grid(unsigned((a.capacity + kThreads - 1) / kThreads), unsigned(parts));
    gather_columns_kernel<T><<<grid, kThreads, 0, s>>>(x, entries, a.cols, a.ld, a.k, a.order,
                                                       a.capacity, out, a.ld_out);
    return cudaGetLastError();
  }
  constexpr long long PER = 16 / (long long)sizeof(T);
  if (a.layout == 1 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ld % PER == 0 &&
      a.cols % PER == 0) {
    const long long units = a.cols / PER;
    const long long tiles = (a.capacity + kUnitSlots - 1) / kUnitSlots;
    // few tiles: fewer units each; else tiles of about equal width
    long long quads = std::max<long long>(4, units * tiles / (4 * device_sms()));
    quads = std::min<long long>(quads, std::min<long long>(units, kMaxQuads));
    const long long parts = (units + quads - 1) / quads;
    quads = (units + parts - 1) / parts;
    if (parts > 65535) return cudaErrorInvalidValue;
    const size_t smem = size_t(kUnitSlots) * size_t(quads | 1) * 16;  // at most 33 KB
    gather_units_kernel<T><<<dim3(unsigned(tiles), unsigned(parts)), kThreads, smem, s>>>(
        x, entries, int(units), a.ld, a.k, a.order, a.capacity, out, a.ld_out, int(quads));
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

template <class T, int BYTES, int K>
cudaError_t combine_k(const CombineArgs& a, bool grad, cudaStream_t s) {
  constexpr int FLIGHT = K == 1 ? 4 : K == 2 ? 2 : 1;
  constexpr unsigned size = sizeof(T);
  Lay l{};
  l.units = int(a.cols * (long long)sizeof(T) / BYTES);
  l.ld_y = unsigned(a.ld) * size;
  l.ld_out = unsigned(a.ld_out) * size;
  l.ld_dout = unsigned(a.ld_dout) * size;
  l.ld_dy = unsigned(a.ld_dy) * size;
  l.capacity = unsigned(a.capacity);
  long long per;                        // rows a block
  if (l.units <= 32) {
    l.rows = 32 / l.units;
    l.inv = (65536 + l.units - 1) / l.units;
    per = (long long)(kThreads / 32) * l.rows * FLIGHT;
  } else {
    // as many warps a row as have two units a lane; the gradient, whose sums then meet in
    // shared memory, takes more than one only until there are 16 warps a multiprocessor
    const long long enough = 16ll * device_sms();
    l.warps = 1;
    while (l.warps < 8 && 64 * l.warps <= l.units && (!grad || a.rows * l.warps < enough)) l.warps *= 2;
    per = kThreads / 32 / l.warps * FLIGHT;
  }
  const long long row_blocks = (a.rows + per - 1) / per;
  const long long blocks = row_blocks + (grad ? clear_blocks(a.capacity, l.units) : 0);
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (grad)
    combine_grad_kernel<T, BYTES, K><<<unsigned(blocks), kThreads, 0, s>>>(a, l, unsigned(row_blocks));
  else
    combine_kernel<T, BYTES, K><<<unsigned(blocks), kThreads, 0, s>>>(a, l);
  return cudaGetLastError();
}

template <class T, int BYTES>
cudaError_t combine(const CombineArgs& a, bool grad, cudaStream_t s) {
  // a row's slots and weights by one or two loads, where they start on such a boundary
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.weights);
  if (a.k == 1) return combine_k<T, BYTES, 1>(a, grad, s);
  if (a.k == 2 && at % 8 == 0) return combine_k<T, BYTES, 2>(a, grad, s);
  if (a.k == 4 && at % 16 == 0) return combine_k<T, BYTES, 4>(a, grad, s);
  if (a.k == 8 && at % 16 == 0) return combine_k<T, BYTES, 8>(a, grad, s);
  return combine_k<T, BYTES, 0>(a, grad, s);
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

int sort_steps(long long entries) {
  // up to one tile: one launch, with the fewer steps when they do
  return entries <= kSortThreads * kFewSteps   ? kFewSteps
         : entries <= kSortThreads * kSteps    ? kSteps
         : entries <= kSortThreads * kOneSteps ? kOneSteps
         : entries <= kFewEntries              ? kFewSteps
                                               : kSteps;
}
int sort_tiles(long long entries) {
  const long long tile = kSortThreads * sort_steps(entries);
  return int((entries + tile - 1) / tile);
}

template <int STEPS>
cudaError_t sort(const SortArgs& a, int tiles, int* launches, cudaStream_t s) {
  const size_t smem = size_t(kSortWarps) * size_t(a.experts) * sizeof(int);  // at most 32 KB
  if (tiles <= 1) {
    sort_place_kernel<true, STEPS><<<1, kSortThreads, smem, s>>>(a, 1);
    *launches = 1;
    return cudaGetLastError();
  }
  sort_count_kernel<STEPS><<<tiles, kSortThreads, smem / kSortWarps, s>>>(a, tiles);
  sort_scan_kernel<<<a.experts, 256, 0, s>>>(a, tiles);
  sort_place_kernel<false, STEPS><<<tiles, kSortThreads, smem, s>>>(a, tiles);
  *launches = 3;
  return cudaGetLastError();
}

}  // namespace

long long sort_workspace_ints(long long entries, int experts) {
  const int tiles = sort_tiles(entries);
  return tiles <= 1 ? 0 : (long long)tiles * experts;
}

cudaError_t launch_sort(const SortArgs& a, int* launches, cudaStream_t s) {
  const int tiles = sort_tiles(a.entries);
  switch (sort_steps(a.entries)) {
    case kFewSteps: return sort<kFewSteps>(a, tiles, launches, s);
    case kSteps: return sort<kSteps>(a, tiles, launches, s);
    default: break;
  }
  // up to kOneSteps steps a warp, always one tile
  sort_place_kernel<true, kOneSteps><<<1, kSortThreads, size_t(kSortWarps) * a.experts * sizeof(int), s>>>(a, 1);
  *launches = 1;
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
