// Kernels of gradient clipping (clip.h).
//
// norm    Blocks take chunks of 32 KB, block b the chunks b, b + blocks, ...: the squares
//         of 16 bytes of values are added up in 32 bits and these sums in 64 (in 64 from the
//         start where 32 would overflow or vanish), so that a norm is right wherever float32
//         holds it.  A block's sum goes to the workspace.
// scale   Every block adds the blocks' sums up in the same order, forms the factor and scales
//         its chunks, the last ones read first: they are still in the L2 cache (what comes
//         before them is read, and what is written stored, so that it leaves first).
// one     Both at once for little: a cluster of eight blocks, whose sums meet in its shared
//         memory.
//
// Both read or write what they have to once; bytes bound them.  170M values of bfloat16 in 300
// tensors (340 MB): the norm 58 us (5.9 TB/s), the scaling 112 (6.1 TB/s with a cold cache), 166
// together; 9.5M values in 1,500 tensors 23 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "clip.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int kThreads = 256;

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

// The sum of the block's values, in every thread; the order is the threads'.
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) all += shared[w];
  return all;
}

// Squares of 16 bytes of values.  Sums of squares between 2^-80 and 2^120 lose nothing to
// float32's range: a square below its smallest normal number, 2^-126, is below 2^-46 of
// the sum.  (Units of zeros go the long way too: the norm of 340 MB of them takes 94 us, of noise 77, both with
// the call.)
template <class T>
__device__ __forceinline__ double squares(uint4 u) {
  constexpr int N = 16 / int(sizeof(T));
  T v[N];
  memcpy(v, &u, 16);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = to_float(v[i]);
    s = fmaf(x, x, s);
  }
  if (s >= 0x1p-80f && s <= 0x1p120f) return double(s);
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double x = to_float(v[i]);
    d = fma(x, x, d);
  }
  return d;
}

// A tensor's chunk: its values from `p` on, split into those before the first 16-byte
// boundary, whole units and the rest.
template <class T>
struct Span {
  int head, units, tail;
  __device__ Span(const T* from, long long left, bool whole) {
    const int n = int(left < kClipChunk / int(sizeof(T)) ? left : kClipChunk / int(sizeof(T)));
    head = whole ? int((16 - reinterpret_cast<uintptr_t>(from) % 16) % 16 / sizeof(T)) : n;
    head = head < n ? head : n;
    units = (n - head) / (16 / int(sizeof(T)));
    tail = n - head - units * (16 / int(sizeof(T)));
  }
};

constexpr int kStep = 4;  // units of a thread on their way

template <class T>
__device__ __forceinline__ double chunk_squares(const T* src, long long left, bool once) {
  const Span<T> c(src, left, true);
  constexpr int N = 16 / int(sizeof(T));
  double sum = 0.0;
  const uint4* q = reinterpret_cast<const uint4*>(src + c.head) + threadIdx.x;
  int n = c.units - int(threadIdx.x);
  for (; n > (kStep - 1) * kThreads; n -= kStep * kThreads, q += kStep * kThreads) {
    uint4 u[kStep];
#pragma unroll
    for (int t = 0; t < kStep; ++t) u[t] = once ? __ldcs(q + t * kThreads) : q[t * kThreads];
#pragma unroll
    for (int t = 0; t < kStep; ++t) sum += squares<T>(u[t]);
  }
  for (; n > 0; n -= kThreads, q += kThreads) sum += squares<T>(*q);
  // what lies in front of and behind the units
  for (int i = threadIdx.x; i < c.head + c.tail; i += kThreads) {
    const double x = to_float(src[i < c.head ? i : i + c.units * N]);
    sum = fma(x, x, sum);
  }
  return sum;
}

// The factor, as a product: one below float32's normal numbers would have few bits left, or none (gradients of
// 1e38 clipped to a norm of 1e-5 came out twice too large).
struct Factor {
  float high, low;  // low: 1, or 2^-100
  __device__ __forceinline__ bool one() const { return high == 1.f && low == 1.f; }
  __device__ __forceinline__ float operator()(float v) const { return v * high * low; }
};

template <class T>
__device__ __forceinline__ uint4 scaled(uint4 u, Factor factor) {
  constexpr int N = 16 / int(sizeof(T));
  T v[N];
  memcpy(v, &u, 16);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = from_float<T>(factor(to_float(v[k])));
  memcpy(&u, v, 16);
  return u;
}

template <class T>
__device__ __forceinline__ void chunk_scale(const T* src, T* dst, long long left, Factor factor) {
  // 16 bytes at a time where both sides reach a boundary together
  const bool whole = (reinterpret_cast<uintptr_t>(src) - reinterpret_cast<uintptr_t>(dst)) % 16 == 0;
  const Span<T> c(src, left, whole);
  constexpr int N = 16 / int(sizeof(T));
  const uint4* q = reinterpret_cast<const uint4*>(src + c.head) + threadIdx.x;
  uint4* to = reinterpret_cast<uint4*>(dst + c.head) + threadIdx.x;
  int n = c.units - int(threadIdx.x);
  for (; n > (kStep - 1) * kThreads; n -= kStep * kThreads, q += kStep * kThreads, to += kStep * kThreads) {
    uint4 u[kStep];
#pragma unroll
    for (int t = 0; t < kStep; ++t) u[t] = q[t * kThreads];
#pragma unroll
    for (int t = 0; t < kStep; ++t) __stcs(to + t * kThreads, scaled<T>(u[t], factor));
  }
  for (; n > 0; n -= kThreads, q += kThreads, to += kThreads) __stcs(to, scaled<T>(*q, factor));
  for (int i = threadIdx.x; i < c.head + c.tail; i += kThreads) {
    const int at = i < c.head ? i : i + c.units * N;
    dst[at] = from_float<T>(factor(to_float(src[at])));
  }
}

// The tensor of a chunk: the last one that does not start behind it.  The chunk is the block's,
// so the search reads one parameter after the other.
template <int N>
__device__ __forceinline__ int tensor_of(const ClipTable<N>& t, unsigned chunk) {
  const unsigned b = chunk >> t.shift;
  int lo = t.bucket[b], hi = t.bucket[b + 1];
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.entry[mid].chunk0 / 4 <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// f(values of the type, the chunk's first value of the gradient and of the output, values from there on)
template <int N, class F>
__device__ __forceinline__ void with_chunk(const ClipTable<N>& t, unsigned chunk, F f) {
  const ClipEntry& e = t.entry[tensor_of(t, chunk)];
  const long long at = (long long)(chunk - e.chunk0 / 4) * kClipChunk;  // bytes
  const char* src = t.src + 2ll * e.src + at;
  char* dst = t.dst + 2ll * e.dst + at;
  const int dtype = e.chunk0 % 4;
  if (dtype == kF32)
    f(reinterpret_cast<const float*>(src), reinterpret_cast<float*>(dst), e.size - at / 4);
  else if (dtype == kBF16)
    f(reinterpret_cast<const __nv_bfloat16*>(src), reinterpret_cast<__nv_bfloat16*>(dst), e.size - at / 2);
  else
    f(reinterpret_cast<const __half*>(src), reinterpret_cast<__half*>(dst), e.size - at / 2);
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
    clip_norm_kernel(const __grid_constant__ ClipTable<N> t, const ClipState c) {
  __shared__ double shared[kThreads / 32];
  double sum = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x)
    with_chunk(t, chunk, [&](const auto* src, auto*, long long left) {
      sum += chunk_squares(src, left, chunk < c.keep);
    });
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) c.part[c.first + blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_of(const ClipState& c, double* shared) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < c.parts; i += kThreads) sum += c.part[i];
  return sqrt(block_sum(sum, shared));
}

__device__ __forceinline__ Factor factor_of(double norm, double max_norm) {
  if (!(norm > max_norm)) return Factor{norm == norm ? 1.f : float(norm), 1.f};
  const double f = max_norm / norm;
  return f < 0x1p-126 && f > 0.0 ? Factor{float(f * 0x1p100), 0x1p-100f} : Factor{float(f), 1.f};
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
    clip_scale_kernel(const __grid_constant__ ClipTable<N> t, const ClipState c) {
  __shared__ double shared[kThreads / 32];
  const double norm = norm_of(c, shared);
  if (c.first == 0 && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = float(norm);
  const Factor factor = factor_of(norm, c.max_norm);
  if (c.in_place && factor.one()) return;
  for (unsigned k = blockIdx.x; k < t.chunks; k += gridDim.x)
    with_chunk(t, t.chunks - 1 - k, [&](const auto* src, auto* dst, long long left) {
      chunk_scale(src, dst, left, factor);
    });
}

// All of it in one launch: a cluster's blocks read each other's sums.
__global__ void __cluster_dims__(kClipCluster, 1, 1) __launch_bounds__(kThreads)
    clip_one_kernel(const __grid_constant__ ClipTable<kClipFew> t, const ClipState c) {
  __shared__ double shared[kThreads / 32];
  __shared__ double mine;
  double sum = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < t.chunks; chunk += kClipCluster)
    with_chunk(t, chunk, [&](const auto* src, auto*, long long left) {
      sum += chunk_squares(src, left, false);
    });
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) mine = sum;
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(&mine));
  sum = 0.0;
#pragma unroll
  for (int b = 0; b < kClipCluster; ++b) {
    double v;
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f64 %0, [a];\n}\n"
        : "=d"(v)
        : "r"(at), "r"(b)
        : "memory");
    sum += v;
  }
  // no block leaves while another may still read its sum
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const double norm = sqrt(sum);
  if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = float(norm);
  const Factor factor = factor_of(norm, c.max_norm);
  if (t.dst && !(c.in_place && factor.one()))
    for (unsigned chunk = blockIdx.x; chunk < t.chunks; chunk += kClipCluster)
      with_chunk(t, chunk, [&](const auto* src, auto* dst, long long left) {
        chunk_scale(src, dst, left, factor);
      });
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(kThreads) clip_finish_kernel(const ClipState c) {
  __shared__ double shared[kThreads / 32];
  const double norm = norm_of(c, shared);
  if (threadIdx.x == 0) *c.norm = float(norm);
}

}  // namespace

template <int N>
cudaError_t launch_clip_norm(const ClipTable<N>& t, const ClipState& c, int blocks, cudaStream_t s) {
  clip_norm_kernel<N><<<blocks, kThreads, 0, s>>>(t, c);
  return cudaGetLastError();
}
template <int N>
cudaError_t launch_clip_scale(const ClipTable<N>& t, const ClipState& c, int blocks, cudaStream_t s) {
  clip_scale_kernel<N><<<blocks, kThreads, 0, s>>>(t, c);
  return cudaGetLastError();
}
template cudaError_t launch_clip_norm<kClipFew>(const ClipTable<kClipFew>&, const ClipState&, int, cudaStream_t);
template cudaError_t launch_clip_norm<kClipTensors>(const ClipTable<kClipTensors>&, const ClipState&, int,
                                                    cudaStream_t);
template cudaError_t launch_clip_scale<kClipFew>(const ClipTable<kClipFew>&, const ClipState&, int, cudaStream_t);
template cudaError_t launch_clip_scale<kClipTensors>(const ClipTable<kClipTensors>&, const ClipState&, int,
                                                     cudaStream_t);

cudaError_t launch_clip_one(const ClipTable<kClipFew>& t, const ClipState& c, cudaStream_t s) {
  clip_one_kernel<<<kClipCluster, kThreads, 0, s>>>(t, c);
  return cudaGetLastError();
}

cudaError_t launch_clip_finish(const ClipState& c, cudaStream_t s) {
  clip_finish_kernel<<<1, kThreads, 0, s>>>(c);
  return cudaGetLastError();
}

}  // namespace mb
