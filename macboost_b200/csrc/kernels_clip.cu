// Kernels of gradient clipping (clip.h).
//
// norm    Blocks take chunks of 32 KB, block b the chunks b, b + blocks, ...: the squares
//         of 16 bytes of values are added up in 32 bits and these sums in 64 (in 64 from the
//         start where 32 would overflow or vanish), so that a norm is right wherever float32
//         holds it.  A block's sum goes to the workspace.
// scale   Every block adds the blocks' sums up in the same order, forms the factor and scales
//         its chunks, the last ones read first: they are still in the L2 cache.
//
// Both read or write what they have to once; bytes bound them.
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
// the sum.
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
  const T* p;
  int head, units, tail;
  __device__ Span(const T* from, long long left, bool whole) : p(from) {
    const int n = int(left < kClipChunk / int(sizeof(T)) ? left : kClipChunk / int(sizeof(T)));
    head = whole ? int((16 - reinterpret_cast<uintptr_t>(from) % 16) % 16 / sizeof(T)) : n;
    head = head < n ? head : n;
    units = (n - head) / (16 / int(sizeof(T)));
    tail = n - head - units * (16 / int(sizeof(T)));
  }
};

template <class T>
__device__ __forceinline__ double chunk_squares(const T* src, long long left) {
  const Span<T> c(src, left, true);
  double sum = 0.0;
  constexpr int STEP = 4;
  const uint4* q = reinterpret_cast<const uint4*>(c.p + c.head);
  for (int i = threadIdx.x; i < c.units; i += STEP * kThreads) {
    uint4 u[STEP];
#pragma unroll
    for (int t = 0; t < STEP; ++t)
      u[t] = i + t * kThreads < c.units ? q[i + t * kThreads] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < STEP; ++t) sum += squares<T>(u[t]);
  }
  for (int i = threadIdx.x; i < c.head; i += kThreads) {
    const double x = to_float(c.p[i]);
    sum = fma(x, x, sum);
  }
  const T* end = c.p + c.head + c.units * (16 / int(sizeof(T)));
  for (int i = threadIdx.x; i < c.tail; i += kThreads) {
    const double x = to_float(end[i]);
    sum = fma(x, x, sum);
  }
  return sum;
}

template <class T>
__device__ __forceinline__ void chunk_scale(const T* src, T* dst, long long left, float factor) {
  // 16 bytes at a time where both sides reach a boundary together
  const bool whole = (reinterpret_cast<uintptr_t>(src) - reinterpret_cast<uintptr_t>(dst)) % 16 == 0;
  const Span<T> c(src, left, whole);
  constexpr int STEP = 4, N = 16 / int(sizeof(T));
  const uint4* q = reinterpret_cast<const uint4*>(c.p + c.head);
  uint4* to = reinterpret_cast<uint4*>(dst + c.head);
  for (int i = threadIdx.x; i < c.units; i += STEP * kThreads) {
    uint4 u[STEP];
#pragma unroll
    for (int t = 0; t < STEP; ++t)
      if (i + t * kThreads < c.units) u[t] = q[i + t * kThreads];
#pragma unroll
    for (int t = 0; t < STEP; ++t) {
      T v[N];
      memcpy(v, &u[t], 16);
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = from_float<T>(to_float(v[k]) * factor);
      memcpy(&u[t], v, 16);
      if (i + t * kThreads < c.units) to[i + t * kThreads] = u[t];
    }
  }
  for (int i = threadIdx.x; i < c.head; i += kThreads) dst[i] = from_float<T>(to_float(c.p[i]) * factor);
  const int end = c.head + c.units * N;
  for (int i = threadIdx.x; i < c.tail; i += kThreads)
    dst[end + i] = from_float<T>(to_float(c.p[end + i]) * factor);
}

// The tensor of a chunk: the last one that does not start behind it.
template <int N>
__device__ __forceinline__ int tensor_of(const ClipTable<N>& t, unsigned chunk) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.chunk0[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
    clip_norm_kernel(const __grid_constant__ ClipTable<N> t, const ClipState c) {
  __shared__ double shared[kThreads / 32];
  double sum = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int i = tensor_of(t, chunk);
    const long long at = (long long)(chunk - t.chunk0[i]) * kClipChunk;  // bytes
    const char* src = static_cast<const char*>(t.src[i]) + at;
    if (t.dtype[i] == kF32)
      sum += chunk_squares(reinterpret_cast<const float*>(src), t.size[i] - at / 4);
    else if (t.dtype[i] == kBF16)
      sum += chunk_squares(reinterpret_cast<const __nv_bfloat16*>(src), t.size[i] - at / 2);
    else
      sum += chunk_squares(reinterpret_cast<const __half*>(src), t.size[i] - at / 2);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) c.part[c.first + blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_of(const ClipState& c, double* shared) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < c.parts; i += kThreads) sum += c.part[i];
  return sqrt(block_sum(sum, shared));
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
    clip_scale_kernel(const __grid_constant__ ClipTable<N> t, const ClipState c) {
  __shared__ double shared[kThreads / 32];
  const double norm = norm_of(c, shared);
  if (c.first == 0 && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = float(norm);
  const float factor = norm > c.max_norm ? float(c.max_norm / norm) : norm == norm ? 1.f : float(norm);
  if (c.in_place && factor == 1.f) return;
  for (unsigned k = blockIdx.x; k < t.chunks; k += gridDim.x) {
    const unsigned chunk = t.chunks - 1 - k;
    const int i = tensor_of(t, chunk);
    const long long at = (long long)(chunk - t.chunk0[i]) * kClipChunk;
    const char* src = static_cast<const char*>(t.src[i]) + at;
    char* dst = static_cast<char*>(t.dst[i]) + at;
    if (t.dtype[i] == kF32)
      chunk_scale(reinterpret_cast<const float*>(src), reinterpret_cast<float*>(dst), t.size[i] - at / 4,
                  factor);
    else if (t.dtype[i] == kBF16)
      chunk_scale(reinterpret_cast<const __nv_bfloat16*>(src), reinterpret_cast<__nv_bfloat16*>(dst),
                  t.size[i] - at / 2, factor);
    else
      chunk_scale(reinterpret_cast<const __half*>(src), reinterpret_cast<__half*>(dst), t.size[i] - at / 2,
                  factor);
  }
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

cudaError_t launch_clip_finish(const ClipState& c, cudaStream_t s) {
  clip_finish_kernel<<<1, kThreads, 0, s>>>(c);
  return cudaGetLastError();
}

}  // namespace mb
