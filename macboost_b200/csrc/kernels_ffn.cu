// The gated block of few rows (ffn.h); more rows are tiles of the tensor cores
// (kernels_head.cu).
//
// Two launches, h between them.  The rows lie in shared memory in float32; a warp streams
// two rows of weights (two gates and their two factors) at a time through registers, 16
// bytes a lane, eight loads on their way, and its sums meet in shuffles.  Reading the weights
// bounds it: one row of 4,096 x 16,384 x 4,096 bfloat16 (403 MB) 69 us, 5.8 TB/s; of 2,048 x 8,192
// float32 41 us.  More rows of bfloat16 are products of warps, or where rows do not start on 16
// bytes up to four of them here.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "activation.cuh"
#include "ffn.h"
#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Few {
  const void* in;      // rows x cols
  long long ld_in;
  const void* w;       // weights, stride ld_w
  long long ld_w;
  int rows, cols, outs, pitch, act;
  void* out;           // rows x outs
  long long ld_out;
  float* pre;          // gated: rows x 2 outs, or null
  long long ld_pre;
  unsigned* status;    // cleared by the first launch: there is no wait to run out
};

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// PER adjacent weights as floats.
template <class T, int PER>
struct Load;
template <class T>
struct Load<T, 1> {
  T v;
  __device__ __forceinline__ void get(const T* p) { v = *p; }
  __device__ __forceinline__ void values(float (&x)[1]) const { x[0] = float(v); }
};
template <>
struct Load<float, 4> {
  float4 v;
  __device__ __forceinline__ void get(const float* p) { v = __ldcs(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void values(float (&x)[4]) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
};
template <>
struct Load<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void get(const __nv_bfloat16* p) { v = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
};

template <class T, int NR, int PER, bool GATE>
__global__ void __launch_bounds__(kThreads) ffn_few_kernel(const Few a) {
  constexpr int C = 2;                        // outputs a warp
  constexpr int R = GATE ? 2 * C : C;         // rows of weights
  constexpr int STEPS = 8 / R;                // of each, on their way at once
  // float32: shorter sums, which are then added up, round less; many rows have no registers for it
  constexpr bool PARTS = sizeof(T) == 4 && NR <= 4;
  extern __shared__ float4 few_shared[];
  float* rows = reinterpret_cast<float*>(few_shared);  // NR x pitch
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (GATE && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  // the rows, PER values at a time, all of a thread's loads on their way: a value after the
  // other took 6 us of 16,384
  for (int n = 0; n < NR; ++n) {
    const T* from = static_cast<const T*>(a.in) + n * a.ld_in;
    const bool whole = PER > 1 && n < a.rows && (reinterpret_cast<uintptr_t>(from) & 15) == 0;
    if (whole) {
#pragma unroll 8
      for (int d = threadIdx.x * PER; d < a.cols; d += kThreads * PER) {
        Load<T, PER> q;
        q.get(from + d);
        float v[PER];
        q.values(v);
#pragma unroll
        for (int i = 0; i < PER; i += 4)
          *reinterpret_cast<float4*>(rows + n * a.pitch + d + i) =
              make_float4(v[i], v[i + (PER > 1)], v[i + 2 * (PER > 2)], v[i + 3 * (PER > 2)]);
      }
    } else {
#pragma unroll 8
      for (int d = threadIdx.x; d < a.cols; d += kThreads)
        rows[n * a.pitch + d] = n < a.rows ? float(from[d]) : 0.f;
    }
  }
  __syncthreads();
  const int stride = int(gridDim.x) * kWarps * C;
  for (int o0 = (int(blockIdx.x) * kWarps + warp) * C; o0 < a.outs; o0 += stride) {
    const T* w[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      w[r] = static_cast<const T*>(a.w) +
             (min(o0 + r % C, a.outs - 1) + (r >= C ? (long long)a.outs : 0)) * a.ld_w;
    float acc[R][NR];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[r][n] = 0.f;
    for (int d0 = lane * PER; d0 < a.cols; d0 += STEPS * 32 * PER) {
      Load<T, PER> q[STEPS][R];
#pragma unroll
      for (int t = 0; t < STEPS; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (d0 + t * 32 * PER < a.cols) q[t][r].get(w[r] + d0 + t * 32 * PER);
      float part[R][NR];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NR; ++n) part[r][n] = PARTS ? 0.f : acc[r][n];
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        const int d = d0 + t * 32 * PER;
        if (d >= a.cols) break;
        float x[NR][PER];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          if constexpr (PER == 1) {
            x[n][0] = rows[n * a.pitch + d];
          } else {
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) {
              const float4 f = *reinterpret_cast<const float4*>(rows + n * a.pitch + d + 4 * i);
              x[n][4 * i] = f.x, x[n][4 * i + 1] = f.y, x[n][4 * i + 2] = f.z, x[n][4 * i + 3] = f.w;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float v[PER];
          q[t][r].values(v);
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int i = 0; i < PER; ++i) part[r][n] = fmaf(v[i], x[n][i], part[r][n]);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[r][n] = PARTS ? acc[r][n] + part[r][n] : part[r][n];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int o = 16; o > 0; o /= 2) acc[r][n] += __shfl_xor_sync(~0u, acc[r][n], o);
    // lane c * NR + n writes output c of row n
    static_assert(C * NR <= 32, "a lane each");
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (lane == c * NR + n && n < a.rows && o0 + c < a.outs) {
          float y = acc[c][n];
          if constexpr (GATE) {
            const float up = acc[C + c][n];
            if (a.pre) {
              float* p = a.pre + n * a.ld_pre + o0 + c;
              p[0] = y;
              p[a.outs] = up;
            }
            float v[1] = {y};
            const float u[1] = {up};
            activate<sizeof(T) == 2>(a.act, v, u);
            y = v[0];
          }
          static_cast<T*>(a.out)[n * a.ld_out + o0 + c] = from_float<T>(y);  // h as in the tiles: rounded here
        }
  }
}

template <class T, int NR, int PER, bool GATE>
cudaError_t few_of(const Few& a, cudaStream_t s) {
  // the limit of the largest call: it is the kernel's, and other threads launch it too
  const auto k = ffn_few_kernel<T, NR, PER, GATE>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kFfnFewSmem));
  if (e != cudaSuccess) return e;
  const size_t smem = size_t(NR) * size_t(a.pitch) * sizeof(float);
  const int per = int(std::max<size_t>(1, std::min<size_t>(4, (200 * 1024) / (smem + 1024))));
  const int blocks = std::min((a.outs + 2 * kWarps - 1) / (2 * kWarps), per * device_sms());
  k<<<blocks, kThreads, smem, s>>>(a);
  return cudaGetLastError();
}

template <class T, int PER, bool GATE>
cudaError_t few_rows(const Few& a, cudaStream_t s) {
  if (a.rows <= 1) return few_of<T, 1, PER, GATE>(a, s);
  if (a.rows <= 2) return few_of<T, 2, PER, GATE>(a, s);
  if (a.rows <= 4) return few_of<T, 4, PER, GATE>(a, s);
  if constexpr (sizeof(T) == 4) {
    if (a.rows <= 8) return few_of<T, 8, PER, GATE>(a, s);
    return few_of<T, 16, PER, GATE>(a, s);
  }
  return cudaErrorInvalidValue;
}

template <class T, bool GATE>
cudaError_t few_type(const Few& a, cudaStream_t s) {
  constexpr int PER = 16 / int(sizeof(T));
  const bool wide = (reinterpret_cast<uintptr_t>(a.w) | uintptr_t(a.ld_w) * sizeof(T) |
                     uintptr_t(a.cols) * sizeof(T)) % 16 == 0;
  return wide ? few_rows<T, PER, GATE>(a, s) : few_rows<T, 1, GATE>(a, s);
}

// ---- bfloat16: up to 48 rows by products of warps ---------------------------------------
//
// What ffn_few_kernel spends on a weight (unpacking, a product a row, rows from shared memory) takes
// longer than fetching it from two rows on.  Here a warp's mma.m16n8k16 has 16 rows of weights as A
// and eight rows of x as B.  The order of K within a product is free, so a lane takes 16 adjacent
// bytes of a row of weights, and the same of a row of x, as its part of two products: no
// shuffles, nothing through shared memory.  A block's warps share K, WARPS chunks of 128 at a
// time, and join their sums in shared memory in one order.  x and h are read over and over from the
// L1 cache, where weights leave no trace.  Gates are an A's first eight rows and their factors its
// last eight, so a lane's sums are of both.
//
// Measured, 2,048 x 8,192 x 2,048 (101 MB of weights): 25 us at 2 to 8 rows (4.1 TB/s, both
// launches), 27 at 16, 35 at 24, 41 at 32; x and h from the L1 and L2 caches bound it from there
// on (at 48 rows the first launch reads 187 MB from L2 and takes 40 us; tiles of the tensor
// cores take 45 to 47 for any of these).  1,024 x 4,096: 10.4, 12.4, 16.5 and 20.6 us at 8, 16, 32 and
// 48 rows against 27 to 33.  Two A's a warp: the same up to 16 rows, 45 and 64 us at 32 and 48.

struct Rows16 {
  uint4 v;
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void stream(const __nv_bfloat16* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  }
};

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                      uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: eights of rows.
template <int WARPS, int NT, bool GATE>
__global__ void __launch_bounds__(WARPS * 32) ffn_rows_kernel(const Few a) {
  constexpr int STEPS = 4;                          // of 32 of K, on their way at once
  constexpr int OUTS = GATE ? 8 : 16;               // of an A
  __shared__ float4 sums[WARPS][NT][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  if (GATE && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  const __nv_bfloat16* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)                      // a row that is not there: another's sums, never written
    x[n] = static_cast<const __nv_bfloat16*>(a.in) + min(8 * n + g, a.rows - 1) * a.ld_in + 8 * t;
  const int units = (a.outs + OUTS - 1) / OUTS;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int o = unit * OUTS;
    const long long lo = min(o + g, a.outs - 1), hi = GATE ? lo + a.outs : min(o + 8 + g, a.outs - 1);
    const __nv_bfloat16* w0 = static_cast<const __nv_bfloat16*>(a.w) + lo * a.ld_w + 8 * t;
    const __nv_bfloat16* w1 = static_cast<const __nv_bfloat16*>(a.w) + hi * a.ld_w + 8 * t;
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
    for (int d0 = warp * 32 * STEPS; d0 < a.cols; d0 += WARPS * 32 * STEPS) {
      Rows16 q0[STEPS], q1[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        q0[i].clear(), q1[i].clear();
        if (d0 + 32 * i + 8 * t < a.cols) q0[i].stream(w0 + d0 + 32 * i), q1[i].stream(w1 + d0 + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        uint4 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          b[n] = make_uint4(0, 0, 0, 0);
          if (d0 + 32 * i + 8 * t < a.cols) b[n] = *reinterpret_cast<const uint4*>(x[n] + d0 + 32 * i);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16(c[n], q0[i].v.x, q1[i].v.x, q0[i].v.y, q1[i].v.y, b[n].x, b[n].y);
          mma16(c[n], q0[i].v.z, q1[i].v.z, q0[i].v.w, q1[i].v.w, b[n].z, b[n].w);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[warp][n][lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
    __syncthreads();
    if (warp < NT) {
      float v[4] = {};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float4 f = sums[w][warp][lane];
        v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
      }
      // v[0], v[1]: output g of rows 2 t and 2 t + 1; v[2], v[3]: their factors, or output g + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 8 * warp + 2 * t + i;
        if (row >= a.rows) continue;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + row * a.ld_out;
        if constexpr (GATE) {
          if (o + g < a.outs) {
            if (a.pre) {
              float* p = a.pre + row * a.ld_pre + o + g;
              p[0] = v[i];
              p[a.outs] = v[2 + i];
            }
            float y[1] = {v[i]};
            const float u[1] = {v[2 + i]};
            activate<true>(a.act, y, u);  // h is rounded, as in the tiles
            out[o + g] = __float2bfloat16_rn(y[0]);
          }
        } else {
          if (o + g < a.outs) out[o + g] = __float2bfloat16_rn(v[i]);
          if (o + 8 + g < a.outs) out[o + 8 + g] = __float2bfloat16_rn(v[2 + i]);
        }
      }
    }
    if (unit + int(gridDim.x) < units) __syncthreads();  // before the next unit's sums
  }
}

template <int NT, bool GATE>
cudaError_t rows_of(const Few& a, cudaStream_t s) {
  const int units = (a.outs + (GATE ? 8 : 16) - 1) / (GATE ? 8 : 16), sms = device_sms();
  // sixteen warps where there is no second block for a multiprocessor
  if (units <= sms)
    ffn_rows_kernel<16, NT, GATE><<<units, 512, 0, s>>>(a);
  else
    ffn_rows_kernel<8, NT, GATE><<<std::min(units, 4 * sms), 256, 0, s>>>(a);
  return cudaGetLastError();
}

// ---- bfloat16, long rows of x: the activation after the product -------------------------
//
// A thread a value: 10 bytes of it, beside 65,536 products and more.
__global__ void __launch_bounds__(kThreads)
    ffn_gate_kernel(int act, const float* pre, long long ld_pre, __nv_bfloat16* hidden, long long ld_hidden,
                    long long rows, int width) {
  const long long all = rows * width, step = (long long)gridDim.x * kThreads;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < all; i += step) {
    const long long n = i / width;
    const int c = int(i - n * width);
    const float* p = pre + n * ld_pre + c;
    float v[1] = {p[0]};
    const float u[1] = {p[width]};
    activate<true>(act, v, u);
    hidden[n * ld_hidden + c] = __float2bfloat16_rn(v[0]);
  }
}

// ---- float32: the gradients of gates and factors ----------------------------------
//
// The tensor cores' epilogue keeps 128 sums a thread in float32, and fetching pre and three
// planes a half on top of that stopped it for 85 us a tile of 256 x 256.  Written out as float32
// and formed here: 30 bytes a value, 2,048 x 4,096 in 42 us (6.0 TB/s).

// Four adjacent values as three planes of bfloat16, `plane` apart.  As the head's planes:
// finite values that would round to infinity are bfloat16's largest and a rest, and the rest
// of what is not finite is zero.
__device__ __forceinline__ void put_planes(__nv_bfloat16* to, long long plane, const float (&x)[4]) {
  constexpr float kLargest = 3.3895313892515355e38f;
  float v[4] = {x[0], x[1], x[2], x[3]};
  // (a NaN is not below anything)
  const bool plain = fabsf(x[0]) < kLargest && fabsf(x[1]) < kLargest && fabsf(x[2]) < kLargest && fabsf(x[3]) < kLargest;
  if (plain) {
#pragma unroll
    for (int z = 0; z < 3; ++z) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
      uint2 w;
      memcpy(&w.x, &lo, 4);
      memcpy(&w.y, &hi, 4);
      *reinterpret_cast<uint2*>(to + z * plane) = w;
      v[0] -= __uint_as_float(w.x << 16), v[1] -= __uint_as_float(w.x & 0xFFFF0000u);
      v[2] -= __uint_as_float(w.y << 16), v[3] -= __uint_as_float(w.y & 0xFFFF0000u);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = fabsf(x[i]) < INFINITY ? fminf(fmaxf(x[i], -kLargest), kLargest) : x[i];
#pragma unroll
  for (int z = 0; z < 3; ++z) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    uint2 w;
    memcpy(&w.x, &lo, 4);
    memcpy(&w.y, &hi, 4);
    *reinterpret_cast<uint2*>(to + z * plane) = w;
    const float t[4] = {__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u),
                        __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = z == 0 ? (fabsf(x[i]) < INFINITY ? x[i] - t[i] : 0.f) : v[i] - t[i];
  }
}

// The same, rounded once (bfloat16).
__device__ __forceinline__ void put_rounded(__nv_bfloat16* to, const float (&x)[4]) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
  uint2 w;
  memcpy(&w.x, &lo, 4);
  memcpy(&w.y, &hi, 4);
  *reinterpret_cast<uint2*>(to) = w;
}

// 128 columns a warp, four adjacent ones a lane.  WIDE: rows of dh, hidden and both halves of pre
// start on 16 bytes; else they are read side by side and change lanes in shared memory.
template <bool F32, bool WIDE>
__global__ void __launch_bounds__(kThreads) ffn_split_kernel(const FfnSplit a, int per) {
  __shared__ float turn[WIDE ? 1 : kWarps][WIDE ? 1 : 128];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long w = (long long)blockIdx.x * kWarps + warp, n = w / per;
  if (n >= a.rows) return;
  const int c0 = int(w - n * per) * 128, c = c0 + lane * 4;
  auto get = [&](const float* p, float (&x)[4]) {
    if constexpr (WIDE) {
      const float4 f = c < a.width ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = c0 + 32 * k + lane < a.width ? p[c0 + 32 * k + lane] : 0.f;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) turn[warp][32 * k + lane] = x[k];
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = turn[warp][4 * lane + k];
    }
  };
  float dh[4], x[4], y[4], h[4], dx[4], dy[4];
  get(a.dh + n * a.ld_dh, dh);
  get(a.pre + n * a.ld_pre, x);
  get(a.pre + n * a.ld_pre + a.width, y);
  if (a.h) get(a.hidden + n * a.ld_hidden, h);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    gate_grad<!F32>(a.act, x[k], y[k], dh[k], dx[k], dy[k]);
    if (c + k >= a.width) dx[k] = dy[k] = 0.f;
  }
  if (c < a.half) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(a.dpre) + n * 2 * a.half + c;
    if constexpr (F32) {
      put_planes(d, a.rows * 2 * a.half, dx);
      put_planes(d + a.half, a.rows * 2 * a.half, dy);
    } else {
      put_rounded(d, dx);
      put_rounded(d + a.half, dy);
    }
  }
  if (a.h && c < a.ld_h) put_planes(static_cast<__nv_bfloat16*>(a.h) + n * a.ld_h + c, a.rows * a.ld_h, h);
}

// ---- float32, few outputs ------------------------------------------------------------
//
// y = h Wo^T: a warp has four rows, a lane every 32nd column of them, and all outputs' sums, which lanes
// then halve among themselves.  The gradients in one pass over pre, h and dy: a warp has 128
// columns, four adjacent ones a lane, of `per` rows; its part of Wo and its sums of dw_out stay in
// registers, dy comes by shuffles.  10,007 x 403 x 10, rows of odd length: 20 and 43 us (and 9 for dw_out's
// sums of rows) in place of 36 (planes of h, tiles) and 94 (dh, the split above, dw_out and its
// sums); loads and stores of a few bytes a lane bound the second (twice as many warps with Wo in
// shared memory: 49).  Whole steps in us, against tiles: 10,007 x 100 x 403 x 10 138 and 197, 500 rows 55
// and 85, 20,000 x 256 x 1,024 x 16 635 and 755, 5,000 x 1,024 x 4,096 x 4 1,533 and 1,674.

template <int OUTS>
__global__ void __launch_bounds__(kThreads)
    ffn_narrow_kernel(const float* __restrict__ h, long long ld_h, const float* __restrict__ w, long long ld_w,
                      float* y, long long ld_y, long long rows, int width, int outs) {
  constexpr int R = 4;
  const int lane = threadIdx.x % 32;
  const long long n0 = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * R;
  if (n0 >= rows) return;
  const float* from[R];
#pragma unroll
  for (int r = 0; r < R; ++r) from[r] = h + min(n0 + r, rows - 1) * ld_h;
  float v[R * OUTS];
#pragma unroll
  for (int i = 0; i < R * OUTS; ++i) v[i] = 0.f;
#pragma unroll 2
  for (int c = lane; c < width; c += 32) {
    float x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = __ldg(from[r] + c);
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      const float f = __ldg(w + min(o, outs - 1) * ld_w + c);
#pragma unroll
      for (int r = 0; r < R; ++r) v[r * OUTS + o] = fmaf(x[r], f, v[r * OUTS + o]);
    }
  }
  // at each step a lane keeps one half of its sums and hands the other over
  int first = 0, n = R * OUTS;
#pragma unroll
  for (int step = 16; step > 0; step /= 2) {
    if (n % 2 == 0) {
      n /= 2;
      const bool high = lane & step;
#pragma unroll
      for (int i = 0; i < R * OUTS / 2; ++i)
        if (i < n) v[i] = (high ? v[n + i] : v[i]) + __shfl_xor_sync(~0u, high ? v[i] : v[n + i], step);
      first += high ? n : 0;
    } else {
#pragma unroll
      for (int i = 0; i < R * OUTS; ++i)
        if (i < n) v[i] += __shfl_xor_sync(~0u, v[i], step);
    }
  }
#pragma unroll
  for (int i = 0; i < R * OUTS; ++i)
    if (i < n) {
      const int r = (first + i) / OUTS, o = (first + i) % OUTS;
      if (n0 + r < rows && o < outs) y[(n0 + r) * ld_y + o] = v[i];
    }
}

template <int OUTS, bool WIDE>
__global__ void __launch_bounds__(kThreads) ffn_narrow_grad_kernel(const FfnNarrow a, int groups, long long chunks) {
  const int lane = threadIdx.x % 32;
  const long long item = (long long)blockIdx.x * kWarps + threadIdx.x / 32, chunk = item / groups;
  if (chunk >= chunks) return;
  const int c = int(item - chunk * groups) * 128 + lane * 4;
  auto get = [&](const float* p, float (&x)[4]) {
    if constexpr (WIDE) {
      const float4 f = c < a.width ? __ldg(reinterpret_cast<const float4*>(p + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = c + k < a.width ? __ldg(p + c + k) : 0.f;
    }
  };
  float w[OUTS][4], sum[OUTS][4];
#pragma unroll
  for (int o = 0; o < OUTS; ++o) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[o][k] = o < a.outs && c + k < a.width ? a.w[o * a.ld_w + c + k] : 0.f;
      sum[o][k] = 0.f;
    }
  }
  const long long lo = chunk * a.per, hi = min(lo + a.per, a.rows);
  float x[4], y[4], h[4], g;  // of the next row
  auto fetch = [&](long long n) {
    g = lane < a.outs ? __ldg(a.dy + n * a.ld_dy + lane) : 0.f;
    if (a.dpre) {
      get(a.pre + n * a.ld_pre, x);
      get(a.pre + n * a.ld_pre + a.width, y);
    }
    if (a.part) get(a.hidden + n * a.ld_hidden, h);
  };
  fetch(lo);
#pragma unroll 1
  for (long long n = lo; n < hi; ++n) {
    float x0[4], y0[4], h0[4], dh[4] = {};
    const float g0 = g;
#pragma unroll
    for (int k = 0; k < 4; ++k) x0[k] = x[k], y0[k] = y[k], h0[k] = h[k];
    if (n + 1 < hi) fetch(n + 1);
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      const float d = __shfl_sync(~0u, g0, o);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        dh[k] = fmaf(d, w[o][k], dh[k]);
        if (a.part) sum[o][k] = fmaf(d, h0[k], sum[o][k]);
      }
    }
    if (!a.dpre) continue;
    float dx[4], dz[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      gate_grad<false>(a.act, x0[k], y0[k], dh[k], dx[k], dz[k]);
      if (c + k >= a.width) dx[k] = dz[k] = 0.f;
    }
    if (c < a.half) {
      __nv_bfloat16* d = static_cast<__nv_bfloat16*>(a.dpre) + n * 2 * a.half + c;
      put_planes(d, a.rows * 2 * a.half, dx);
      put_planes(d + a.half, a.rows * 2 * a.half, dz);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int o = 0; o < OUTS; ++o)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o < a.outs && c + k < a.width) a.part[(chunk * a.outs + o) * a.width + c + k] = sum[o][k];
}

template <int OUTS>
cudaError_t narrow_grad(const FfnNarrow& a, cudaStream_t s) {
  const int groups = (a.half + 127) / 128;
  const long long chunks = (a.rows + a.per - 1) / a.per, blocks = (chunks * groups + kWarps - 1) / kWarps;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  const bool wide = (reinterpret_cast<uintptr_t>(a.pre) | reinterpret_cast<uintptr_t>(a.hidden) | uintptr_t(a.ld_pre) * 4 |
                     uintptr_t(a.ld_hidden) * 4 | uintptr_t(a.width) * 4) % 16 == 0;
  if (wide)
    ffn_narrow_grad_kernel<OUTS, true><<<unsigned(blocks), kThreads, 0, s>>>(a, groups, chunks);
  else
    ffn_narrow_grad_kernel<OUTS, false><<<unsigned(blocks), kThreads, 0, s>>>(a, groups, chunks);
  return cudaGetLastError();
}

template <int OUTS>
cudaError_t narrow(const FfnArgs& a, cudaStream_t s) {
  const long long blocks = (a.rows + 4 * kWarps - 1) / (4 * kWarps);
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  ffn_narrow_kernel<OUTS><<<unsigned(blocks), kThreads, 0, s>>>(
      static_cast<const float*>(a.hidden), a.ld_hidden, static_cast<const float*>(a.w_out), a.ld_out,
      static_cast<float*>(a.y), a.ld_y, a.rows, int(a.width), int(a.outs));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ffn_narrow(const FfnArgs& a, cudaStream_t s) {
  if (a.outs <= 4) return narrow<4>(a, s);
  if (a.outs <= 8) return narrow<8>(a, s);
  if (a.outs <= 12) return narrow<12>(a, s);
  return a.outs <= kFfnNarrow ? narrow<16>(a, s) : cudaErrorInvalidValue;
}

cudaError_t launch_ffn_narrow_grad(const FfnNarrow& a, cudaStream_t s) {
  if (a.outs <= 4) return narrow_grad<4>(a, s);
  if (a.outs <= 8) return narrow_grad<8>(a, s);
  if (a.outs <= 12) return narrow_grad<12>(a, s);
  return a.outs <= kFfnNarrow ? narrow_grad<16>(a, s) : cudaErrorInvalidValue;
}

cudaError_t launch_ffn_split(const FfnSplit& a, cudaStream_t s) {
  const int per = (a.half + 127) / 128;  // warps a row
  const long long blocks = (a.rows * per + kWarps - 1) / kWarps;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  const uintptr_t hidden = a.h ? reinterpret_cast<uintptr_t>(a.hidden) | uintptr_t(a.ld_hidden) * 4 : 0;
  const bool wide = (reinterpret_cast<uintptr_t>(a.dh) | reinterpret_cast<uintptr_t>(a.pre) | hidden |
                     uintptr_t(a.ld_dh) * 4 | uintptr_t(a.ld_pre) * 4 | uintptr_t(a.width) * 4) % 16 == 0;
  if (a.dtype != kF32 && wide)
    ffn_split_kernel<false, true><<<unsigned(blocks), kThreads, 0, s>>>(a, per);
  else if (a.dtype != kF32)
    ffn_split_kernel<false, false><<<unsigned(blocks), kThreads, 0, s>>>(a, per);
  else if (wide)
    ffn_split_kernel<true, true><<<unsigned(blocks), kThreads, 0, s>>>(a, per);
  else
    ffn_split_kernel<true, false><<<unsigned(blocks), kThreads, 0, s>>>(a, per);
  return cudaGetLastError();
}

cudaError_t launch_ffn_gate(const FfnArgs& a, const float* pre, int64_t ld_pre, cudaStream_t s) {
  const long long blocks = (a.rows * a.width + kThreads - 1) / kThreads;
  ffn_gate_kernel<<<unsigned(std::min<long long>(blocks, 8 * device_sms())), kThreads, 0, s>>>(
      a.act, pre, ld_pre, static_cast<__nv_bfloat16*>(a.hidden), a.ld_hidden, a.rows, int(a.width));
  return cudaGetLastError();
}

namespace {

// Both products' arguments.
Few few_in(const FfnArgs& f) {
  Few a{};
  a.in = f.x;
  a.ld_in = f.ld_x;
  a.w = f.w_in;
  a.ld_w = f.ld_in;
  a.rows = int(f.rows);
  a.cols = int(f.cols);
  a.outs = int(f.width);
  a.pitch = int(ffn_pitch(f.cols));
  a.act = f.act;
  a.out = f.hidden;
  a.ld_out = f.ld_hidden;
  a.pre = f.pre;
  a.ld_pre = f.ld_pre;
  a.status = static_cast<unsigned*>(f.workspace);
  return a;
}

Few few_out(const FfnArgs& f) {
  Few a{};
  a.in = f.hidden;
  a.ld_in = f.ld_hidden;
  a.w = f.w_out;
  a.ld_w = f.ld_out;
  a.rows = int(f.rows);
  a.cols = int(f.width);
  a.outs = int(f.outs);
  a.pitch = int(ffn_pitch(f.width));
  a.out = f.y;
  a.ld_out = f.ld_y;
  return a;
}

}  // namespace

cudaError_t launch_ffn_few(const FfnArgs& f, cudaStream_t s) {
  const Few in = few_in(f), out = few_out(f);
  const bool f32 = f.dtype == kF32;
  const cudaError_t e = f32 ? few_type<float, true>(in, s) : few_type<__nv_bfloat16, true>(in, s);
  if (e != cudaSuccess) return e;
  return f32 ? few_type<float, false>(out, s) : few_type<__nv_bfloat16, false>(out, s);
}

template <bool GATE>
static cudaError_t rows_type(const Few& a, cudaStream_t s) {
  if (a.rows <= 8) return rows_of<1, GATE>(a, s);
  if (a.rows <= 16) return rows_of<2, GATE>(a, s);
  if (a.rows <= 24) return rows_of<3, GATE>(a, s);
  if (a.rows <= 32) return rows_of<4, GATE>(a, s);
  if (a.rows <= 48) return rows_of<6, GATE>(a, s);
  return cudaErrorInvalidValue;
}

cudaError_t launch_ffn_rows(const FfnArgs& f, cudaStream_t s) {
  const cudaError_t e = rows_type<true>(few_in(f), s);
  return e != cudaSuccess ? e : rows_type<false>(few_out(f), s);
}

}  // namespace mb
