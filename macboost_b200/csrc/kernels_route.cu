// Choice of k models a row from gate logits, with its weights and gradient.
//
//   ids[n, :]     the k largest of l[n, :] in descending order, equal values by
//                 ascending index; -inf and NaN are never chosen (id -1, weight 0)
//   weights[n, j] exp(l_j - m) / S, m the row's largest logit, S the sum of
//                 exp(l - m) over the chosen (norm 0) or over all (norm 1)
//   gradient      with M = sum_j w_j dw_j over the choices that exist:
//                 norm 0: dl = w_j (dw_j - M) at choice j, 0 elsewhere
//                 norm 1: dl = w_j (dw_j - M) at choice j, -p_e M elsewhere, where
//                 p_e = w_0 exp(l_e - l_{id 0}): choice 0 has the largest
//                 probability, at least 1/E, so no sum over the row is taken again
//
// Three shapes.  Up to 16 logits: a lane a row, the number of logits a constant of the
// kernel, so that a row is registers and a choice 5 E instructions.  Up to 64: L lanes
// a row, a choice a local maximum and log2 L shuffles.  Both pass the logits through
// shared memory, since a lane's own loads would touch one 32-byte sector for every few
// values of a row.  Wider: a warp a row.  Each lane keeps the best two of its values
// and two reductions name the winner, so a choice is about 20 instructions however wide
// the row; a lane that has given both away looks through its values again, and its warp
// with it.  Lane j keeps choice j, and the exponentials, divisions and stores are one for all choices.
// All are bound by instructions: 1M x 10, two choices, 14 us and 11 its gradient; 65,537 x
// 256, eight choices of the full softmax, 48 us (16 lanes a row and a shuffle tree a
// choice: 70) and 27 its gradient (5 TB/s).
#include <cuda_runtime.h>

#include <cmath>

#include "mixture.h"

namespace mb {

namespace {

constexpr int kWarps = 4;               // warps a block
constexpr int kStaged = 64;             // widest row that passes through shared memory
constexpr int kTile = 544;              // floats of a warp's tile: 32 x 17, 16 x 33 or 8 x 65

__device__ __forceinline__ float not_nan(float v) { return v != v ? -INFINITY : v; }

// exp(x) of a probability beside the largest one, x <= 0: the argument's rounding, |x|
// 2^-24 of e^x, is at most 2^-24 / e of 1.
__device__ __forceinline__ float exp_term(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// A choice's weight: 0 where there is none, also beside an infinite logit, whose row's sum is
// NaN.
__device__ __forceinline__ float weight(int id, float e, float total) {
  return id < 0 ? 0.f : e / (total > 0.f || total != total ? total : 1.f);
}

// A warp's rows (nr x E, row stride ld) between global memory and its tile, whose
// rows are E | 1 floats apart so that a column is free of bank conflicts.  i / E by
// a 16-bit reciprocal: exact for i < 512 and E <= 64.
template <class F>
__device__ __forceinline__ void each_value(int nr, int E, int lane, F f) {
  const unsigned inv = (65536u + unsigned(E) - 1u) / unsigned(E);
  for (int i = lane; i < nr * E; i += 32) {
    const int r = int((unsigned(i) * inv) >> 16);
    f(r, i - r * E);
  }
}

// Rows of L x V logits at most; E1: their number when a lane has a row (L = 1), else 0; K:
// choices of a lane's row that stay in registers, else 0.
template <int L, int V, int E1, int K>
__global__ void __launch_bounds__(kWarps * 32, E1 && E1 <= 12 ? 12 : 8)
    route_kernel(const RouteArgs a) {
  constexpr int R = 32 / L;             // rows a warp
  __shared__ float tile[kWarps][E1 ? 32 * (E1 | 1) : kTile];
  // the choices, written out together: k <= E1, else k <= min(16 L, 32)
  constexpr int kChoices = K ? 1 : E1 ? 32 * E1 : R * 32;
  __shared__ int s_id[kWarps][kChoices];
  __shared__ float s_e[kWarps][kChoices];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sub = lane % L, r = lane / L;
  const long long row0 = (long long)(blockIdx.x * (long long)kWarps + warp) * R;
  if (row0 >= a.rows) return;           // whole warps only: no block barrier below
  const int nr = int(a.rows - row0 < R ? a.rows - row0 : R);
  const int E = E1 ? E1 : a.experts, k = K ? K : a.k;
  float* t = tile[warp];
  const int sp = E | 1;
  if (E1 && nr == 32 && a.ld == E1) {
    // a whole tile of adjacent rows: 32 E consecutive values
    const float* p = a.logits + row0 * E1 + lane;
    float u[E1 ? E1 : 1];
#pragma unroll
    for (int i = 0; i < E1; ++i) u[i] = p[i * 32];
#pragma unroll
    for (int i = 0; i < E1; ++i) {
      const int at = i * 32 + lane;
      t[E1 % 2 ? at : at + at / (E1 ? E1 : 1)] = u[i];
    }
  } else {
    each_value(nr, E, lane, [&](int rr, int c) { t[rr * sp + c] = a.logits[(row0 + rr) * a.ld + c]; });
  }
  __syncwarp();
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * L + sub;
    v[i] = e < E && r < nr ? t[r * sp + e] : -INFINITY;
  }
  float top = 0.f, total = 0.f;
  int my_id[K ? K : 1];
  float my_e[K ? K : 1];
#pragma unroll
  for (int j = 0; j < (K ? K : k); ++j) {
    // NaN is never greater, so it is never chosen
    float best = -INFINITY;
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (v[i] > best) {
        best = v[i];
        at = i;
      }
    int id = at * L + sub;
#pragma unroll
    for (int o = L / 2; o > 0; o /= 2) {
      const float b2 = __shfl_xor_sync(~0u, best, o);
      const int i2 = __shfl_xor_sync(~0u, id, o);
      if (b2 > best || (b2 == best && i2 < id)) {
        best = b2;
        id = i2;
      }
    }
    const bool found = best > -INFINITY;
    if (j == 0) {
      top = found ? best : 0.f;
      if (a.norm == kRouteAll) {
#pragma unroll
        for (int i = 0; i < V; ++i) total += exp_term(not_nan(v[i]) - top);
#pragma unroll
        for (int o = L / 2; o > 0; o /= 2) total += __shfl_xor_sync(~0u, total, o);
      }
    }
    const float e = expf(best - top);   // 0 for -inf
    if (a.norm == kRouteChosen) total += e;
    if constexpr (K > 0) {
      my_id[j] = found ? id : -1;
      my_e[j] = e;
    } else if (sub == 0) {
      s_id[warp][r * k + j] = found ? id : -1;
      s_e[warp][r * k + j] = e;
    }
    if (j + 1 < k) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i * L + sub == id) v[i] = -INFINITY;
    }
  }
  if constexpr (K > 0) {
    // one store of K values a lane
    if (r < nr) {
      const long long at = (row0 + r) * K;
      if constexpr (K == 2) {
        *reinterpret_cast<int2*>(a.ids + at) = make_int2(my_id[0], my_id[1]);
        *reinterpret_cast<float2*>(a.weights + at) =
            make_float2(weight(my_id[0], my_e[0], total), weight(my_id[1], my_e[1], total));
      } else {
        a.ids[at] = my_id[0];
        a.weights[at] = weight(my_id[0], my_e[0], total);
      }
    }
    return;
  }
  // the group's lanes divide their row's choices by the same total
  __syncwarp();
  for (int j = sub; j < k; j += L)
    s_e[warp][r * k + j] = weight(s_id[warp][r * k + j], s_e[warp][r * k + j], total);
  __syncwarp();
  int* ids = a.ids + row0 * k;
  float* weights = a.weights + row0 * k;
  for (int i = lane; i < nr * k; i += 32) {
    ids[i] = s_id[warp][i];
    weights[i] = s_e[warp][i];
  }
}

// Floats in the order of unsigned integers; -0 and 0 are equal, NaN is as -inf.
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __float_as_uint(not_nan(v) + 0.f);
  return b ^ (unsigned(int(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned u) {
  return __uint_as_float(u ^ (unsigned(int(~u) >> 31) | 0x80000000u));
}
// A warp a row of up to 32 V logits.
template <int V>
__global__ void __launch_bounds__(kWarps * 32) route_wide_kernel(const RouteArgs a) {
  const int lane = threadIdx.x % 32;
  const long long row = blockIdx.x * (long long)kWarps + threadIdx.x / 32;
  if (row >= a.rows) return;
  const int E = a.experts, k = a.k;
  const float* p = a.logits + row * a.ld;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < E ? p[e] : -INFINITY;
  }
  const unsigned none = ordered(-INFINITY);
  // the lane's best two as keys with their indexes, the lower index first among equals
  unsigned k0 = none, k1 = none, i0 = 0, i1 = 0;
  auto put = [&](unsigned x, unsigned i) {
    const bool first = x > k0, second = x > k1;
    k1 = first ? k0 : second ? x : k1;
    i1 = first ? i0 : second ? i : i1;
    k0 = first ? x : k0;
    i0 = first ? i : i0;
  };
#pragma unroll
  for (int i = 0; i < V; ++i) put(ordered(v[i]), i * 32 + lane);
  unsigned mine = none, first = none;
  int id = -1;
  for (int j = 0; j < k; ++j) {
    const unsigned most = __reduce_max_sync(~0u, k0);
    if (most == none) break;            // nothing left to choose
    if (j == 0) first = most;
    const unsigned win = __reduce_min_sync(~0u, k0 == most ? i0 : ~0u);
    if (lane == j) {
      mine = most;
      id = int(win);
    }
    const bool won = k0 == most && i0 == win;
    k0 = won ? k1 : k0;
    i0 = won ? i1 : i0;
    k1 = won ? none : k1;
    if (__any_sync(~0u, won && k0 == none) && won) {
      // the best two behind the lane's last choice in (value, index) order
      k0 = k1 = none;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const unsigned x = ordered(v[i]), at = i * 32 + lane;
        if (x < most || (x == most && at > win)) put(x, at);
      }
    }
  }
  const float top = first == none ? 0.f : from_ordered(first);
  const float e = expf(from_ordered(mine) - top);  // 0 where there is no choice
  float total = 0.f;
  if (a.norm == kRouteAll) {
#pragma unroll
    for (int i = 0; i < V; ++i) total += exp_term(not_nan(v[i]) - top);
  } else {
    total = lane < k ? e : 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) total += __shfl_xor_sync(~0u, total, o);
  if (lane < k) {
    a.ids[row * k + lane] = id;
    a.weights[row * k + lane] = weight(id, e, total);
  }
}

// One choice's weight and upstream gradient, zero where there is none.
__device__ __forceinline__ void choice(const RouteArgs& a, long long row, int j, int* id, float* w,
                                       float* dw) {
  const int e = a.ids[row * a.k + j];
  const bool ok = unsigned(e) < unsigned(a.experts);
  *id = ok ? e : -1;
  *w = ok ? a.weights[row * a.k + j] : 0.f;
  *dw = ok ? a.dweights[row * a.k + j] : 0.f;
}

// Rows of up to 64 logits: 32 rows a warp when E <= 16 (E1 = E), 16 or 8 above, one
// lane a row, through the warp's tile; K as above.
template <int E1, int K>
__global__ void __launch_bounds__(kWarps * 32) route_grad_narrow_kernel(const RouteArgs a) {
  __shared__ float tile[kWarps][E1 ? 32 * (E1 | 1) : kTile];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int E = E1 ? E1 : a.experts, k = K ? K : a.k, sp = E | 1;
  const int R = E1 ? 32 : E <= 32 ? 16 : 8;
  const long long row0 = (long long)(blockIdx.x * (long long)kWarps + warp) * R;
  if (row0 >= a.rows) return;
  const int nr = int(a.rows - row0 < R ? a.rows - row0 : R);
  float* t = tile[warp];
  if (a.norm == kRouteAll)
    each_value(nr, E, lane, [&](int r, int c) { t[r * sp + c] = a.logits[(row0 + r) * a.ld + c]; });
  __syncwarp();
  if (lane < nr) {
    const long long row = row0 + lane;
    float* mine = t + lane * sp;
    float mean = 0.f, w0 = 0.f;
    int id0 = -1;
    int ids[K ? K : 1];
    float w[K ? K : 1], dw[K ? K : 1];
    if constexpr (K == 2) {
      const int2 i2 = *reinterpret_cast<const int2*>(a.ids + row * 2);
      const float2 w2 = *reinterpret_cast<const float2*>(a.weights + row * 2);
      const float2 d2 = *reinterpret_cast<const float2*>(a.dweights + row * 2);
      ids[0] = i2.x, ids[1] = i2.y;
      w[0] = w2.x, w[1] = w2.y;
      dw[0] = d2.x, dw[1] = d2.y;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (unsigned(ids[j]) >= unsigned(E)) {
          ids[j] = -1;
          w[j] = dw[j] = 0.f;
        }
    } else if constexpr (K == 1) {
      choice(a, row, 0, &ids[0], &w[0], &dw[0]);
    }
#pragma unroll
    for (int j = 0; j < (K ? K : k); ++j) {
      constexpr int one = 0;
      const int at = K ? j : one;
      if (!K) choice(a, row, j, &ids[at], &w[at], &dw[at]);
      if (j == 0) {
        id0 = ids[at];
        w0 = w[at];
      }
      mean += w[at] * dw[at];
    }
    if (a.norm == kRouteAll && id0 >= 0) {
      const float l0 = mine[id0];
#pragma unroll
      for (int e = 0; e < (E1 ? E1 : E); ++e) mine[e] = -mean * (w0 * exp_term(not_nan(mine[e]) - l0));
    } else {
#pragma unroll
      for (int e = 0; e < (E1 ? E1 : E); ++e) mine[e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < (K ? K : k); ++j) {
      const int at = K ? j : 0;
      if (!K) choice(a, row, j, &ids[at], &w[at], &dw[at]);
      if (ids[at] >= 0) mine[ids[at]] = w[at] * (dw[at] - mean);
    }
  }
  __syncwarp();
  if (E1 && nr == 32 && a.ld_d == E1) {
    float* p = a.dlogits + row0 * E1 + lane;
#pragma unroll
    for (int i = 0; i < E1; ++i) {
      const int at = i * 32 + lane;
      p[i * 32] = t[E1 % 2 ? at : at + at / (E1 ? E1 : 1)];
    }
  } else {
    each_value(nr, E, lane,
               [&](int r, int c) { a.dlogits[(row0 + r) * a.ld_d + c] = t[r * sp + c]; });
  }
}

// Wider rows: a warp a row, lane j holding choice j.  VEC: rows of both matrices are
// 16-byte aligned and a multiple of 4 long.
template <bool VEC>
__global__ void __launch_bounds__(kWarps * 32) route_grad_kernel(const RouteArgs a) {
  const int lane = threadIdx.x % 32;
  const long long row = blockIdx.x * (long long)kWarps + threadIdx.x / 32;
  if (row >= a.rows) return;
  const int E = a.experts;
  int id = -1;
  float w = 0.f, dw = 0.f;
  if (lane < a.k) choice(a, row, lane, &id, &w, &dw);
  float mean = w * dw;
#pragma unroll
  for (int o = 16; o > 0; o /= 2) mean += __shfl_xor_sync(~0u, mean, o);
  const int id0 = __shfl_sync(~0u, id, 0);
  const float* l = a.logits + row * a.ld;
  float* d = a.dlogits + row * a.ld_d;
  const bool all = a.norm == kRouteAll && id0 >= 0;
  const float scale = all ? -mean * __shfl_sync(~0u, w, 0) : 0.f;
  const float l0 = all ? l[id0] : 0.f;
  if (VEC) {
    for (int e = lane * 4; e < E; e += 128) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (all) {
        q = *reinterpret_cast<const float4*>(l + e);
        q.x = scale * exp_term(not_nan(q.x) - l0);
        q.y = scale * exp_term(not_nan(q.y) - l0);
        q.z = scale * exp_term(not_nan(q.z) - l0);
        q.w = scale * exp_term(not_nan(q.w) - l0);
      }
      *reinterpret_cast<float4*>(d + e) = q;
    }
  } else {
    for (int e = lane; e < E; e += 32) d[e] = all ? scale * exp_term(not_nan(l[e]) - l0) : 0.f;
  }
  __syncwarp();  // the warp's own stores before the choices' values replace some of them
  if (id >= 0) d[id] = w * (dw - mean);
}

unsigned blocks_for(long long rows, int per) { return unsigned((rows + per - 1) / per); }

template <int L, int V, int E1, int K>
cudaError_t go_k(const RouteArgs& a, bool grad, cudaStream_t s) {
  // at least 32 rows a block and below 2^31 rows: the grid fits
  if (grad) {
    const int R = E1 ? 32 : a.experts <= 32 ? 16 : 8;
    route_grad_narrow_kernel<E1, K><<<blocks_for(a.rows, kWarps * R), kWarps * 32, 0, s>>>(a);
  } else {
    route_kernel<L, V, E1, K><<<blocks_for(a.rows, kWarps * (32 / L)), kWarps * 32, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <int L, int V, int E1>
cudaError_t go(const RouteArgs& a, bool grad, cudaStream_t s) {
  if constexpr (E1 > 0) {
    if (a.k == 1) return go_k<L, V, E1, 1>(a, grad, s);
    // two choices by one 8-byte access, where the arrays start on 8 bytes
    if constexpr (E1 > 1) {
      const auto at = reinterpret_cast<uintptr_t>(a.ids) | reinterpret_cast<uintptr_t>(a.weights) |
                      reinterpret_cast<uintptr_t>(a.dweights);
      if (a.k == 2 && at % 8 == 0) return go_k<L, V, E1, 2>(a, grad, s);
    }
  }
  return go_k<L, V, E1, 0>(a, grad, s);
}

template <int V>
cudaError_t wide(const RouteArgs& a, cudaStream_t s) {
  route_wide_kernel<V><<<blocks_for(a.rows, kWarps), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t narrow(const RouteArgs& a, bool grad, cudaStream_t s) {
  switch (a.experts) {
#define MB_ROUTE(E) case E: return go<1, E, E>(a, grad, s);
    MB_ROUTE(1) MB_ROUTE(2) MB_ROUTE(3) MB_ROUTE(4) MB_ROUTE(5) MB_ROUTE(6) MB_ROUTE(7)
    MB_ROUTE(8) MB_ROUTE(9) MB_ROUTE(10) MB_ROUTE(11) MB_ROUTE(12) MB_ROUTE(13) MB_ROUTE(14)
    MB_ROUTE(15) MB_ROUTE(16)
#undef MB_ROUTE
    default: break;
  }
  return a.experts <= 32 ? go<2, 16, 0>(a, grad, s) : go<4, 16, 0>(a, grad, s);
}

}  // namespace

cudaError_t launch_route(const RouteArgs& a, cudaStream_t s) {
  const int E = a.experts;
  if (E <= kStaged) return narrow(a, false, s);
  if (E <= 128) return wide<4>(a, s);
  if (E <= 256) return wide<8>(a, s);
  if (E <= 512) return wide<16>(a, s);
  return wide<32>(a, s);
}

cudaError_t launch_route_grad(const RouteArgs& a, cudaStream_t s) {
  const int E = a.experts;
  if (E <= kStaged) return narrow(a, true, s);
  const auto bits = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits);
  if (bits % 16 == 0 && (a.ld | a.ld_d | E) % 4 == 0)
    route_grad_kernel<true><<<blocks_for(a.rows, kWarps), kWarps * 32, 0, s>>>(a);
  else
    route_grad_kernel<false><<<blocks_for(a.rows, kWarps), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mb
