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
// A row belongs to L lanes that hold V logits each in registers; a choice is a
// local maximum, log2 L shuffles and the removal of the winner.  Rows of up to 64
// logits (L <= 4) pass through shared memory, since a lane's own loads would touch
// one 32-byte sector for every few values of a 4 E-byte row; wider rows are loaded
// directly, 4 L consecutive bytes a row and instruction.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>

#include "mixture.h"

namespace mb {

namespace {

constexpr int kWarps = 4;               // warps a block
constexpr int kStaged = 64;             // widest row that passes through shared memory
constexpr int kTile = 544;              // floats of a warp's tile: 32 x 17, 16 x 33 or 8 x 65

__device__ __forceinline__ float not_nan(float v) { return v != v ? -INFINITY : v; }

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

template <int L, int V>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const RouteArgs a) {
  constexpr bool kThrough = L <= 4;
  constexpr int R = 32 / L;             // rows a warp
  __shared__ float tile[kThrough ? kWarps : 1][kThrough ? kTile : 1];
  // the choices, written out together: R * k <= 512 since k <= E <= 16 L and k <= 32
  __shared__ int s_id[kWarps][512];
  __shared__ float s_e[kWarps][512];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sub = lane % L, r = lane / L;
  const long long row0 = (long long)(blockIdx.x * (long long)kWarps + warp) * R;
  if (row0 >= a.rows) return;           // whole warps only: no block barrier below
  const int nr = int(a.rows - row0 < R ? a.rows - row0 : R);
  const int E = a.experts, k = a.k;
  float v[V];
  if (kThrough) {
    float* t = tile[warp];
    const int sp = E | 1;
    each_value(nr, E, lane, [&](int rr, int c) { t[rr * sp + c] = a.logits[(row0 + rr) * a.ld + c]; });
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * L + sub;
      v[i] = e < E && r < nr ? not_nan(t[r * sp + e]) : -INFINITY;
    }
  } else {
    const float* p = a.logits + (row0 + (r < nr ? r : 0)) * a.ld;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * L + sub;
      v[i] = e < E && r < nr ? not_nan(p[e]) : -INFINITY;
    }
  }
  float top = 0.f, total = 0.f;
  for (int j = 0; j < k; ++j) {
    float best = v[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < V; ++i)
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
        for (int i = 0; i < V; ++i) total += expf(v[i] - top);
#pragma unroll
        for (int o = L / 2; o > 0; o /= 2) total += __shfl_xor_sync(~0u, total, o);
      }
    }
    const float e = expf(best - top);   // 0 for -inf
    if (a.norm == kRouteChosen) total += e;
    if (sub == 0) {
      s_id[warp][r * k + j] = found ? id : -1;
      s_e[warp][r * k + j] = e;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * L + sub == id) v[i] = -INFINITY;
  }
  // the group's lanes divide their row's choices by the same total
  __syncwarp();
  const float over = total > 0.f || total != total ? total : 1.f;
  for (int j = sub; j < k; j += L) s_e[warp][r * k + j] = s_e[warp][r * k + j] / over;
  __syncwarp();
  for (int i = lane; i < nr * k; i += 32) {
    a.ids[row0 * k + i] = s_id[warp][i];
    a.weights[row0 * k + i] = s_e[warp][i];
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

// Rows of up to 64 logits: 32 rows a warp when E <= 16, 16 or 8 above, one lane a row,
// through the warp's tile.
__global__ void __launch_bounds__(kWarps * 32) route_grad_narrow_kernel(const RouteArgs a) {
  __shared__ float tile[kWarps][kTile];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int E = a.experts, k = a.k, sp = E | 1;
  const int R = E <= 16 ? 32 : E <= 32 ? 16 : 8;
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
    for (int j = 0; j < k; ++j) {
      int id;
      float w, dw;
      choice(a, row, j, &id, &w, &dw);
      if (j == 0) {
        id0 = id;
        w0 = w;
      }
      mean += w * dw;
    }
    if (a.norm == kRouteAll && id0 >= 0) {
      const float l0 = mine[id0];
      for (int e = 0; e < E; ++e) mine[e] = -mean * (w0 * expf(not_nan(mine[e]) - l0));
    } else {
      for (int e = 0; e < E; ++e) mine[e] = 0.f;
    }
    for (int j = 0; j < k; ++j) {
      int id;
      float w, dw;
      choice(a, row, j, &id, &w, &dw);
      if (id >= 0) mine[id] = w * (dw - mean);
    }
  }
  __syncwarp();
  each_value(nr, E, lane, [&](int r, int c) { a.dlogits[(row0 + r) * a.ld_d + c] = t[r * sp + c]; });
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
        q.x = scale * expf(not_nan(q.x) - l0);
        q.y = scale * expf(not_nan(q.y) - l0);
        q.z = scale * expf(not_nan(q.z) - l0);
        q.w = scale * expf(not_nan(q.w) - l0);
      }
      *reinterpret_cast<float4*>(d + e) = q;
    }
  } else {
    for (int e = lane; e < E; e += 32) d[e] = all ? scale * expf(not_nan(l[e]) - l0) : 0.f;
  }
  __syncwarp();  // the warp's own stores before the choices' values replace some of them
  if (id >= 0) d[id] = w * (dw - mean);
}

template <int L, int V>
cudaError_t go(const RouteArgs& a, cudaStream_t s) {
  const long long per = (long long)kWarps * (32 / L);
  const long long blocks = (a.rows + per - 1) / per;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  route_kernel<L, V><<<unsigned(blocks), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_route(const RouteArgs& a, cudaStream_t s) {
  const int E = a.experts;
  if (E <= 4) return go<1, 4>(a, s);
  if (E <= 8) return go<1, 8>(a, s);
  if (E <= 16) return go<1, 16>(a, s);
  if (E <= 32) return go<2, 16>(a, s);
  if (E <= 64) return go<4, 16>(a, s);
  if (E <= 128) return go<8, 16>(a, s);
  if (E <= 256) return go<16, 16>(a, s);
  if (E <= 512) return go<32, 16>(a, s);
  return go<32, 32>(a, s);
}

cudaError_t launch_route_grad(const RouteArgs& a, cudaStream_t s) {
  const int E = a.experts;
  const long long per = E > kStaged ? kWarps : kWarps * (E <= 16 ? 32 : E <= 32 ? 16 : 8);
  const long long blocks = (a.rows + per - 1) / per;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  const auto bits = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits);
  const bool vec = bits % 16 == 0 && (a.ld | a.ld_d | E) % 4 == 0;
  if (E <= kStaged)
    route_grad_narrow_kernel<<<unsigned(blocks), kWarps * 32, 0, s>>>(a);
  else if (vec)
    route_grad_kernel<true><<<unsigned(blocks), kWarps * 32, 0, s>>>(a);
  else
    route_grad_kernel<false><<<unsigned(blocks), kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mb
