// Rows routed among several models: the choice of models from gate logits, rows
// sorted by model and gathered into each model's segment, the models' outputs
// combined, and the gradients of each step.  Everything works on device memory,
// enqueued on the caller's stream, and allocates nothing.
//
// N rows choose k of E models each ("entries", numbered n * k + j).  The sorted
// plan gives every entry a slot: segment e is offsets[e] .. offsets[e] +
// counts[e] - 1, its entries ascending, and starts at a multiple of `align`.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace mb {

constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;       // MACBOOST_F32 ...
constexpr int kRouteChosen = 0, kRouteAll = 1;     // MACBOOST_ROUTE_*
constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 32;

// Bytes of a value of `dtype`, 0 for an unknown code.
inline int dtype_bytes(int dtype) { return dtype == kF32 ? 4 : dtype == kBF16 || dtype == kF16 ? 2 : 0; }

// The device exists and is an sm_100a GPU (cached per device after the first
// success, so that a call of a few microseconds does not ask the driver again).
int use_device(int device, std::string& err);
// Multiprocessors of the current device, cached.
int device_sms();

struct RouteArgs {
  const float* logits;
  long long rows, ld;
  int experts, k, norm;
  int* ids;              // rows x k
  float* weights;        // rows x k
  const float* dweights; // gradient: rows x k
  float* dlogits;        // gradient: rows x ld_d
  long long ld_d;
};
cudaError_t launch_route(const RouteArgs& a, cudaStream_t s);
cudaError_t launch_route_grad(const RouteArgs& a, cudaStream_t s);

struct SortArgs {
  const int* ids;
  long long entries;     // rows * k, < 2^31
  long long capacity;    // entries + experts * (align - 1), < 2^31
  int experts, align;
  long long* offsets;
  int *counts, *order, *slots;
  int* tile_counts;      // workspace: experts x tiles
};
// The ints of the workspace of a sort of `entries`; 0 for one that is a single launch.
long long sort_workspace_ints(long long entries, int experts);
cudaError_t launch_sort(const SortArgs& a, int* launches, cudaStream_t s);

struct GatherArgs {
  const void* x;
  long long rows, cols, ld;
  int layout;            // 0 feature-major, 1 row-major
  int k, experts;
  const long long* offsets;
  const int *order, *slots;
  long long capacity;
  void* out;
  long long ld_out;
  int layout_out;
  int dtype;
};
cudaError_t launch_gather(const GatherArgs& a, cudaStream_t s);

struct CombineArgs {
  const void* y;
  long long capacity, cols, ld;
  const int* order;      // gradient only
  const int* slots;
  const float* weights;  // null: ones
  long long rows;
  int k;
  void* out;             // forward
  long long ld_out;
  const void* dout;      // gradient
  long long ld_dout;
  void* dy;
  long long ld_dy;
  float* dweights;       // null: not wanted
  int dtype;
};
cudaError_t launch_combine(const CombineArgs& a, cudaStream_t s);
cudaError_t launch_combine_grad(const CombineArgs& a, cudaStream_t s);

// The calls behind the C entry points: arguments checked, errors as messages.
int route_device(int device, const RouteArgs& a, cudaStream_t s, std::string& err);
int route_grad_device(int device, const RouteArgs& a, cudaStream_t s, std::string& err);
int64_t sort_rows_workspace(int64_t rows, int64_t k, int64_t experts);
int sort_rows_device(int device, const int32_t* ids, int64_t rows, int64_t k, int64_t experts,
                     int64_t align, int64_t* offsets, int32_t* counts, int32_t* order,
                     int32_t* slots, void* workspace, int64_t workspace_bytes, cudaStream_t s,
                     std::string& err);
int gather_rows_device(int device, const GatherArgs& a, cudaStream_t s, std::string& err);
int combine_rows_device(int device, const CombineArgs& a, cudaStream_t s, std::string& err);
int combine_rows_grad_device(int device, const CombineArgs& a, cudaStream_t s, std::string& err);

}  // namespace mb
