// Host side of the mixture operators (mixture.h): argument checks and launches.
#include "mixture.h"

#include <algorithm>
#include <atomic>

#include "engine.h"

namespace mb {

namespace {

constexpr int kMaxDevices = 64;
std::atomic<int> g_sms[kMaxDevices];  // 0: not yet checked

struct Guard {
  int prev = -1, want;
  explicit Guard(int d) : want(d) {
    cudaGetDevice(&prev);
    if (prev != d) cudaSetDevice(d);
  }
  ~Guard() {
    if (prev >= 0 && prev != want) cudaSetDevice(prev);
  }
};

int fail(std::string& err, const std::string& msg) {
  err = msg;
  return -1;
}

int launched(cudaError_t e, const char* what, int n, std::string& err) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, std::string(what) + " launch: " + cudaGetErrorString(e));
  }
  g_kernel_launches.fetch_add(n, std::memory_order_relaxed);
  return 0;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

constexpr int64_t kMaxIndex = 2147483647;

int check_choices(int64_t rows, int64_t k, int64_t experts, std::string& err) {
  if (rows < 0) return fail(err, "rows must be >= 0");
  if (experts < 1 || experts > kMaxExperts)
    return fail(err, "experts must be in 1..." + std::to_string(kMaxExperts) + ", got " +
                         std::to_string(experts));
  if (k < 1 || k > kMaxChoices || k > experts)
    return fail(err, "k must be in 1...min(experts, " + std::to_string(kMaxChoices) + "), got " +
                         std::to_string(k));
  if (rows > kMaxIndex / k)
    return fail(err, "rows * k must be below 2^31");
  return 0;
}

int check_dtype(int dtype, std::string& err) {
  if (!dtype_bytes(dtype))
    return fail(err, "unknown dtype " + std::to_string(dtype) + " (0 float32, 1 bfloat16, 2 float16)");
  return 0;
}

}  // namespace

int use_device(int device, std::string& err) {
  if (device >= 0 && device < kMaxDevices && g_sms[device].load(std::memory_order_relaxed) > 0)
    return 0;
  int n = 0;
  const cudaError_t ce = cudaGetDeviceCount(&n);
  if (ce != cudaSuccess || n == 0) {
    cudaGetLastError();
    return fail(err, ce != cudaSuccess
                         ? std::string("no CUDA device available: ") + cudaGetErrorString(ce)
                         : std::string("no CUDA device available"));
  }
  if (device < 0 || device >= std::min(n, kMaxDevices))
    return fail(err, "device " + std::to_string(device) + " does not exist (" + std::to_string(n) +
                         " visible)");
  int major = 0, sms = 0;
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (major != 10 || sms < 1)
    return fail(err, "device " + std::to_string(device) + " is not an sm_100a (B200) GPU");
  g_sms[device].store(sms, std::memory_order_relaxed);
  return 0;
}

int device_sms() {
  int d = 0;
  cudaGetDevice(&d);
  const int n = d >= 0 && d < kMaxDevices ? g_sms[d].load(std::memory_order_relaxed) : 0;
  return n > 0 ? n : 148;
}

static int check_route(const RouteArgs& a, std::string& err) {
  if (check_choices(a.rows, a.k, a.experts, err)) return -1;
  if (a.ld < a.experts) return fail(err, "logits need ld >= experts");
  if (a.norm != kRouteChosen && a.norm != kRouteAll)
    return fail(err, "norm must be 0 (over the chosen) or 1 (over all)");
  if (a.rows > 0 && (!a.logits || !a.ids || !a.weights)) return fail(err, "null argument");
  if (!aligned(a.logits, 4) || !aligned(a.ids, 4) || !aligned(a.weights, 4))
    return fail(err, "logits, ids and weights must be 4-byte aligned");
  return 0;
}

int route_device(int device, const RouteArgs& a, cudaStream_t s, std::string& err) {
  if (check_route(a, err)) return -1;
  if (a.rows == 0) return 0;
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_route(a, s), "route", 1, err);
}

int route_grad_device(int device, const RouteArgs& a, cudaStream_t s, std::string& err) {
  if (check_route(a, err)) return -1;
  if (a.ld_d < a.experts) return fail(err, "dlogits need ld >= experts");
  if (a.rows > 0 && (!a.dweights || !a.dlogits)) return fail(err, "null argument");
  if (!aligned(a.dweights, 4) || !aligned(a.dlogits, 4))
    return fail(err, "dweights and dlogits must be 4-byte aligned");
  if (a.rows == 0) return 0;
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_route_grad(a, s), "route gradient", 1, err);
}

int64_t sort_rows_workspace(int64_t rows, int64_t k, int64_t experts) {
  std::string err;
  if (check_choices(rows, k, experts, err)) return -1;
  return 4 * sort_workspace_ints(rows * k, int(experts));
}

int sort_rows_device(int device, const int32_t* ids, int64_t rows, int64_t k, int64_t experts,
                     int64_t align, int64_t* offsets, int32_t* counts, int32_t* order,
                     int32_t* slots, void* workspace, int64_t workspace_bytes, cudaStream_t s,
                     std::string& err) {
  if (check_choices(rows, k, experts, err)) return -1;
  if (align < 1 || align > 1024) return fail(err, "align must be in 1...1024");
  SortArgs a{};
  a.ids = ids;
  a.entries = rows * k;
  a.capacity = a.entries + experts * (align - 1);
  if (a.capacity > kMaxIndex) return fail(err, "rows * k + experts * (align - 1) must be below 2^31");
  if (!offsets || !counts || (a.entries > 0 && (!ids || !slots)) || (a.capacity > 0 && !order))
    return fail(err, "null argument");
  if (!aligned(ids, 4) || !aligned(counts, 4) || !aligned(order, 4) || !aligned(slots, 4) ||
      !aligned(offsets, 8) || !aligned(workspace, 4))
    return fail(err, "ids, counts, order, slots and workspace must be 4-byte aligned, offsets "
                     "8-byte aligned");
  const int64_t need = sort_rows_workspace(rows, k, experts);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(err, "workspace holds " + std::to_string(workspace ? workspace_bytes : 0) +
                         " bytes, the sort needs " + std::to_string(need));
  a.experts = int(experts);
  a.align = int(align);
  a.offsets = reinterpret_cast<long long*>(offsets);
  a.counts = counts;
  a.order = order;
  a.slots = slots;
  a.tile_counts = static_cast<int*>(workspace);
  if (use_device(device, err)) return -1;
  Guard g(device);
  int n = 0;
  const cudaError_t e = launch_sort(a, &n, s);
  return launched(e, "row sort", n, err);
}

// rows x cols values of `dtype` in `layout` at p with stride ld.
static int check_matrix(const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld,
                        int layout, int dtype, std::string& err) {
  if (ld < (layout == 0 ? rows : cols))
    return fail(err, std::string(name) + (layout == 0 ? " needs ld >= its rows" : " needs ld >= cols"));
  if (layout == 1 && ld > kMaxIndex / dtype_bytes(dtype))
    return fail(err, std::string(name) + " needs rows of less than 2^31 bytes");
  if (rows > 0 && !p) return fail(err, "null argument");
  if (!aligned(p, size_t(dtype_bytes(dtype))))
    return fail(err, std::string(name) + " must be aligned to its values");
  return 0;
}

int gather_rows_device(int device, const GatherArgs& a, cudaStream_t s, std::string& err) {
  if (check_choices(a.rows, a.k, a.experts, err) || check_dtype(a.dtype, err)) return -1;
  if (a.cols < 1) return fail(err, "cols must be >= 1");
  if ((a.layout != 0 && a.layout != 1) || (a.layout_out != 0 && a.layout_out != 1))
    return fail(err, "layout must be 0 (feature-major) or 1 (row-major)");
  if (a.capacity < a.rows * a.k || a.capacity > kMaxIndex)
    return fail(err, "capacity must be at least rows * k and below 2^31");
  if (check_matrix("x", a.x, a.rows, a.cols, a.ld, a.layout, a.dtype, err) ||
      check_matrix("out", a.out, a.capacity, a.cols, a.ld_out, a.layout_out, a.dtype, err))
    return -1;
  if (a.capacity == 0) return 0;
  if (!a.offsets || !a.order || (a.rows > 0 && !a.slots)) return fail(err, "null argument");
  if (!aligned(a.offsets, 8) || !aligned(a.order, 4) || !aligned(a.slots, 4))
    return fail(err, "offsets must be 8-byte aligned, order and slots 4-byte aligned");
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_gather(a, s), "row gather", 1, err);
}

static int check_combine(const CombineArgs& a, std::string& err) {
  if (check_dtype(a.dtype, err)) return -1;
  if (a.rows < 0) return fail(err, "rows must be >= 0");
  if (a.k < 1 || a.k > kMaxChoices)
    return fail(err, "k must be in 1..." + std::to_string(kMaxChoices) + ", got " + std::to_string(a.k));
  if (a.cols < 1) return fail(err, "cols must be >= 1");
  if (a.capacity < 0 || a.capacity > kMaxIndex || a.rows > kMaxIndex / a.k)
    return fail(err, "capacity and rows * k must be in 0...2^31 - 1");
  if (check_matrix("y", a.y, a.capacity, a.cols, a.ld, 1, a.dtype, err)) return -1;
  if (a.rows > 0 && !a.slots) return fail(err, "null argument");
  if (!aligned(a.slots, 4) || !aligned(a.weights, 4))
    return fail(err, "slots and weights must be 4-byte aligned");
  return 0;
}

int combine_rows_device(int device, const CombineArgs& a, cudaStream_t s, std::string& err) {
  if (check_combine(a, err) ||
      check_matrix("out", a.out, a.rows, a.cols, a.ld_out, 1, a.dtype, err))
    return -1;
  if (a.rows == 0) return 0;
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_combine(a, s), "combine", 1, err);
}

int combine_rows_grad_device(int device, const CombineArgs& a, cudaStream_t s, std::string& err) {
  if (check_combine(a, err) ||
      check_matrix("dout", a.dout, a.rows, a.cols, a.ld_dout, 1, a.dtype, err) ||
      check_matrix("dy", a.dy, a.capacity, a.cols, a.ld_dy, 1, a.dtype, err))
    return -1;
  if (a.capacity > 0 && !a.order) return fail(err, "null argument");
  if (!aligned(a.order, 4) || !aligned(a.dweights, 4))
    return fail(err, "order and dweights must be 4-byte aligned");
  if (a.rows == 0 && a.capacity == 0) return 0;
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_combine_grad(a, s), "combine gradient", 1, err);
}

}  // namespace mb
