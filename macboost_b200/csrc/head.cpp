// Host side of the softmax head (head.h): argument checks, the plan of pieces and
// splits, tensor maps and launches.
#include "head.h"

#include <algorithm>
#include <cstdlib>

#include "engine.h"
#include "kernels.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int64_t kMaxIndex = 2147483647;
// The gradient's g of one piece of the classes: large enough that the pieces' products
// fill the GPU several times over, far below the logits of a large head.
constexpr int64_t kPieceBytes = int64_t(256) << 20;
// Tile rows walked together keep about this much of A in the L2 cache (126 MB).
constexpr int64_t kGroupBytes = int64_t(32) << 20;

int fail(std::string& err, const std::string& msg) {
  err = msg;
  return -1;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t parts(int64_t v, int64_t m) { return (v + m - 1) / m; }

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

// ---- the plan -------------------------------------------------------------------

struct Plan {
  int planes;
  bool pack_h, pack_w;
  int64_t ldp;                        // stride of packed rows
  int64_t piece, pieces, ld_g;        // classes a piece, pieces, stride of g
  int tile_n;                         // columns of the gradients' tiles
  int dh_splits, dw_splits;
  // offsets into the workspace
  int64_t status = 0, h = 0, w = 0, part = 0, target = 0, g = 0, acc = 0, dh_part = 0, dw_part = 0;
  int64_t bytes = 0;
};

// TMA reads rows in place when they start on 16 bytes.
bool in_place(int dtype, const void* p, int64_t ld) {
  return dtype == kBF16 && aligned(p, 16) && ld % 8 == 0;
}

// Parts of K of a product whose tiles walk `kblocks`: none longer than what each pair of
// CTAs gets of `all` steps in total, so that they end together, and none shorter than 8
// blocks (float32: 2, of six products), so that the sums of parts stay few.  bfloat16 sums
// stay in the tensor core, which truncates them at each step of 16: a sum whose terms have one
// sign lost 1e-7 of itself a step (dw of 300,000 rows, 0.18%).  So its parts are 512 blocks
// (2,048 steps, 2^-12) at most, and the parts are added up in float32.
int splits_for(int64_t kblocks, int64_t all, int dtype) {
  const int64_t least = dtype == kF32 ? 2 : 8, steps = dtype == kF32 ? 6 : 1;
  const int64_t most = std::max(least, (all / 74 - kHeadEpilogue) / steps);
  const int64_t load = std::min<int64_t>(std::min(parts(kblocks, most), kblocks / least), 100);
  return int(std::max<int64_t>({1, load, dtype == kF32 ? 1 : parts(kblocks, 512)}));
}

Plan make_plan(int dtype, int64_t rows, int64_t cols, int64_t classes, bool grad, bool pack_h,
               bool pack_w, bool want_dh, bool want_dw) {
  Plan p{};
  p.planes = dtype == kF32 ? 3 : 1;
  p.pack_h = pack_h || grad;  // the gradient's copy has zeros in rows without a label
  p.pack_w = pack_w;
  p.ldp = up(cols, 8);
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  if (p.pack_h) p.h = take(p.planes * rows * p.ldp * 2);
  if (p.pack_w) p.w = take(p.planes * classes * p.ldp * 2);
  if (!grad) {
    p.part = take(2 * parts(classes, kHeadTileN) * rows * 8);
    p.target = take(rows * 4);
  } else {
    p.tile_n = cols <= 128 ? 128 : 256;
    p.piece = std::max<int64_t>(kHeadTileN, kPieceBytes / (p.planes * rows * 2) / kHeadTileN * kHeadTileN);
    p.piece = std::min(p.piece, up(classes, kHeadTileK));
    p.pieces = parts(classes, p.piece);
    p.ld_g = p.piece;
    p.g = take(p.planes * rows * p.ld_g * 2);
    const int64_t tm = kHeadPair * kHeadTileM, tn = parts(cols, p.tile_n);
    const int64_t dh_tiles = want_dh ? parts(rows, tm) * tn : 0;
    const int64_t dw_tiles = want_dw ? parts(p.piece, tm) * tn : 0;
    const int64_t dh_blocks = parts(p.piece, kHeadTileK), dw_blocks = parts(rows, kHeadTileK);
    const int64_t steps = dtype == kF32 ? 6 : 1;
    const int64_t all = dh_tiles * (dh_blocks * steps + kHeadEpilogue) +
                        dw_tiles * (dw_blocks * steps + kHeadEpilogue);
    p.dh_splits = splits_for(dh_blocks, all, dtype);
    p.dw_splits = splits_for(dw_blocks, all, dtype);
    if (want_dh && p.pieces > 1) p.acc = take(rows * cols * 4);
    if (want_dh && p.dh_splits > 1) p.dh_part = take(p.dh_splits * rows * cols * 4);
    if (want_dw && p.dw_splits > 1) p.dw_part = take(p.dw_splits * p.piece * cols * 4);
  }
  p.bytes = at;
  return p;
}

bool is_narrow(int64_t cols, int64_t classes) {
  return cols <= kNarrowCols && classes <= kNarrowClasses;
}
// Its workspace: the status word, and a dw of each block.
int64_t narrow_bytes(int64_t rows, int64_t cols, int64_t classes, bool grad) {
  return 256 + (grad ? up(narrow_blocks(rows) * cols * classes * 4, 256) : 0);
}

int few_padded(int64_t rows) {
  int n = 1;
  while (n < rows) n *= 2;
  return n;
}
bool is_few(int dtype, int64_t rows, int64_t cols) {
  return rows <= (dtype == kF32 ? 16 : 4) && few_padded(rows) * int64_t(few_pitch(cols)) * 4 <= kFewSmem;
}
// Blocks of the first kernel (two a multiprocessor) and parts of the classes for dh (as
// many as give every multiprocessor a few blocks); 148 multiprocessors whatever the GPU
// has, since a workspace is sized before a device is named.
struct FewPlan {
  HeadFew f{};
  int64_t part, target, g, dh_part, bytes;
};
FewPlan few_plan(int dtype, int64_t rows, int64_t cols, int64_t classes, bool grad) {
  FewPlan p{};
  const int64_t nr = few_padded(rows), c = nr <= 4 ? 8 : 32 / nr;
  p.f.blocks = int(std::min<int64_t>(296, parts(classes, 8 * c)));
  const int64_t columns = parts(cols, dtype == kF32 ? 1024 : 2048);
  p.f.chunks = int(std::max<int64_t>(1, std::min<int64_t>(592 / columns, classes / 64)));
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.part = take(grad ? 0 : p.f.blocks * rows * 8);
  p.target = take(grad ? 0 : rows * 4);
  p.g = take(grad ? classes * nr * 4 : 0);
  p.dh_part = take(grad ? p.f.chunks * rows * cols * 4 : 0);
  p.bytes = at;
  return p;
}

// ---- tensor maps ----------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A matrix of planes x outer x inner 16-bit values, stride ld, fetched in boxes of 64
// inner x `box` outer values into 128-byte swizzled rows; zeros outside.
int encode(CUtensorMap* m, const void* p, int64_t inner, int64_t outer, int64_t ld, int planes,
           int box, std::string& err) {
  EncodeFn fn = encode_fn();
  if (!fn) return fail(err, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * cuuint64_t(outer) * 2};
  const cuuint32_t boxes[3] = {64, cuuint32_t(box), 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides,
                        boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(err, "cuTensorMapEncodeTiled failed with " + std::to_string(int(r)));
  return 0;
}

// Rows of a K-major box: all of a tile's, or the matrix's when it has fewer (in groups
// of 8, a swizzle atom).
int box_rows(int64_t rows, int tile) { return int(std::min<int64_t>(tile, up(rows, 8))); }

// ---- checks ---------------------------------------------------------------------

int check_shape(int dtype, int64_t rows, int64_t cols, int64_t classes, std::string& err) {
  if (dtype != kF32 && dtype != kBF16)
    return fail(err, "the head takes dtype 0 (float32) or 1 (bfloat16), got " + std::to_string(dtype));
  if (rows < 0 || rows > (int64_t(1) << 30)) return fail(err, "rows must be in 0...2^30");
  if (cols < 1 || cols > (int64_t(1) << 20)) return fail(err, "cols must be in 1...2^20");
  if (classes < 1 || classes > (int64_t(1) << 30)) return fail(err, "classes must be in 1...2^30");
  return 0;
}

int check_matrix(const char* name, const void* p, int64_t cols, int64_t ld, int dtype, std::string& err) {
  if (!p) return fail(err, "null argument");
  if (ld < cols) return fail(err, std::string(name) + " needs ld >= cols");
  if (!aligned(p, size_t(dtype_bytes(dtype))))
    return fail(err, std::string(name) + " must be aligned to its values");
  return 0;
}

int check(const HeadArgs& a, bool grad, std::string& err) {
  if (check_shape(a.dtype, a.rows, a.cols, a.classes, err)) return -1;
  // without rows only dw (all zeros) is left to write
  if (a.rows == 0 && !(grad && a.dw)) return 0;
  if (a.rows > 0 && (check_matrix("h", a.h, a.cols, a.ld_h, a.dtype, err) ||
                     check_matrix("w", a.w, a.cols, a.ld_w, a.dtype, err)))
    return -1;
  if (a.rows > 0 && (!a.labels || (grad ? !a.lse || !a.dloss : !a.loss || !a.lse_out)))
    return fail(err, "null argument");
  for (const void* p : {static_cast<const void*>(a.labels), static_cast<const void*>(a.loss),
                        static_cast<const void*>(a.lse_out), static_cast<const void*>(a.lse),
                        static_cast<const void*>(a.dloss)})
    if (!aligned(p, 4)) return fail(err, "labels, loss, lse and dloss must be 4-byte aligned");
  if (grad) {
    if (a.dh && check_matrix("dh", a.dh, a.cols, a.ld_dh, a.dtype, err)) return -1;
    if (a.dw && check_matrix("dw", a.dw, a.cols, a.ld_dw, a.dtype, err)) return -1;
  }
  if (!aligned(a.workspace, 256)) return fail(err, "workspace must be 256-byte aligned");
  return 0;
}

int check_workspace(const HeadArgs& a, int64_t need, std::string& err) {
  if (a.workspace && a.workspace_bytes >= need) return 0;
  return fail(err, "workspace holds " + std::to_string(a.workspace ? a.workspace_bytes : 0) +
                       " bytes, the head needs " + std::to_string(need));
}

#define HEAD_CUDA(call, what)                                                     \
  do {                                                                            \
    const cudaError_t e_ = (call);                                                \
    if (e_ != cudaSuccess) {                                                      \
      cudaGetLastError();                                                         \
      return fail(err, std::string(what) + ": " + cudaGetErrorString(e_));        \
    }                                                                             \
  } while (0)

struct Operands {
  const void *h, *w;
  int64_t ld_h, ld_w, launches;
};

// Operands packed where the plan says so, in one launch; the loss clears the status word.
int operands(const HeadArgs& a, const Plan& p, bool grad, Operands* o, cudaStream_t s, std::string& err) {
  char* base = static_cast<char*>(a.workspace);
  o->h = a.h;
  o->ld_h = a.ld_h;
  o->w = a.w;
  o->ld_w = a.ld_w;
  HeadPack h, w;
  if (p.pack_h) {
    h.src = a.h;
    h.rows = a.rows;
    h.cols = a.cols;
    h.ld = a.ld_h;
    h.labels = grad ? a.labels : nullptr;
    h.classes = a.classes;
    h.dst = base + p.h;
    h.ldp = p.ldp;
    o->h = h.dst;
    o->ld_h = p.ldp;
  }
  if (p.pack_w) {
    w.src = a.w;
    w.rows = a.classes;
    w.cols = a.cols;
    w.ld = a.ld_w;
    w.dst = base + p.w;
    w.ldp = p.ldp;
    o->w = w.dst;
    o->ld_w = p.ldp;
  }
  if (!p.pack_h && !p.pack_w) {
    HEAD_CUDA(cudaMemsetAsync(base, 0, 4, s), "clearing the head's status word");
    return 0;
  }
  unsigned* status = grad ? nullptr : reinterpret_cast<unsigned*>(base);
  HEAD_CUDA(launch_head_pack(a.dtype, h, w, status, s), "head pack launch");
  o->launches = 1;
  return 0;
}

void settings(HeadLaunch& l, const HeadArgs& a) {
  l.f32 = a.dtype == kF32;
  l.status = static_cast<unsigned*>(a.workspace);
  l.wait_ns = kDefaultWaitNs;
  if (const char* s = std::getenv("MACBOOST_WAIT_LIMIT_US")) {
    char* end = nullptr;
    const long long us = std::strtoll(s, &end, 10);
    if (end != s && us > 0 && us <= 60000000ll) l.wait_ns = static_cast<unsigned long long>(us) * 1000ull;
  }
  const char* t = std::getenv("MACBOOST_TEST_STALL_TILES");
  l.stall = t && t[0] == '1';
}

// The inputs themselves, for float32 logits that the planes cannot form.
void inputs(HeadRows& r, const HeadArgs& a) {
  if (a.dtype != kF32) return;
  r.h = static_cast<const float*>(a.h);
  r.w = static_cast<const float*>(a.w);
  r.ld_h = a.ld_h;
  r.ld_w = a.ld_w;
  r.cols = int(a.cols);
}

// The logits of classes v0 ... v0 + n - 1: A = h, B = w, both along cols.
int logits_job(HeadJob& j, const HeadArgs& a, const Plan& p, const Operands& o, int64_t v0, int64_t n,
               std::string& err) {
  j.M = int(a.rows);
  j.N = int(n);
  j.a_box = box_rows(a.rows, kHeadTileM);
  j.b_box = box_rows(n, kHeadTileN / kHeadPair);
  if (encode(&j.a, o.h, a.cols, a.rows, o.ld_h, p.planes, j.a_box, err) ||
      encode(&j.b, o.w, a.cols, a.classes, o.ld_w, p.planes, j.b_box, err))
    return -1;
  if (parts(a.rows, kHeadPair * kHeadTileM) * parts(n, kHeadTileN) > kMaxIndex)
    return fail(err, "rows * classes are too many for one call");
  j.tiles_m = int(parts(a.rows, kHeadPair * kHeadTileM));
  j.tiles_n = int(parts(n, kHeadTileN));
  j.splits = 1;
  j.kblocks = int(parts(a.cols, kHeadTileK));
  j.group = int(std::max<int64_t>(1, kGroupBytes / (kHeadPair * kHeadTileM * a.cols * 2 * p.planes)));
  j.group = std::min(j.group, j.tiles_m);
  j.b_row0 = int(v0);
  j.divide();
  return 0;
}

int narrow(int device, const HeadArgs& a, bool grad, cudaStream_t s, std::string& err) {
  if (check_workspace(a, narrow_bytes(a.rows, a.cols, a.classes, grad), err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  float* part = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + 256);
  HEAD_CUDA(launch_head_narrow(a, grad, part, narrow_blocks(a.rows), s), "narrow head launch");
  g_kernel_launches.fetch_add(grad && a.dw ? 2 : 1, std::memory_order_relaxed);
  return 0;
}

int few(int device, const HeadArgs& a, bool grad, cudaStream_t s, std::string& err) {
  FewPlan p = few_plan(a.dtype, a.rows, a.cols, a.classes, grad);
  if (check_workspace(a, p.bytes, err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  char* base = static_cast<char*>(a.workspace);
  p.f.part = reinterpret_cast<float2*>(base + p.part);
  p.f.target = reinterpret_cast<float*>(base + p.target);
  p.f.g = reinterpret_cast<float*>(base + p.g);
  p.f.dh_part = reinterpret_cast<float*>(base + p.dh_part);
  HEAD_CUDA(launch_head_few(a, grad, p.f, s), "head launch");
  if (!grad) {
    HEAD_CUDA(launch_head_finish(p.f.part, p.f.target, a.labels, a.rows, a.classes, p.f.blocks, a.loss,
                                 a.lse_out, s),
              "head finish launch");
    g_kernel_launches.fetch_add(2, std::memory_order_relaxed);
    return 0;
  }
  if (a.dh)
    HEAD_CUDA(launch_head_reduce(HeadReduce{p.f.dh_part, p.f.chunks, a.rows, a.cols, nullptr, 0, 1, a.dh,
                                            a.ld_dh, a.dtype == kF32},
                                 s),
              "head reduce launch");
  g_kernel_launches.fetch_add(a.dh ? 3 : 1, std::memory_order_relaxed);
  return 0;
}

}  // namespace

int64_t head_workspace(int dtype, int64_t rows, int64_t cols, int64_t classes, bool grad, bool strided) {
  std::string err;
  if (check_shape(dtype, rows, cols, classes, err)) return -1;
  if (is_narrow(cols, classes)) return narrow_bytes(rows, cols, classes, grad);
  if (is_few(dtype, rows, cols)) {
    const int64_t loss = few_plan(dtype, rows, cols, classes, false).bytes;
    return grad ? std::max(loss, few_plan(dtype, rows, cols, classes, true).bytes) : loss;
  }
  const bool pack = dtype == kF32 || strided || cols % 8 != 0;
  const int64_t loss = make_plan(dtype, rows, cols, classes, false, pack, pack, true, true).bytes;
  if (!grad) return loss;
  // a gradient alone can split K further than both together
  int64_t most = loss;
  for (int m = 1; m < 4; ++m)
    most = std::max(most, make_plan(dtype, std::max<int64_t>(rows, 1), cols, classes, true, pack, pack,
                                    m & 1, m & 2).bytes);
  return most;
}

int head_loss_device(int device, const HeadArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, false, err)) return -1;
  if (a.rows == 0) return 0;
  if (is_narrow(a.cols, a.classes)) return narrow(device, a, false, s, err);
  if (is_few(a.dtype, a.rows, a.cols)) return few(device, a, false, s, err);
  const Plan p = make_plan(a.dtype, a.rows, a.cols, a.classes, false, !in_place(a.dtype, a.h, a.ld_h),
                           !in_place(a.dtype, a.w, a.ld_w), true, true);
  if (check_workspace(a, p.bytes, err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  char* base = static_cast<char*>(a.workspace);
  Operands o{};
  if (operands(a, p, false, &o, s, err)) return -1;
  HeadLaunch l{};
  settings(l, a);
  l.jobs = 1;
  if (logits_job(l.job[0], a, p, o, 0, a.classes, err)) return -1;
  l.r.labels = a.labels;
  l.r.part = reinterpret_cast<float2*>(base + p.part);
  l.r.target = reinterpret_cast<float*>(base + p.target);
  l.r.rows = int(a.rows);
  l.r.classes = int(a.classes);
  inputs(l.r, a);
  HEAD_CUDA(launch_head(kHeadLse, kHeadTileN, l, s), "head launch");
  HEAD_CUDA(launch_head_finish(l.r.part, l.r.target, a.labels, a.rows, a.classes,
                               2 * l.job[0].tiles_n, a.loss, a.lse_out, s),
            "head finish launch");
  g_kernel_launches.fetch_add(o.launches + 2, std::memory_order_relaxed);
  return 0;
}

int head_grad_device(int device, const HeadArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, true, err)) return -1;
  if (!a.dh && !a.dw) return 0;
  if (a.rows == 0) {
    if (!a.dw) return 0;
    if (check_matrix("dw", a.dw, a.cols, a.ld_dw, a.dtype, err)) return -1;
    if (use_device(device, err)) return -1;
    Guard gd(device);
    const size_t size = size_t(dtype_bytes(a.dtype));
    HEAD_CUDA(cudaMemset2DAsync(a.dw, size_t(a.ld_dw) * size, 0, size_t(a.cols) * size,
                                size_t(a.classes), s),
              "clearing dw");
    return 0;
  }
  if (is_narrow(a.cols, a.classes)) return narrow(device, a, true, s, err);
  if (is_few(a.dtype, a.rows, a.cols)) return few(device, a, true, s, err);
  const Plan p = make_plan(a.dtype, a.rows, a.cols, a.classes, true, !in_place(a.dtype, a.h, a.ld_h),
                           !in_place(a.dtype, a.w, a.ld_w), a.dh != nullptr, a.dw != nullptr);
  if (check_workspace(a, p.bytes, err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  char* base = static_cast<char*>(a.workspace);
  Operands o{};
  if (operands(a, p, true, &o, s, err)) return -1;
  int64_t launches = o.launches;
  const bool f32 = a.dtype == kF32;
  const int64_t tm = kHeadPair * kHeadTileM;
  auto four = [&](const void* q, int64_t ld) {
    return int(aligned(q, size_t(4 * dtype_bytes(a.dtype))) && ld % 4 == 0);
  };
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(p.piece, a.classes - v0);
    HeadLaunch l{};
    settings(l, a);
    l.jobs = 1;
    if (logits_job(l.job[0], a, p, o, v0, n, err)) return -1;
    l.r.labels = a.labels;
    l.r.lse = a.lse;
    l.r.dloss = a.dloss;
    l.r.g = base + p.g;
    l.r.ld_g = p.ld_g;
    l.r.plane_g = a.rows * p.ld_g;
    l.r.rows = int(a.rows);
    l.r.classes = int(a.classes);
    l.r.v0 = int(v0);
    inputs(l.r, a);
    HEAD_CUDA(launch_head(kHeadG, kHeadTileN, l, s), "head launch");

    HeadLaunch q{};
    settings(q, a);
    HeadReduce red[2]{};
    int reds = 0;
    HeadJob dh{}, dw{};
    if (a.dh) {  // dh = g w: A = g along its classes, B = w's columns
      dh.a_box = box_rows(a.rows, kHeadTileM);
      if (encode(&dh.a, base + p.g, n, a.rows, p.ld_g, p.planes, dh.a_box, err) ||
          encode(&dh.b, o.w, a.cols, a.classes, o.ld_w, p.planes, 64, err))
        return -1;
      dh.b_mn = 1;
      dh.tiles_m = int(parts(a.rows, tm));
      dh.tiles_n = int(parts(a.cols, p.tile_n));
      dh.kblocks = int(parts(n, kHeadTileK));
      dh.splits = std::min(p.dh_splits, dh.kblocks);
      dh.b_k0 = int(v0);
      dh.M = int(a.rows);
      dh.N = int(a.cols);
      dh.out = a.dh;
      dh.ld_out = a.ld_dh;
      dh.out_f32 = f32;
      dh.wide = four(a.dh, a.ld_dh);
      float* acc = p.pieces > 1 ? reinterpret_cast<float*>(base + p.acc) : nullptr;
      const int in = i > 0, last = i + 1 == p.pieces;
      if (dh.splits > 1) {
        dh.acc = reinterpret_cast<float*>(base + p.dh_part);
        red[reds++] = HeadReduce{dh.acc, dh.splits, a.rows, a.cols, acc, in, last, a.dh, a.ld_dh, f32};
      } else {
        dh.acc = acc;
        dh.acc_in = in;
        dh.final = last;
      }
    }
    if (a.dw) {  // dw = g^T h: A = g's columns, B = h's columns, along the rows
      if (encode(&dw.a, base + p.g, n, a.rows, p.ld_g, p.planes, 64, err) ||
          encode(&dw.b, o.h, a.cols, a.rows, o.ld_h, p.planes, 64, err))
        return -1;
      dw.a_mn = dw.b_mn = 1;
      dw.tiles_m = int(parts(n, tm));
      dw.tiles_n = int(parts(a.cols, p.tile_n));
      dw.kblocks = int(parts(a.rows, kHeadTileK));
      dw.splits = std::min(p.dw_splits, dw.kblocks);
      dw.M = int(n);
      dw.N = int(a.cols);
      dw.out = static_cast<char*>(a.dw) + v0 * a.ld_dw * dtype_bytes(a.dtype);
      dw.ld_out = a.ld_dw;
      dw.out_f32 = f32;
      dw.wide = four(dw.out, a.ld_dw);
      dw.final = 1;
      if (dw.splits > 1) {
        dw.acc = reinterpret_cast<float*>(base + p.dw_part);
        dw.final = 0;
        red[reds++] = HeadReduce{dw.acc, dw.splits, n, a.cols, nullptr, 0, 1, dw.out, a.ld_dw, f32};
      }
    }
    for (HeadJob* j : {&dh, &dw})
      if (j->tiles_m > 0) {
        j->group = std::min(16, j->tiles_m);
        j->divide();
      }
    // the heavier tiles first
    const bool dw_first = !a.dh || (a.dw && dw.kblocks / dw.splits > dh.kblocks / dh.splits);
    if (a.dh && a.dw) {
      q.jobs = 2;
      q.job[0] = dw_first ? dw : dh;
      q.job[1] = dw_first ? dh : dw;
    } else {
      q.jobs = 1;
      q.job[0] = a.dh ? dh : dw;
    }
    HEAD_CUDA(launch_head(kHeadOut, p.tile_n, q, s), "head launch");
    for (int r = 0; r < reds; ++r) HEAD_CUDA(launch_head_reduce(red[r], s), "head reduce launch");
    launches += 2 + reds;
  }
  g_kernel_launches.fetch_add(launches, std::memory_order_relaxed);
  return 0;
}

int head_check_device(int device, const void* workspace, std::string& err) {
  if (!workspace) return fail(err, "null argument");
  if (use_device(device, err)) return -1;
  Guard gd(device);
  HEAD_CUDA(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
  unsigned word = 0;
  HEAD_CUDA(cudaMemcpy(&word, workspace, 4, cudaMemcpyDeviceToHost), "reading the head's status word");
  if (word == kHeadExpired)
    return fail(err, "device " + std::to_string(device) +
                         ": head kernel gave up waiting for a shared-memory transfer");
  return 0;
}

}  // namespace mb
