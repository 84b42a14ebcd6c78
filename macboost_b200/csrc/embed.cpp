// Host side of the embeddings (embed.h): argument checks, the workspace and launches.
#include "embed.h"

#include <algorithm>

#include "engine.h"
#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int64_t kMaxIndex = 2147483647;

int fail(std::string& err, const std::string& msg) {
  err = msg;
  return -1;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

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

int launched(cudaError_t e, const char* what, int n, std::string& err) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, std::string(what) + " launch: " + cudaGetErrorString(e));
  }
  g_kernel_launches.fetch_add(n, std::memory_order_relaxed);
  return 0;
}

int check_shape(int64_t entries, int64_t cols, int64_t rows, int64_t k, std::string& err) {
  // one row more stands for what adds nothing
  if (entries < 1 || entries >= (int64_t(1) << 30)) return fail(err, "entries must be in 1...2^30 - 1");
  if (cols < 1 || cols > (int64_t(1) << 20)) return fail(err, "cols must be in 1...2^20");
  if (k < 1 || k > (int64_t(1) << 20)) return fail(err, "k must be in 1...2^20");
  if (rows < 0) return fail(err, "rows must be >= 0");
  if (rows > kMaxIndex / k) return fail(err, "rows * k must be below 2^31");
  return 0;
}

int check_matrix(const char* name, const void* p, int64_t cols, int64_t ld, int dtype, std::string& err) {
  if (ld < cols) return fail(err, std::string(name) + " needs ld >= cols");
  if (ld > kMaxIndex / dtype_bytes(dtype))
    return fail(err, std::string(name) + " needs rows of less than 2^31 bytes");
  if (!p) return fail(err, "null argument");
  if (!aligned(p, size_t(dtype_bytes(dtype))))
    return fail(err, std::string(name) + " must be aligned to its values");
  return 0;
}

int check(const EmbedArgs& a, bool grad, std::string& err) {
  if (!dtype_bytes(a.dtype))
    return fail(err, "unknown dtype " + std::to_string(a.dtype) + " (0 float32, 1 bfloat16, 2 float16)");
  if (check_shape(a.entries, a.cols, a.rows, a.k, err)) return -1;
  if (!aligned(a.ids, 4) || !aligned(a.starts, 4))
    return fail(err, "ids and starts must be 4-byte aligned");
  // without rows only a gradient (all zeros) is left to write
  if (a.rows > 0) {
    if (!a.ids) return fail(err, "null argument");
    if (check_matrix(grad ? "dout" : "out", grad ? a.dout : a.out, a.cols, a.ld_out, a.dtype, err)) return -1;
  }
  if (a.rows > 0 || grad)
    if (check_matrix(grad ? "dtable" : "table", grad ? a.dtable : a.table, a.cols, a.ld, a.dtype, err))
      return -1;
  return 0;
}

}  // namespace

EmbedPlan embed_plan(int64_t entries, int64_t cols, int64_t rows, int64_t k) {
  EmbedPlan p{};
  p.n = rows * k;
  int bits = 1;
  while ((int64_t(1) << bits) <= entries) ++bits;  // keys 0 ... entries
  // one block's sort takes as long as seven launches from some 5,000 entries on (8,192 of 32,000
  // x 512: 53 against 43 us; 4,096: 27 against 41), but a large table is cleared meanwhile (16,384 of
  // 131,072 x 1,024: 88 against 100)
  p.one = p.n <= kEmbedOne / 4 || (p.n <= kEmbedOne && entries * cols >= int64_t(1) << 26);
  const int most = p.one ? kEmbedOneBits : 10;
  p.digits = (bits + most - 1) / most;
  p.bits = (bits + p.digits - 1) / p.digits;
  p.tiles = int((p.n + kEmbedTile - 1) / kEmbedTile);
  // The shorter the chunks the more groups of lanes, and the more borders.  Units are of four
  // values.  Gradients on one B200, with chunks of 16, 64 and 128: 16,384 entries of 131,072 x
  // 512 (32,768 units at 64) 71, 79 us; 40,000 of 1,000 x 256 (40,000; long stretches) 63, 54; 65,536 x 4 of
  // 40,000 x 64 (65,536) 84, 78; 32,768 of 32,000 x 2,048 (262,144) 152, 115, 124; 131,072 of 32,000 x
  // 1,024 (524,288) 207, 190, 161; 65,537 x 100 of 12,700 x 64 (1.6M) 441 at 64, 428 at 128, 438 at 256.
  p.stretches = p.n / entries >= 16;
  const int64_t units = p.n / 64 * cols / 4;
  p.chunk = units < (p.stretches ? 40000 : 60000) ? 16 : units < 400000 ? 64 : 128;
  p.chunks = (p.n + p.chunk - 1) / p.chunk;
  p.by_row = entries < p.chunks;
  int64_t at = kStatusBytes;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  for (int i = 0; i < (p.one ? 1 : 2); ++i) {
    p.keys[i] = take(p.n * 4);
    p.order[i] = take(p.n * 4);
  }
  p.counts = take(p.one ? 0 : (int64_t(p.tiles) << p.bits) * 4);
  p.totals = take(p.one ? 0 : (int64_t(1) << p.bits) * 4);
  p.heads = take(p.chunks * cols * 4);
  p.tails = take(p.chunks * cols * 4);
  p.begins = take(p.by_row ? entries * 4 : 0);
  p.ends = take(entries * 4);
  int64_t n = p.chunks;
  for (int l = 0; l < kEmbedLevels; ++l) {
    n /= kEmbedGroup;
    p.groups[l] = n;
    p.sums[l] = take(n * cols * 4);
  }
  p.bytes = at;
  return p;
}

int embed_device(int device, const EmbedArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, false, err)) return -1;
  if (a.rows == 0) return 0;
  if (use_device(device, err)) return -1;
  Guard g(device);
  return launched(launch_embed(a, s), "embedding", 1, err);
}

int64_t embed_workspace(int64_t entries, int64_t cols, int64_t rows, int64_t k) {
  std::string err;
  if (check_shape(entries, cols, rows, k, err)) return -1;
  return rows == 0 ? 0 : embed_plan(entries, cols, rows, k).bytes;
}

int embed_grad_device(int device, const EmbedArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, true, err)) return -1;
  if (a.rows == 0) {
    if (use_device(device, err)) return -1;
    Guard g(device);
    const size_t size = size_t(dtype_bytes(a.dtype));
    const cudaError_t e = cudaMemset2DAsync(a.dtable, size_t(a.ld) * size, 0, size_t(a.cols) * size,
                                            size_t(a.entries), s);
    return launched(e, "clearing dtable", 0, err);
  }
  if (!aligned(a.workspace, 256)) return fail(err, "workspace must be 256-byte aligned");
  const EmbedPlan p = embed_plan(a.entries, a.cols, a.rows, a.k);
  if (!a.workspace || a.workspace_bytes < p.bytes)
    return fail(err, "workspace holds " + std::to_string(a.workspace ? a.workspace_bytes : 0) +
                         " bytes, the gradient needs " + std::to_string(p.bytes));
  if (use_device(device, err)) return -1;
  Guard g(device);
  int n = 0;
  const cudaError_t e = launch_embed_grad(a, p, &n, s);
  return launched(e, "embedding gradient", n, err);
}

}  // namespace mb
