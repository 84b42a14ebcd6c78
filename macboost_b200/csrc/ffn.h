// A gated feed-forward block and its gradient.
//
//   a = x Wg^T,  b = x Wu^T      (w_in: width rows of Wg, then width rows of Wu)
//   h = act(a) b,  y = h Wo^T
//   dh = dy Wo,  da = dh b act'(a),  db = dh act(a)
//   dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x,  dWo = dy^T h
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace mb {

constexpr int kSilu = 0, kGelu = 1, kGeluTanh = 2;   // MACBOOST_ACT_*

struct FfnArgs {
  int dtype = 0, act = 0;
  const void* x = nullptr;       // rows x cols
  int64_t rows = 0, cols = 0, ld_x = 0;
  const void* w_in = nullptr;    // 2 width x cols
  int64_t width = 0, ld_in = 0;
  const void* w_out = nullptr;   // outs x width
  int64_t outs = 0, ld_out = 0;
  void* hidden = nullptr;        // rows x width: forward output, gradient input
  int64_t ld_hidden = 0;
  float* pre = nullptr;          // rows x 2 width, the same; forward: may be null
  int64_t ld_pre = 0;
  void* y = nullptr;             // forward: rows x outs
  int64_t ld_y = 0;
  const void* dy = nullptr;      // gradient: rows x outs
  int64_t ld_dy = 0;
  void* dx = nullptr;            // each may be null
  int64_t ld_dx = 0;
  void* dw_in = nullptr;
  int64_t ld_din = 0;
  void* dw_out = nullptr;
  int64_t ld_dout = 0;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

int64_t ffn_workspace(int dtype, int64_t rows, int64_t cols, int64_t width, int64_t outs, bool grad,
                      bool strided);
int ffn_device(int device, const FfnArgs& a, cudaStream_t s, std::string& err);
int ffn_grad_device(int device, const FfnArgs& a, cudaStream_t s, std::string& err);
// Wait for `device` and report a wait of these kernels that ran out (as the head's).
int ffn_check_device(int device, const void* workspace, std::string& err);

// ---- between ffn.cpp and kernels_ffn.cu -------------------------------------------

// Up to four rows (float32: 16) whose x and h fit in shared memory go to the CUDA cores:
// reading the weights bounds them.  In us, against tiles of the tensor cores: float32 1, 4 rows of
// 2,048 x 8,192 41, 55 against 249; 8 of 1,024 x 4,096 33 against 94; bfloat16 1, 2, 4 of 2,048 x 8,192 25,
// 33, 43 against 39, of 1,024 x 4,096 10.5, 14.5, 18.6 against 27 (2 and 4 only where the
// products of warps cannot).
constexpr int64_t kFfnFewRows = 4, kFfnFewRowsF32 = 16;
constexpr int64_t kFfnFewSmem = 128 * 1024;
inline int64_t ffn_pitch(int64_t cols) { return (cols + 63) / 64 * 64; }  // floats between rows there
cudaError_t launch_ffn_few(const FfnArgs& a, cudaStream_t s);
// Products of warps: two to 16 rows of bfloat16 whose matrices' rows start on 16 bytes and are whole
// 16 bytes long, and up to 48 where they take no more than this many products.  In us, against tiles:
// 32 x 2,048 x 8,192 (1.6e9) 41 against 47 and 40 rows (2.0e9) 53 against 47; 32 x 1,024 x 16,384 (1.6e9) 50
// against 47; 48 x 1,536 x 4,096 (0.9e9) 30 against 37; 24 x 4,096 x 16,384 (4.8e9) 132 against 103.
constexpr int64_t kFfnWarpRows = 16, kFfnWarpMost = 48;
constexpr double kFfnWarpProducts = 1.4e9;
// Terms of a bfloat16 sum that the tensor core, which truncates it at each step of 16, holds in one place:
// 2,048 steps lose 2^-12 at most.  A million terms of one sign in one place lost 0.6%, more than a rounding to
// bfloat16; a block's eight warps share a sum.
constexpr int64_t kFfnLong = 32768, kFfnWarpLong = 8 * kFfnLong;
cudaError_t launch_ffn_rows(const FfnArgs& a, cudaStream_t s);
// bfloat16: hidden from pre (rows x 2 width, stride ld_pre).
cudaError_t launch_ffn_gate(const FfnArgs& a, const float* pre, int64_t ld_pre, cudaStream_t s);
// From dh (float32, stride ld_dh) and pre to the gradients of both halves, zeros from width to half:
// float32 in planes (3 x rows x 2 half), and those of hidden (3 x rows x ld_h) unless h is null; bfloat16,
// whose dh is here where outs are long, rounded (rows x 2 half).
struct FfnSplit {
  int dtype, act;
  long long rows;
  int width, half, ld_h;
  const float* dh;
  long long ld_dh;
  const float* pre;
  long long ld_pre;
  const float* hidden;
  long long ld_hidden;
  void *dpre, *h;
};
cudaError_t launch_ffn_split(const FfnSplit& a, cudaStream_t s);

// float32 with few outputs (a class margin each, say): y, dh and dw_out are too little for tiles that
// want planes of h first, and go to the CUDA cores.  Forward passes of 64 columns as graphs, these and tiles, in us
// at 17, 200, 800 and 6,400 rows: 403 x 10 18, 19, 20, 31 and 27, 29, 29, 46; 1,024 x 16 20, 23, 25, 50 and 26, 27, 28, 60;
// 4,096 x 1 35, 36, 47, 119 and 39, 40, 53, 185.  Where both limits meet tiles end up to 15% sooner on few rows
// (4,096 x 4 41, 45, 56, 141 and 40, 41, 53, 186; 16,384 x 1 113, 120, 164, 424 and 103, 108, 186, 647), but the
// gradient does not: 17 rows of 16,384 x 1 64, of 17 outputs, as tiles, 126.
constexpr int64_t kFfnNarrow = 16, kFfnNarrowValues = 16384;  // outs; outs * width
constexpr int64_t kFfnNarrowWarps = 1184;                     // of the gradient, at least: eight a multiprocessor
cudaError_t launch_ffn_narrow(const FfnArgs& a, cudaStream_t s);
struct FfnNarrow {
  int act, outs;
  long long rows, per;       // rows, and those of a warp
  int width, half;
  const float* dy;
  long long ld_dy;
  const float* w;            // outs x width
  long long ld_w;
  const float* pre;
  long long ld_pre;
  const float* hidden;
  long long ld_hidden;
  void* dpre;                // planes as FfnSplit's, or null
  float* part;               // dw_out's sums of `per` rows, outs x width each, or null
};
cudaError_t launch_ffn_narrow_grad(const FfnNarrow& a, cudaStream_t s);

}  // namespace mb
