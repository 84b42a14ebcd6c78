// A softmax head: the cross entropy of softmax(h W^T) over many classes, and its
// gradient, without the logits in memory.
//
//   l = h W^T (rows x classes),  lse_n = log sum_v exp(l_nv),
//   loss_n = lse_n - l[n, label_n]           (0 for a label outside 0..classes-1)
//   g = dloss_n (exp(l - lse_n) - [v = label_n])   (0 for such a row)
//   dh = g W,  dW = g^T h
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace mb {

struct HeadArgs {
  int dtype = 0;               // kF32 or kBF16
  const void* h = nullptr;     // rows x cols, stride ld_h
  int64_t rows = 0, cols = 0, ld_h = 0;
  const void* w = nullptr;     // classes x cols, stride ld_w
  int64_t classes = 0, ld_w = 0;
  const int32_t* labels = nullptr;
  float* loss = nullptr;       // forward outputs
  float* lse_out = nullptr;
  const float* lse = nullptr;  // gradient inputs
  const float* dloss = nullptr;
  void* dh = nullptr;          // either may be null
  int64_t ld_dh = 0;
  void* dw = nullptr;
  int64_t ld_dw = 0;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

int64_t head_workspace(int dtype, int64_t rows, int64_t cols, int64_t classes, bool grad,
                       bool strided);
int head_loss_device(int device, const HeadArgs& a, cudaStream_t s, std::string& err);
int head_grad_device(int device, const HeadArgs& a, cudaStream_t s, std::string& err);
// Wait for `device` and report a wait of these kernels that ran out.  The word at the start
// of the workspace is cleared by the loss call, and marked by a wait of either call; the
// gradient call leaves it, since it works from an lse that a wait may have cost.
int head_check_device(int device, const void* workspace, std::string& err);

// ---- between head.cpp and kernels_head.cu ---------------------------------------

// The mark: a value that a workspace without a loss call hardly holds.
constexpr unsigned kHeadExpired = 0x9E37C0DEu;
constexpr int kHeadTileM = 128;      // accumulator rows a CTA (TMEM lanes)
constexpr int kHeadTileN = 256;      // accumulator columns
constexpr int kHeadTileK = 64;       // one 128-byte swizzle row of 16-bit values
constexpr int kHeadPair = 2;         // CTAs that share a tile
constexpr int kHeadEpilogue = 12;    // a tile's epilogue, in steps of one K block

// Division of numbers below 2^31 by a constant, by multiplication (Granlund and Montgomery,
// "Division by Invariant Integers using Multiplication", 1994): with p = 31 + ceil(log2 d) and m = ceil(2^p
// / d), n / d is n m >> p.  A tile's place takes four divisions, and a role that has to
// divide in full between tiles leaves the tensor cores waiting for about a microsecond.
struct HeadDiv {
  unsigned d, m, s;
  void set(int64_t by) {
    d = unsigned(by);
    unsigned log = 0;
    while ((uint64_t(1) << log) < d) ++log;
    s = log > 0 ? log - 1 : 0;
    m = d > 1 ? unsigned(((uint64_t(1) << (31 + log)) + d - 1) / d) : 0;
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const {
    return d == 1 ? n : int(__umulhi(unsigned(n), m) >> s);
  }
#endif
};

// One product C = A B^T over K, as tiles.  Operands are 16-bit values in `planes`
// planes (the terms of a float32, or the value itself) behind tensor maps of
// (inner, outer, plane).  a_mn / b_mn: the inner dimension is the tile's own (M or N),
// not K.
struct HeadJob {
  CUtensorMap a, b;
  int a_mn, b_mn;
  int tiles_m, tiles_n, splits;      // splits: parts of K, each with its own output
  int kblocks;                       // ceil(K / kHeadTileK)
  int part, longer;                  // a part's K blocks; the first `longer` have one more
  int group;                         // tile rows walked together (L2 reuse)
  HeadDiv by_split, by_group, by_rows, by_last;  // see divide()
  int a_row0, b_row0;                // first outer coordinate of A and B (K-major) ...
  int a_k0, b_k0;                    // ... and first K coordinate of each
  int a_box, b_box;                  // rows of a K-major operand's box
  int b_from, b_skip;                // B's K coordinate is b_skip lower from K = b_from on
  int M, N;                          // the product's rows and columns
  int m_from, m_to;                  // rows that are not written out; those behind move up
  int plain;                         // in a launch with another epilogue: the plain one
  // output of the plain epilogue
  float* acc;                        // float32 sums, stride N, M * N apart per split
  int acc_in, final;                 // add what acc holds; write out (else acc)
  void* out;
  long long ld_out;
  int out_f32;
  int wide;                          // rows of out start on four values; 2: on 16 bytes of bfloat16

  void divide() {                    // once tiles, group, splits and kblocks are known
    by_split.set(int64_t(tiles_m) * tiles_n);
    by_group.set(int64_t(group) * tiles_n);
    by_rows.set(group);
    const int last = tiles_m % group;
    by_last.set(last ? last : group);
    part = kblocks / splits;
    longer = kblocks % splits;
  }
};

struct HeadRows {                    // what the logits' epilogues know of each row
  const int* labels;
  const float* lse;
  const float* dloss;
  float2* part;                      // forward: (max, sum) of each row and half tile
  float* target;                     // forward: the label's logit
  void* g;                           // gradient: planes x rows x ld_g of bfloat16
  long long ld_g, plane_g;
  int rows, classes, v0;             // v0: first class of this piece
  const float *h, *w;                // float32: the inputs themselves (redo_logits)
  long long ld_h, ld_w;
  int cols;
};

struct HeadGate {                    // what the epilogues of a gated block know (ffn.h)
  int act, width, rows;
  void* hidden;                      // forward: rows x width
  long long ld_hidden;
  float* pre;                        // rows x 2 width, forward: or null
  long long ld_pre;
  void* dpre;                        // gradient: rows x 2 half of bfloat16, zeros from `width` to `half`
  long long ld_d;
  int half;                          // width, up to a whole K block
  int wide, wide_pre;                // rows of hidden, and of both halves of pre, start on 16 bytes
};

struct HeadLaunch {
  HeadJob job[2];
  int jobs;
  int f32;                           // three planes an operand, six products
  HeadRows r;
  HeadGate g;
  unsigned* status;
  unsigned long long wait_ns;
  int stall;                         // test hook: no copy is issued, so waits run out
};

// A narrow head takes none of this: kernels of its own, in float32 (kernels_head.cu).
constexpr int kNarrowCols = 64, kNarrowClasses = 32;
// Blocks: enough to fill the GPU four times, one for 128 rows at most.
inline int narrow_blocks(int64_t rows) {
  const int64_t n = (rows + 127) / 128;
  return int(n < 592 ? n : 592);
}
cudaError_t launch_head_narrow(const HeadArgs& h, bool grad, float* part, int blocks, cudaStream_t s);

// Nor does a head of few rows, whose h fits in shared memory: float32 to 16 rows,
// bfloat16 to 4.  Measured at 1,024 x 131,072 bfloat16, loss: 4 rows 61 us here and 72 us
// on the tensor cores, 8 rows 105 and 72.
constexpr int64_t kFewSmem = 128 * 1024;
// Floats between its rows there: whole steps of 64 columns.
#ifdef __CUDACC__
__host__ __device__
#endif
inline int few_pitch(long long cols) { return int((cols + 63) / 64 * 64); }
struct HeadFew {
  int blocks, chunks;                // of the first kernel; of the classes for dh
  float2* part;
  float* target;
  float* g;
  float* dh_part;
};
cudaError_t launch_head_few(const HeadArgs& h, bool grad, const HeadFew& f, cudaStream_t s);

// kHeadOut: the head's sums written out; kHeadBlock: the gated block's.
enum { kHeadLse = 0, kHeadG = 1, kHeadOut = 2, kHeadGate = 3, kHeadGateGrad = 4, kHeadBlock = 5 };
cudaError_t launch_head(int epilogue, int tile_n, const HeadLaunch& a, cudaStream_t s);
// Source rows (float32 or bfloat16) to planes of bfloat16 (3 or 1), stride ldp; rows
// whose label (unless null) is none of the classes become zeros.
struct HeadPack {
  const void* src = nullptr;
  long long rows = 0, cols = 0, ld = 0;
  const int* labels = nullptr;
  long long classes = 0;
  void* dst = nullptr;
  long long ldp = 0;
};
constexpr int kHeadPacks = 5;        // matrices of a launch, at most
cudaError_t launch_head_pack(int dtype, const HeadPack* list, int count, unsigned* status, cudaStream_t s);
cudaError_t launch_head_finish(const float2* part, const float* target, const int* labels,
                               int64_t rows, int64_t classes, int64_t parts, float* loss,
                               float* lse, cudaStream_t s);
// out = (acc_in ? acc : 0) + sum of the splits' parts, to out or back to acc.
struct HeadReduce {
  const float* part;
  int splits;
  int64_t M, N;
  float* acc;
  int acc_in, final;
  void* out;
  int64_t ld_out;
  int out_f32;
  int64_t m_from, m_to;              // as a job's
};
cudaError_t launch_head_reduce(const HeadReduce& a, cudaStream_t s);

// What a workspace begins with: the status word of the calls whose waits may run out.  Calls whose waits
// cannot leave it alone too, so that the word outlives those that follow in the same workspace.
constexpr int64_t kStatusBytes = 256;

// Host side of products as tiles, for the blocks that use them (head.cpp).
// TMA reads rows in place when they start on 16 bytes.
bool head_in_place(int dtype, const void* p, int64_t ld);
// A matrix of planes x outer x inner 16-bit values, stride ld, fetched in boxes of 64
// inner x `box` outer values into 128-byte swizzled rows; zeros outside.
int head_encode(CUtensorMap* m, const void* p, int64_t inner, int64_t outer, int64_t ld, int planes,
                int box, std::string& err);
// Rows of a K-major box: all of a tile's, or the matrix's when it has fewer.
int head_box_rows(int64_t rows, int tile);
// The status word, the limit of waits and the test hook.
void head_settings(HeadLaunch& l, int dtype, void* workspace);

}  // namespace mb
