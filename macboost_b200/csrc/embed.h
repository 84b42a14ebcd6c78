// Embeddings: rows of a table looked up by ids and added up, and the table's gradient.
//
//   out[n] = scale * sum over j of table[starts[j] + ids[n, j]]        (n < rows, j < k)
//   dtable[e] = scale * sum of dout[n] over the entries (n, j) that looked up e
//
// An entry whose id is negative, or whose row of the table does not exist, adds nothing.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace mb {

struct EmbedArgs {
  int dtype;
  const void* table;       // forward: entries x cols, stride ld
  long long entries, cols, ld;
  const int* ids;          // rows x k
  long long rows, k;
  const int* starts;       // k of them, or null: zeros
  float scale;
  void* out;               // forward: rows x cols, stride ld_out
  long long ld_out;
  const void* dout;        // gradient: rows x cols, stride ld_out
  void* dtable;            // gradient: entries x cols, stride ld
  void* workspace;
  long long workspace_bytes;
};

int embed_device(int device, const EmbedArgs& a, cudaStream_t s, std::string& err);
int64_t embed_workspace(int64_t entries, int64_t cols, int64_t rows, int64_t k);
int embed_grad_device(int device, const EmbedArgs& a, cudaStream_t s, std::string& err);

// ---- between embed.cpp and kernels_embed.cu --------------------------------------

// The gradient's sort: a stable radix sort of the entries by row of the table, `digits` of
// `bits` bits each; what adds nothing gets the row `entries`, behind all others.
constexpr int kEmbedOne = 16384;          // entries of a sort that is one block's, in one launch
constexpr int kEmbedOneBits = 9;          // of its digits, at most; else 10
constexpr int kEmbedTile = 2048;          // entries a block of a larger sort
constexpr int kEmbedGroup = 64;           // chunks (or sums of them) added up at once
constexpr int kEmbedLevels = 2;           // sums of 64 and of 64 x 64 chunks

struct EmbedPlan {
  long long n;                            // entries of the sort, rows * k
  int digits, bits, tiles;
  bool one;                               // that is one block's, in one launch
  bool stretches;                         // of 16 entries and more, on average
  int chunk;                              // sorted entries that a group of lanes adds up
  long long chunks;
  bool by_row;                            // the join goes by rows of the table, not by chunks
  // offsets into the workspace
  long long keys[2], order[2], counts, totals, heads, tails, begins, ends, sums[kEmbedLevels], bytes;
  long long groups[kEmbedLevels];         // sums a level
};
EmbedPlan embed_plan(int64_t entries, int64_t cols, int64_t rows, int64_t k);

cudaError_t launch_embed(const EmbedArgs& a, cudaStream_t s);
cudaError_t launch_embed_grad(const EmbedArgs& a, const EmbedPlan& p, int* launches, cudaStream_t s);

}  // namespace mb
