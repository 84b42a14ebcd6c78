// The norm of many gradients taken together, and their clipping.
//
//   norm = sqrt(sum over all tensors and values of g^2)
//   factor = max_norm / norm where norm > max_norm, else 1 (NaN for a norm that is NaN)
//   out = factor * g, rounded once
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace mb {

struct ClipArgs {
  int64_t count;
  const int32_t* dtypes;          // host arrays of `count`
  const void* const* grads;
  const int64_t* sizes;
  void* const* outs;              // null: only the norm
  double max_norm;
  float* norm;                    // device
  void* workspace;
  int64_t workspace_bytes;
};

int64_t clip_workspace(int64_t count, const int32_t* dtypes, const int64_t* sizes);
int clip_device(int device, const ClipArgs& a, cudaStream_t s, std::string& err);

// ---- between clip.cpp and kernels_clip.cu -----------------------------------------

// A tensor's values in chunks, a chunk a block's at a time.  Tables of tensors travel as a
// launch's parameters (at most 32,764 bytes): nothing is copied to the device first, so a
// captured graph holds its tables.  16 bytes a tensor: where it starts behind the lowest
// address of its table, in units of two bytes, so a table's tensors lie within 8 GB.
constexpr int kClipChunk = 32 * 1024;      // bytes
constexpr int kClipTensors = 2032;         // of a launch
constexpr int kClipFew = 64;               // of a launch with a small table
constexpr int kClipBlocks = 592;           // of a launch, at most: four a multiprocessor
constexpr int64_t kClipMost = int64_t(1) << 31;  // values of an entry; a larger tensor is several
// One launch for gradients that a cluster of eight blocks takes in a few rounds, up to 1 MB: 8.3 us
// either way, but the host launches once; with four times as many rounds 12 to 16 us against 8.3.
constexpr int kClipCluster = 8, kClipOne = 32;  // blocks; chunks

struct ClipEntry {
  uint32_t src, dst;                       // behind the table's bases, in units of two bytes
  uint32_t size;                           // values
  uint32_t chunk0;                         // first chunk * 4 + dtype
};

constexpr int kClipBuckets = 64;

template <int N>
struct ClipTable {
  const char* src;
  char* dst;                               // null: only the norm
  int tensors;
  unsigned chunks;
  // where a search begins and ends: the tensors of chunks 0, 1 << shift, 2 << shift ..., and the last
  int shift;
  uint16_t bucket[kClipBuckets + 1];
  ClipEntry entry[N];
};

struct ClipState {
  double* part;                            // a block's sum of squares, of all launches
  int parts, first;                        // of all launches; this launch's first
  double max_norm;
  float* norm;
  int in_place;                            // every out is its gradient: a factor of 1 writes nothing
  unsigned keep;                           // chunks from here on are expected in the L2 cache again
};
template <int N>
cudaError_t launch_clip_norm(const ClipTable<N>& t, const ClipState& c, int blocks, cudaStream_t s);
template <int N>
cudaError_t launch_clip_scale(const ClipTable<N>& t, const ClipState& c, int blocks, cudaStream_t s);
cudaError_t launch_clip_one(const ClipTable<kClipFew>& t, const ClipState& c, cudaStream_t s);
cudaError_t launch_clip_finish(const ClipState& c, cudaStream_t s);

}  // namespace mb
