// Host side of gradient clipping (clip.h): argument checks, tables and launches.
#include "clip.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include "engine.h"
#include "mixture.h"

namespace mb {

namespace {

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

int64_t chunks_of(int dtype, int64_t size) {
  const int64_t per = kClipChunk / dtype_bytes(dtype);
  return (size + per - 1) / per;
}

int check_list(int64_t count, const int32_t* dtypes, const int64_t* sizes, std::string& err) {
  if (count < 0 || count > (int64_t(1) << 24)) return fail(err, "count must be in 0...2^24");
  if (count > 0 && (!dtypes || !sizes)) return fail(err, "null argument");
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!dtype_bytes(dtypes[i]))
      return fail(err, "unknown dtype " + std::to_string(dtypes[i]) + " (0 float32, 1 bfloat16, 2 float16)");
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40)) return fail(err, "sizes must be in 0...2^40");
    chunks += chunks_of(dtypes[i], sizes[i]);
    if (chunks > (int64_t(1) << 27)) return fail(err, "the gradients hold too many values for one call");
  }
  return 0;
}

// The launches: tensors from `begin` on, those without values left out.
struct Group {
  int64_t begin, end, chunks;
  int tensors;
};
std::vector<Group> groups_of(int64_t count, const int32_t* dtypes, const int64_t* sizes) {
  std::vector<Group> all;
  Group g{0, 0, 0, 0};
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    if (g.tensors == kClipTensors) {
      g.end = i;
      all.push_back(g);
      g = Group{i, i, 0, 0};
    }
    ++g.tensors;
    g.chunks += chunks_of(dtypes[i], sizes[i]);
  }
  g.end = count;
  if (g.tensors > 0) all.push_back(g);
  return all;
}

int blocks_of(const Group& g) { return int(std::min<int64_t>(g.chunks, kClipBlocks)); }

template <int N>
void fill(ClipTable<N>& t, const ClipArgs& a, const Group& g) {
  t.tensors = 0;
  unsigned chunk = 0;
  for (int64_t i = g.begin; i < g.end; ++i) {
    if (a.sizes[i] == 0) continue;
    const int n = t.tensors++;
    t.src[n] = a.grads[i];
    t.dst[n] = a.outs ? a.outs[i] : nullptr;
    t.size[n] = a.sizes[i];
    t.chunk0[n] = chunk;
    t.dtype[n] = static_cast<unsigned char>(a.dtypes[i]);
    chunk += unsigned(chunks_of(a.dtypes[i], a.sizes[i]));
  }
  t.chunks = chunk;
}

template <int N>
cudaError_t run(const ClipArgs& a, const Group& g, const ClipState& c, bool scale, cudaStream_t s) {
  const auto t = std::make_unique<ClipTable<N>>();
  fill(*t, a, g);
  return scale ? launch_clip_scale<N>(*t, c, blocks_of(g), s) : launch_clip_norm<N>(*t, c, blocks_of(g), s);
}

}  // namespace

int64_t clip_workspace(int64_t count, const int32_t* dtypes, const int64_t* sizes) {
  std::string err;
  if (check_list(count, dtypes, sizes, err)) return -1;
  int64_t parts = 0;
  for (const Group& g : groups_of(count, dtypes, sizes)) parts += blocks_of(g);
  return parts * int64_t(sizeof(double));
}

int clip_device(int device, const ClipArgs& a, cudaStream_t s, std::string& err) {
  if (check_list(a.count, a.dtypes, a.sizes, err)) return -1;
  if (!(a.max_norm >= 0)) return fail(err, "max_norm must be >= 0");
  if (!a.norm || (a.count > 0 && !a.grads)) return fail(err, "null argument");
  if (!aligned(a.norm, 4)) return fail(err, "norm must be 4-byte aligned");
  bool in_place = true;
  for (int64_t i = 0; i < a.count; ++i) {
    if (a.sizes[i] == 0) continue;
    if (!a.grads[i] || (a.outs && !a.outs[i])) return fail(err, "null argument");
    const size_t size = size_t(dtype_bytes(a.dtypes[i]));
    if (!aligned(a.grads[i], size) || (a.outs && !aligned(a.outs[i], size)))
      return fail(err, "gradients must be aligned to their values");
    in_place = in_place && a.outs && a.outs[i] == a.grads[i];
  }
  const std::vector<Group> groups = groups_of(a.count, a.dtypes, a.sizes);
  ClipState c{};
  c.part = static_cast<double*>(a.workspace);
  for (const Group& g : groups) c.parts += blocks_of(g);
  if (!aligned(a.workspace, 8)) return fail(err, "workspace must be 8-byte aligned");
  const int64_t need = c.parts * int64_t(sizeof(double));
  if (need > 0 && (!a.workspace || a.workspace_bytes < need))
    return fail(err, "workspace holds " + std::to_string(a.workspace ? a.workspace_bytes : 0) +
                         " bytes, the norm needs " + std::to_string(need));
  c.max_norm = a.max_norm;
  c.norm = a.norm;
  c.in_place = in_place;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  int launches = 0;
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < (a.outs ? 2 : 1) && e == cudaSuccess; ++pass) {
    c.first = 0;
    for (size_t i = 0; i < groups.size() && e == cudaSuccess; ++i) {
      // the last gradients read are the first ones scaled
      const Group& g = groups[pass ? groups.size() - 1 - i : i];
      e = g.tensors <= kClipFew ? run<kClipFew>(a, g, c, pass, s) : run<kClipTensors>(a, g, c, pass, s);
      c.first += blocks_of(g);
      ++launches;
    }
  }
  if (e == cudaSuccess && (!a.outs || groups.empty())) {
    e = launch_clip_finish(c, s);
    ++launches;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, std::string("clip launch: ") + cudaGetErrorString(e));
  }
  g_kernel_launches.fetch_add(launches, std::memory_order_relaxed);
  return 0;
}

}  // namespace mb
