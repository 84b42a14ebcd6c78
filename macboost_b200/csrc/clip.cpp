// Host side of gradient clipping (clip.h): argument checks, tables and launches.
#include "clip.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <utility>
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

// Chunks that the norm's launch leaves in the L2 cache for the scaling: 80 MB of its 126.
constexpr unsigned kKeep = (80u << 20) / kClipChunk;

// A launch's tensors, those without values left out and large ones in several entries.
struct Group {
  std::vector<ClipEntry> entries;
  uintptr_t src = UINTPTR_MAX, src_end = 0, dst = UINTPTR_MAX, dst_end = 0;
  unsigned chunks = 0;
  int blocks() const { return int(std::min<unsigned>(chunks, kClipBlocks)); }
};

constexpr uintptr_t kReach = uintptr_t(1) << 33;  // 2^32 units of two bytes

// f(dtype, address of the gradient, of the output, values) for each entry.
template <class F>
void each_entry(const ClipArgs& a, F f) {
  for (int64_t i = 0; i < a.count; ++i) {
    const uintptr_t size = uintptr_t(dtype_bytes(a.dtypes[i]));
    uintptr_t src = a.grads ? reinterpret_cast<uintptr_t>(a.grads[i]) : 0;
    uintptr_t dst = a.outs ? reinterpret_cast<uintptr_t>(a.outs[i]) : 0;
    for (int64_t left = a.sizes[i]; left > 0; left -= kClipMost) {
      const int64_t n = std::min(left, kClipMost);
      f(a.dtypes[i], src, dst, n);
      src += uintptr_t(n) * size;
      if (dst) dst += uintptr_t(n) * size;
    }
  }
}

std::vector<Group> groups_of(const ClipArgs& a) {
  std::vector<Group> all;
  // first the groups' sizes and reach, the entries' addresses from their start
  std::vector<std::pair<uintptr_t, uintptr_t>> at;
  auto close = [&] {
    Group& g = all.back();
    for (size_t i = 0; i < g.entries.size(); ++i) {
      g.entries[i].src = uint32_t((at[i].first - g.src) / 2);
      g.entries[i].dst = uint32_t((at[i].second - g.dst) / 2);
    }
    at.clear();
  };
  each_entry(a, [&](int dtype, uintptr_t src, uintptr_t dst, int64_t n) {
    bool fits = !all.empty() && all.back().entries.size() < size_t(kClipTensors);
    if (fits) {
      const Group& g = all.back();
      fits = std::max(g.src_end, src) - std::min(g.src, src) < kReach &&
             std::max(g.dst_end, dst) - std::min(g.dst, dst) < kReach;
    }
    if (!fits) {
      if (!all.empty()) close();
      all.emplace_back();
      const size_t most = size_t(std::min<int64_t>(a.count, kClipTensors));
      all.back().entries.reserve(most);
      at.reserve(most);
    }
    Group& g = all.back();
    g.src = std::min(g.src, src);
    g.src_end = std::max(g.src_end, src);
    g.dst = std::min(g.dst, dst);
    g.dst_end = std::max(g.dst_end, dst);
    at.emplace_back(src, dst);
    g.entries.push_back(ClipEntry{0, 0, uint32_t(n), g.chunks * 4 + unsigned(dtype)});
    g.chunks += unsigned(chunks_of(dtype, n));
  });
  if (!all.empty()) close();
  return all;
}

template <int N>
void fill(ClipTable<N>& t, const Group& g, bool outs) {
  t.src = reinterpret_cast<const char*>(g.src);
  t.dst = outs ? reinterpret_cast<char*>(g.dst) : nullptr;
  t.tensors = int(g.entries.size());
  t.chunks = g.chunks;
  std::copy(g.entries.begin(), g.entries.end(), t.entry);
  t.shift = 0;
  while (((t.chunks - 1) >> t.shift) >= unsigned(kClipBuckets)) ++t.shift;
  int i = 0;
  for (int b = 0; b <= kClipBuckets; ++b) {
    const uint64_t chunk = uint64_t(b) << t.shift;
    while (i + 1 < t.tensors && g.entries[size_t(i) + 1].chunk0 / 4 <= chunk) ++i;
    t.bucket[b] = static_cast<uint16_t>(i);
  }
}

template <int N>
cudaError_t run(const Group& g, const ClipState& c, bool outs, int pass, cudaStream_t s) {
  // its entries beyond the tensors' are not read
  const std::unique_ptr<ClipTable<N>> t(new ClipTable<N>);
  fill(*t, g, outs);
  return pass ? launch_clip_scale<N>(*t, c, g.blocks(), s) : launch_clip_norm<N>(*t, c, g.blocks(), s);
}

}  // namespace

int64_t clip_workspace(int64_t count, const int32_t* dtypes, const int64_t* sizes) {
  std::string err;
  if (check_list(count, dtypes, sizes, err)) return -1;
  // a block of every launch: no more than chunks, nor than there are launches for tensors that
  // lie anywhere
  int64_t chunks = 0, tensors = 0;
  for (int64_t i = 0; i < count; ++i) {
    chunks += chunks_of(dtypes[i], sizes[i]);
    tensors += (sizes[i] + kClipMost - 1) / kClipMost;
  }
  return std::min(chunks, tensors * kClipBlocks) * int64_t(sizeof(double));
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
  const std::vector<Group> groups = groups_of(a);
  ClipState c{};
  c.part = static_cast<double*>(a.workspace);
  for (const Group& g : groups) c.parts += g.blocks();
  if (!aligned(a.workspace, 8)) return fail(err, "workspace must be 8-byte aligned");
  const int64_t need = clip_workspace(a.count, a.dtypes, a.sizes);
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
  const bool outs = a.outs != nullptr;
  if (groups.size() == 1 && groups[0].entries.size() <= size_t(kClipFew) && groups[0].chunks <= unsigned(kClipOne)) {
    ClipTable<kClipFew> t;
    fill(t, groups[0], outs);
    e = launch_clip_one(t, c, s);
    launches = 1;
  } else if (groups.empty()) {
    e = launch_clip_finish(c, s);
    launches = 1;
  } else {
    for (int pass = 0; pass < (outs ? 2 : 1) && e == cudaSuccess; ++pass) {
      c.first = 0;
      for (size_t i = 0; i < groups.size() && e == cudaSuccess; ++i) {
        // the last gradients read are the first ones scaled
        const size_t at = pass ? groups.size() - 1 - i : i;
        const Group& g = groups[at];
        c.keep = outs && at + 1 == groups.size() && g.chunks > kKeep ? g.chunks - kKeep : 0;
        e = g.entries.size() <= size_t(kClipFew) ? run<kClipFew>(g, c, outs, pass, s)
                                                 : run<kClipTensors>(g, c, outs, pass, s);
        c.first += g.blocks();
        ++launches;
      }
    }
    if (e == cudaSuccess && !outs) {
      e = launch_clip_finish(c, s);
      ++launches;
    }
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, std::string("clip launch: ") + cudaGetErrorString(e));
  }
  g_kernel_launches.fetch_add(launches, std::memory_order_relaxed);
  return 0;
}

}  // namespace mb
