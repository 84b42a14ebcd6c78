// Host side of gradient clipping (clip.h): argument checks, tables and launches.
#include "clip.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include "engine.h"
#include "head.h"
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

// Chunks of `size` values; a division for each of a few thousand tensors would take as long as
// the launches.
int64_t chunks_of(int dtype, int64_t size) {
  static_assert(kClipChunk == 1 << 15, "values of a chunk as a power of two");
  const int bits = dtype == kF32 ? 13 : 14;
  return (size + (int64_t(1) << bits) - 1) >> bits;
}

// The list's types and sizes; `room`: the workspace it needs.
int check_list(int64_t count, const int32_t* dtypes, const int64_t* sizes, int64_t* room, std::string& err) {
  if (count < 0 || count > (int64_t(1) << 24)) return fail(err, "count must be in 0...2^24");
  if (count > 0 && (!dtypes || !sizes)) return fail(err, "null argument");
  int64_t chunks = 0, entries = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int dtype = dtypes[i];
    if (!dtype_bytes(dtype))
      return fail(err, "unknown dtype " + std::to_string(dtype) + " (0 float32, 1 bfloat16, 2 float16)");
    if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 40)) return fail(err, "sizes must be in 0...2^40");
    chunks += chunks_of(dtype, sizes[i]);
    entries += (sizes[i] + kClipMost - 1) / kClipMost;  // a shift
    if (chunks > (int64_t(1) << 27)) return fail(err, "the gradients hold too many values for one call");
  }
  // a block's sum of every launch: no more than chunks, nor than entries that all lie far apart ask for
  *room = chunks > 0 ? kStatusBytes + std::min(chunks, entries * kClipBlocks) * int64_t(sizeof(double)) : 0;
  return 0;
}

// Chunks that the norm's launch leaves in the L2 cache for the scaling: 80 MB of its 126.  340 MB of
// bfloat16 take 166 us so, 173 with nothing read or stored so that it leaves first.
constexpr unsigned kKeep = (80u << 20) / kClipChunk;

// The list's entries one after the other: tensors without values left out, large ones in
// several.
struct Entry {
  uintptr_t src, dst;
  int64_t size;
  int dtype;
};
struct Cursor {
  int64_t tensor = 0, done = 0;
  bool next(const ClipArgs& a, Entry* e) {
    while (tensor < a.count && a.sizes[tensor] == done) {
      ++tensor;
      done = 0;
    }
    if (tensor >= a.count) return false;
    e->dtype = a.dtypes[tensor];
    const uintptr_t at = uintptr_t(done) * uintptr_t(e->dtype == kF32 ? 4 : 2);
    e->src = reinterpret_cast<uintptr_t>(a.grads[tensor]) + at;
    e->dst = a.outs ? reinterpret_cast<uintptr_t>(a.outs[tensor]) + at : 0;
    e->size = std::min(a.sizes[tensor] - done, kClipMost);
    done += e->size;
    return true;
  }
};

// A launch's entries, from a place of the list on, and their lowest addresses.
struct Group {
  Cursor from;
  int entries = 0;
  uintptr_t src = UINTPTR_MAX, dst = UINTPTR_MAX;
  unsigned chunks = 0;
  int blocks() const { return int(std::min<unsigned>(chunks, kClipBlocks)); }
};

constexpr uintptr_t kReach = uintptr_t(1) << 33;  // 2^32 units of two bytes

std::vector<Group> groups_of(const ClipArgs& a) {
  std::vector<Group> all;
  uintptr_t src_end = 0, dst_end = 0;
  Cursor at;
  Entry e;
  for (Cursor before = at; at.next(a, &e); before = at) {
    if (all.empty() || all.back().entries == kClipTensors ||
        std::max(src_end, e.src) - std::min(all.back().src, e.src) >= kReach ||
        std::max(dst_end, e.dst) - std::min(all.back().dst, e.dst) >= kReach) {
      all.emplace_back();
      all.back().from = before;
      src_end = dst_end = 0;
    }
    Group& g = all.back();
    ++g.entries;
    g.src = std::min(g.src, e.src);
    g.dst = std::min(g.dst, e.dst);
    src_end = std::max(src_end, e.src);
    dst_end = std::max(dst_end, e.dst);
    g.chunks += unsigned(chunks_of(e.dtype, e.size));
  }
  return all;
}

template <int N>
void fill(ClipTable<N>& t, const ClipArgs& a, const Group& g) {
  t.src = reinterpret_cast<const char*>(g.src);
  t.dst = a.outs ? reinterpret_cast<char*>(g.dst) : nullptr;
  t.tensors = g.entries;
  t.chunks = g.chunks;
  t.shift = 0;
  while (((t.chunks - 1) >> t.shift) >= unsigned(kClipBuckets)) ++t.shift;
  Cursor at = g.from;
  Entry e;
  unsigned chunk = 0;
  int bucket = 0;
  for (int i = 0; i < g.entries && at.next(a, &e); ++i) {
    t.entry[i] = ClipEntry{uint32_t((e.src - g.src) / 2), uint32_t((e.dst - g.dst) / 2), uint32_t(e.size),
                           chunk * 4 + unsigned(e.dtype)};
    chunk += unsigned(chunks_of(e.dtype, e.size));
    // the buckets whose first chunk is this entry's
    for (; bucket <= kClipBuckets && (uint64_t(bucket) << t.shift) < chunk; ++bucket)
      t.bucket[bucket] = static_cast<uint16_t>(i);
  }
  for (; bucket <= kClipBuckets; ++bucket) t.bucket[bucket] = static_cast<uint16_t>(g.entries - 1);
}

// The launches of a group: its sums, then (another time) its outputs.
template <int N>
struct Launch {
  std::unique_ptr<ClipTable<N>> table;
  cudaError_t operator()(const ClipArgs& a, const Group& g, const ClipState& c, int pass, cudaStream_t s) {
    if (!table) {
      table.reset(new ClipTable<N>);  // entries beyond the tensors' are not read
      fill(*table, a, g);
    }
    return pass ? launch_clip_scale<N>(*table, c, g.blocks(), s) : launch_clip_norm<N>(*table, c, g.blocks(), s);
  }
};

}  // namespace

int64_t clip_workspace(int64_t count, const int32_t* dtypes, const int64_t* sizes) {
  std::string err;
  int64_t room = 0;
  return check_list(count, dtypes, sizes, &room, err) ? -1 : room;
}

int clip_device(int device, const ClipArgs& a, cudaStream_t s, std::string& err) {
  int64_t need = 0;
  if (check_list(a.count, a.dtypes, a.sizes, &need, err)) return -1;
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
  if (a.workspace) c.part = reinterpret_cast<double*>(static_cast<char*>(a.workspace) + kStatusBytes);
  for (const Group& g : groups) c.parts += g.blocks();
  if (!aligned(a.workspace, 8)) return fail(err, "workspace must be 8-byte aligned");
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
  if (groups.size() == 1 && groups[0].entries <= kClipFew && groups[0].chunks <= unsigned(kClipOne)) {
    ClipTable<kClipFew> t;
    fill(t, a, groups[0]);
    e = launch_clip_one(t, c, s);
    launches = 1;
  } else if (groups.empty()) {
    e = launch_clip_finish(c, s);
    launches = 1;
  } else {
    std::vector<Launch<kClipFew>> few(groups.size());
    std::vector<Launch<kClipTensors>> many(groups.size());
    for (int pass = 0; pass < (outs ? 2 : 1) && e == cudaSuccess; ++pass) {
      c.first = 0;
      for (size_t i = 0; i < groups.size() && e == cudaSuccess; ++i) {
        // the last gradients read are the first ones scaled
        const size_t at = pass ? groups.size() - 1 - i : i;
        const Group& g = groups[at];
        c.keep = outs && at + 1 == groups.size() && g.chunks > kKeep ? g.chunks - kKeep : 0;
        e = g.entries <= kClipFew ? few[at](a, g, c, pass, s) : many[at](a, g, c, pass, s);
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
