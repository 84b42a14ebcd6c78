// Host side of the gated block (ffn.h): argument checks, the plan of tiles and splits, and
// launches.  Its products are tiles of the head's kernel (head.h).
#include "ffn.h"

#include <algorithm>
#include <climits>
#include <initializer_list>

#include "engine.h"
#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

// Tile rows walked together keep about this much of A in the L2 cache (126 MB).
constexpr int64_t kGroupBytes = int64_t(32) << 20;
constexpr int64_t kTileM = kHeadPair * kHeadTileM;

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

#define FFN_CUDA(call, what)                                                      \
  do {                                                                            \
    const cudaError_t e_ = (call);                                                \
    if (e_ != cudaSuccess) {                                                      \
      cudaGetLastError();                                                         \
      return fail(err, std::string(what) + ": " + cudaGetErrorString(e_));        \
    }                                                                             \
  } while (0)

// ---- the plan -------------------------------------------------------------------

bool is_few(int dtype, int64_t rows, int64_t cols, int64_t width) {
  int64_t n = 1;
  while (n < rows) n *= 2;
  return rows <= (dtype == kF32 ? kFfnFewRowsF32 : kFfnFewRows) && n * ffn_pitch(std::max(cols, width)) * 4 <= kFfnFewSmem;
}

// The products of warps: all rows in place, 16 bytes at a time.
bool is_warps(const FfnArgs& a) {
  auto whole = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) | uintptr_t(ld) * 2) % 16 == 0; };
  const double products = double(a.rows) * double(a.width) * double(2 * a.cols + a.outs);
  if (a.rows < 2 || a.rows > kFfnWarpMost || (a.rows > kFfnWarpRows && products > kFfnWarpProducts)) return false;
  if (std::max(a.cols, a.width) > kFfnWarpLong) return false;
  return a.dtype == kBF16 && a.cols % 8 == 0 && a.width % 8 == 0 &&
         whole(a.x, a.ld_x) && whole(a.w_in, a.ld_in) && whole(a.w_out, a.ld_out) && whole(a.hidden, a.ld_hidden);
}

// bfloat16 sums of more terms than the tensor core may truncate in one place: epilogues that need
// all of a sum cannot have it, so the product goes to memory, in parts of K, and a launch follows.
bool is_long(int dtype, int64_t k) { return dtype == kBF16 && k > kFfnLong; }

bool is_narrow(int dtype, int64_t width, int64_t outs) {
  return dtype == kF32 && outs <= kFfnNarrow && outs * width <= kFfnNarrowValues;
}
// Rows that a warp of the narrow gradient adds up, one after the other: no more than 256, since the error of
// their float32 sum grows with them (dw_out of 500,000 rows x 2,048 that are all alike was 7e-5 off with
// 6,757), in whole rounds of the warps: 200,000 rows x 256 with 16 outputs 890 us with 256 rows, 780 with 169.
int64_t narrow_rows(int64_t rows, int64_t half) {
  const int64_t even = parts(rows, std::max<int64_t>(1, kFfnNarrowWarps / parts(half, 128)));
  return std::max<int64_t>(8, parts(even, parts(even, 256)));
}

// A product's tiles.
struct Shape {
  int64_t m, n, k;
  int tile_n, splits;
  int box;                           // rows of a K-major B that a CTA fetches
  int64_t tiles() const { return parts(m, kTileM) * parts(n, tile_n); }
  int64_t blocks() const { return parts(k, kHeadTileK); }
};
Shape shape(int64_t m, int64_t n, int64_t k) {
  const int tile = n <= 128 ? 128 : 256;
  return Shape{m, n, k, tile, 1, tile / kHeadPair};
}

// The first product: 128 gates and their factors a tile, or 64 where that ends sooner.  Narrow tiles
// cost six tenths of a wide one each (bfloat16: more bytes for what they compute).  Whole forward passes
// of 1,024 x 4,096 in us, 128 and 64 gates: bfloat16, 256 rows 34.9 and 32.9, 512 rows 39 and 43, 2,048
// rows 76 and 93; float32, 256 rows 124 and 109, 2,048 rows 318 and 296, 4,096 rows 562 and 577.
Shape gate_shape(int dtype, int64_t rows, int64_t width, int64_t cols) {
  auto rounds = [&](int64_t gates) { return double(parts(parts(rows, kTileM) * parts(width, gates), 74)); };
  const int gates = rounds(64) * (dtype == kF32 ? 0.55 : 0.6) < rounds(128) ? 64 : 128;
  return Shape{rows, width, cols, gates, 1, gates};
}

// Parts of K of one or two products of a launch: those that end first by an estimate, in steps
// of one K block (0.42 us for 256 columns).  A pair's time is the longest tile's, or its share
// of all steps and half a tile more; the sums of parts are written and read once more, at
// 6 TB/s.  Bounds of a part as in the head: no shorter than 8 blocks (float32: 2),
// bfloat16 no longer than 512.  `whole`: the second one's epilogue needs all of its sums
// (of 512 blocks at most there too: longer ones take a launch more, is_long).
void choose_splits(int dtype, Shape* a, Shape* b, bool whole = false) {
  constexpr int64_t kPairs = 74;
  const int64_t steps = dtype == kF32 ? 6 : 1, shortest = dtype == kF32 ? 2 : 8;
  auto least = [&](const Shape& q) { return dtype == kF32 ? int64_t(1) : parts(q.blocks(), 512); };
  auto most = [&](const Shape& q) { return std::max(least(q), std::min<int64_t>(q.blocks() / shortest, 32)); };
  auto tile = [&](const Shape& q, int64_t s) {
    return (double(parts(q.blocks(), s) * steps) + kHeadEpilogue) * q.tile_n / 256;
  };
  auto sums = [&](const Shape& q, int64_t s) {
    return s > 1 ? double(2 * s + 1) * double(q.m) * double(q.n) * 4 / 6e6 / 0.42 + 8 : 0.0;
  };
  double best = 0;
  const int64_t first = b && !whole ? least(*b) : 1, last = b && !whole ? most(*b) : 1;
  for (int64_t s = least(*a); s <= most(*a); ++s)
    for (int64_t t = first; t <= last; ++t) {
      const double ta = tile(*a, s), tb = b ? tile(*b, t) : 0;
      const int64_t na = a->tiles() * s, nb = b ? b->tiles() * t : 0;
      const double all = double(na) * ta + double(nb) * tb, longest = std::max(ta, tb);
      const double shortest_tile = nb ? std::min(ta, tb) : ta;
      double time = longest;
      if (na + nb > kPairs)
        time = nb ? std::max(longest, all / kPairs + shortest_tile / 2) : double(parts(na, kPairs)) * ta;
      time += sums(*a, s) + (b ? sums(*b, t) : 0);
      if (best == 0 || time < best) {
        best = time;
        a->splits = int(s);
        if (b) b->splits = int(t);
      }
    }
}

struct Plan {
  Shape y{}, gates{}, dh{}, dx{}, dw_in{}, dw_out{};  // gates: where cols are long
  // offsets into the workspace, 0 for none: packed operands, sums of parts of K
  int64_t x = 0, w_in = 0, w_out = 0, hidden = 0, dy = 0, dpre = 0, dh_at = 0, bytes = 0;
  int64_t part = 0, part_in = 0;     // y's, gates', dh's, dw_out's or dx's; dw_in's
  int64_t pre = 0;                   // where cols are long and no pre is kept
  int64_t half = 0;                  // columns of each half of dpre: width, up to a whole K block
};

struct Packed {
  bool x, w_in, w_out, hidden, dy;
};

Plan make_plan(int dtype, int64_t rows, int64_t cols, int64_t width, int64_t outs, bool grad, const Packed& pk) {
  Plan p{};
  const int64_t planes = dtype == kF32 ? 3 : 1;
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  auto packed = [&](int64_t r, int64_t c) { return take(planes * r * up(c, 8) * 2); };
  if (pk.x) p.x = packed(rows, cols);
  if (pk.w_in) p.w_in = packed(2 * width, cols);
  if (pk.w_out) p.w_out = packed(outs, width);
  if (pk.hidden) p.hidden = packed(rows, width);
  auto sums = [&](const Shape& q) { return q.splits > 1 ? q.splits * q.m * q.n * 4 : 0; };
  if (!grad) {
    p.y = shape(rows, outs, width);
    choose_splits(dtype, &p.y, nullptr);
    if (is_long(dtype, cols)) {
      p.gates = shape(rows, 2 * width, cols);
      choose_splits(dtype, &p.gates, nullptr);
      p.pre = take(rows * 2 * width * 4);
    }
    p.part = take(std::max(sums(p.y), sums(p.gates)));
  } else {
    if (pk.dy) p.dy = packed(rows, outs);
    p.half = up(width, kHeadTileK);
    p.dpre = take(planes * rows * 2 * p.half * 2);
    // dh in float32, where a launch of its own goes on with it
    const bool split = dtype == kF32 || is_long(dtype, outs);
    if (split) p.dh_at = take(rows * up(width, 4) * 4);
    p.dx = shape(rows, cols, 2 * p.half);
    p.dw_in = shape(p.half + width, cols, rows);
    p.dw_out = shape(outs, width, rows);
    choose_splits(dtype, &p.dx, &p.dw_in);
    p.dh = shape(rows, width, outs);
    if (split) {
      choose_splits(dtype, &p.dw_out, nullptr);
      if (dtype == kBF16) choose_splits(dtype, &p.dh, nullptr);
    } else {
      choose_splits(dtype, &p.dw_out, &p.dh, true);
    }
    // dh and dw_out are done before the others begin
    const int64_t chunks = is_narrow(dtype, width, outs) ? parts(rows, narrow_rows(rows, p.half)) : 0;
    p.part = take(std::max({sums(p.dh), sums(p.dw_out), sums(p.dx), chunks * outs * width * 4}));
    p.part_in = take(sums(p.dw_in));
  }
  p.bytes = at;
  return p;
}

// ---- checks ---------------------------------------------------------------------

int check_shape(int dtype, int64_t rows, int64_t cols, int64_t width, int64_t outs, std::string& err) {
  if (dtype != kF32 && dtype != kBF16)
    return fail(err, "the block takes dtype 0 (float32) or 1 (bfloat16), got " + std::to_string(dtype));
  if (rows < 0 || rows > (int64_t(1) << 30)) return fail(err, "rows must be in 0...2^30");
  if (cols < 1 || cols > (int64_t(1) << 20)) return fail(err, "cols must be in 1...2^20");
  if (width < 1 || width > (int64_t(1) << 20)) return fail(err, "width must be in 1...2^20");
  if (outs < 1 || outs > (int64_t(1) << 20)) return fail(err, "outs must be in 1...2^20");
  const int64_t tiles = parts(rows, kTileM) * parts(2 * std::max({cols, width, outs}), 128);
  if (tiles > INT_MAX) return fail(err, "rows * width are too many for one call");
  return 0;
}

int check_matrix(const char* name, const void* p, int64_t cols, int64_t ld, int dtype, std::string& err) {
  if (!p) return fail(err, "null argument");
  if (ld < cols) return fail(err, std::string(name) + " needs a stride of at least its columns");
  if (ld > (int64_t(1) << 31)) return fail(err, std::string(name) + " needs a stride of at most 2^31");
  if (!aligned(p, size_t(dtype_bytes(dtype))))
    return fail(err, std::string(name) + " must be aligned to its values");
  return 0;
}

int check(const FfnArgs& a, bool grad, std::string& err) {
  if (check_shape(a.dtype, a.rows, a.cols, a.width, a.outs, err)) return -1;
  if (a.act < kSilu || a.act > kGeluTanh)
    return fail(err, "unknown activation " + std::to_string(a.act) + " (0 silu, 1 gelu, 2 gelu_tanh)");
  if (a.rows > 0) {
    if (check_matrix("x", a.x, a.cols, a.ld_x, a.dtype, err) ||
        check_matrix("w_in", a.w_in, a.cols, a.ld_in, a.dtype, err) ||
        check_matrix("w_out", a.w_out, a.width, a.ld_out, a.dtype, err) ||
        check_matrix("hidden", a.hidden, a.width, a.ld_hidden, a.dtype, err))
      return -1;
    if ((grad || a.pre) && check_matrix("pre", a.pre, 2 * a.width, a.ld_pre, kF32, err)) return -1;
    if (!grad && check_matrix("y", a.y, a.outs, a.ld_y, a.dtype, err)) return -1;
    if (grad && check_matrix("dy", a.dy, a.outs, a.ld_dy, a.dtype, err)) return -1;
    if (grad && a.dx && check_matrix("dx", a.dx, a.cols, a.ld_dx, a.dtype, err)) return -1;
  }
  if (grad && a.dw_in && check_matrix("dw_in", a.dw_in, a.cols, a.ld_din, a.dtype, err)) return -1;
  if (grad && a.dw_out && check_matrix("dw_out", a.dw_out, a.width, a.ld_dout, a.dtype, err)) return -1;
  if (!aligned(a.workspace, 256)) return fail(err, "workspace must be 256-byte aligned");
  return 0;
}

int check_workspace(const FfnArgs& a, int64_t need, std::string& err) {
  if (a.workspace && a.workspace_bytes >= need) return 0;
  return fail(err, "workspace holds " + std::to_string(a.workspace ? a.workspace_bytes : 0) +
                       " bytes, the block needs " + std::to_string(need));
}

// ---- operands and products --------------------------------------------------------

// A matrix as the tiles read it: in place, or packed into the workspace.
struct Operand {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

struct Call {
  const FfnArgs& a;
  const Plan& p;
  cudaStream_t s;
  std::string& err;
  int64_t launches = 0;
  char* base() const { return static_cast<char*>(a.workspace); }
  int planes() const { return a.dtype == kF32 ? 3 : 1; }

  Operand operand(const void* src, int64_t rows, int64_t cols, int64_t ld, int64_t at, HeadPack* todo) const {
    Operand o{src, rows, cols, ld};
    if (at) {
      o.p = base() + at;
      o.ld = up(cols, 8);
      todo->src = src;
      todo->rows = rows;
      todo->cols = cols;
      todo->ld = ld;
      todo->dst = base() + at;
      todo->ldp = o.ld;
    }
    return o;
  }
  // Matrices that are to be packed, in one launch; `status`: it clears the status word as well.
  int pack(std::initializer_list<const HeadPack*> list, bool status) {
    unsigned* word = static_cast<unsigned*>(a.workspace);
    HeadPack todo[kHeadPacks];
    int count = 0;
    for (const HeadPack* q : list)
      if (q->src) todo[count++] = *q;
    if (count == 0) {
      if (status) FFN_CUDA(cudaMemsetAsync(word, 0, 4, s), "clearing the block's status word");
      return 0;
    }
    FFN_CUDA(launch_head_pack(a.dtype, todo, count, status ? word : nullptr, s), "pack launch");
    ++launches;
    return 0;
  }
  // C = A B^T along K; mn: the operand's rows are K, its columns C's rows (columns).
  int job(HeadJob& j, const Operand& A, bool a_mn, const Operand& B, bool b_mn, const Shape& h) {
    j.a_mn = a_mn;
    j.b_mn = b_mn;
    j.a_box = a_mn ? 64 : head_box_rows(A.rows, kHeadTileM);
    j.b_box = b_mn ? 64 : head_box_rows(h.n, h.box);
    if (head_encode(&j.a, A.p, A.cols, A.rows, A.ld, planes(), j.a_box, err) ||
        head_encode(&j.b, B.p, B.cols, B.rows, B.ld, planes(), j.b_box, err))
      return -1;
    j.tiles_m = int(parts(h.m, kTileM));
    j.tiles_n = int(parts(h.n, h.tile_n));
    j.kblocks = int(parts(h.k, kHeadTileK));
    j.splits = std::min(h.splits, j.kblocks);
    if (h.tiles() * j.splits > INT_MAX) return fail(err, "rows * width are too many for one call");
    j.M = int(h.m);
    j.N = int(h.n);
    // tile rows whose part of A stays in the L2 cache while the columns go by
    const int64_t bytes = kTileM * int64_t(j.kblocks / j.splits) * kHeadTileK * 2 * planes();
    j.group = int(std::max<int64_t>(1, std::min<int64_t>({kGroupBytes / std::max<int64_t>(bytes, 1), 16, j.tiles_m})));
    j.divide();
    return 0;
  }
  // Where a product goes, by way of sums of parts of K if it is split.
  void target(HeadJob& j, const Shape& h, void* out, int64_t ld, int64_t part, HeadReduce* red, int* reds) const {
    target(j, h, out, ld, a.dtype, part, red, reds);
  }
  void target(HeadJob& j, const Shape& h, void* out, int64_t ld, int dtype, int64_t part, HeadReduce* red,
              int* reds) const {
    j.out = out;
    j.ld_out = ld;
    j.out_f32 = dtype == kF32;
    j.wide = aligned(out, size_t(4 * dtype_bytes(dtype))) && ld % 4 == 0;
    if (!j.out_f32 && aligned(out, 16) && ld % 8 == 0) j.wide = 2;
    j.final = 1;
    if (j.splits > 1) {
      j.acc = reinterpret_cast<float*>(base() + part);
      j.final = 0;
      red[(*reds)++] = HeadReduce{j.acc, j.splits, h.m, h.n, nullptr, 0, 1, out, ld, j.out_f32,
                                  j.m_from, j.m_to};
    }
  }
  int products(int epilogue, HeadLaunch& l, int tile_n, const HeadReduce* red, int reds) {
    FFN_CUDA(launch_head(epilogue, tile_n, l, s), "block launch");
    for (int r = 0; r < reds; ++r) FFN_CUDA(launch_head_reduce(red[r], s), "block reduce launch");
    launches += 1 + reds;
    return 0;
  }
};

// What both gated epilogues know.
void gate(HeadGate& g, const FfnArgs& a) {
  g.act = a.act;
  g.width = int(a.width);
  g.rows = int(a.rows);
  g.hidden = a.hidden;
  g.ld_hidden = a.ld_hidden;
  g.pre = a.pre;
  g.ld_pre = a.ld_pre;
  g.wide = aligned(a.hidden, 16) && a.ld_hidden % (16 / dtype_bytes(a.dtype)) == 0;
  g.wide_pre = aligned(a.pre, 16) && a.ld_pre % 4 == 0 && a.width % 4 == 0;
}

Packed packed(const FfnArgs& a, bool grad) {
  auto no = [&](const void* p, int64_t ld) { return !head_in_place(a.dtype, p, ld); };
  return Packed{no(a.x, a.ld_x), no(a.w_in, a.ld_in), no(a.w_out, a.ld_out), no(a.hidden, a.ld_hidden),
                grad && no(a.dy, a.ld_dy)};
}

}  // namespace

int64_t ffn_workspace(int dtype, int64_t rows, int64_t cols, int64_t width, int64_t outs, bool grad,
                      bool strided) {
  std::string err;
  if (check_shape(dtype, rows, cols, width, outs, err)) return -1;
  auto pack = [&](int64_t c) { return dtype == kF32 || strided || c % 8 != 0; };
  const Packed pk{pack(cols), pack(cols), pack(width), pack(width), pack(outs)};
  const int64_t forward =
      is_few(dtype, rows, cols, width) ? 256 : make_plan(dtype, rows, cols, width, outs, false, pk).bytes;
  return grad ? std::max(forward, make_plan(dtype, std::max<int64_t>(rows, 1), cols, width, outs, true, pk).bytes)
              : forward;
}

int ffn_device(int device, const FfnArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, false, err)) return -1;
  if (a.rows == 0) return 0;
  const bool warps = is_warps(a);
  if (warps || is_few(a.dtype, a.rows, a.cols, a.width)) {
    if (check_workspace(a, 256, err)) return -1;
    if (use_device(device, err)) return -1;
    Guard gd(device);
    FFN_CUDA(warps ? launch_ffn_rows(a, s) : launch_ffn_few(a, s), "block launch");
    g_kernel_launches.fetch_add(2, std::memory_order_relaxed);
    return 0;
  }
  const Plan p = make_plan(a.dtype, a.rows, a.cols, a.width, a.outs, false, packed(a, false));
  if (check_workspace(a, p.bytes, err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  Call c{a, p, s, err};
  HeadPack px, pin, pout, ph;
  const Operand x = c.operand(a.x, a.rows, a.cols, a.ld_x, p.x, &px);
  const Operand w_in = c.operand(a.w_in, 2 * a.width, a.cols, a.ld_in, p.w_in, &pin);
  const Operand w_out = c.operand(a.w_out, a.outs, a.width, a.ld_out, p.w_out, &pout);
  const Operand h = c.operand(a.hidden, a.rows, a.width, a.ld_hidden, p.hidden, &ph);
  // w_out beside the others, for the second product
  const HeadPack none;
  const bool narrow = is_narrow(a.dtype, a.width, a.outs);
  if (c.pack({&px, &pin, narrow ? &none : &pout}, true)) return -1;

  // gates and factors: half of a tile's columns each
  const Shape in = is_long(a.dtype, a.cols) ? p.gates : gate_shape(a.dtype, a.rows, a.width, a.cols);
  HeadLaunch l{};
  head_settings(l, a.dtype, a.workspace);
  l.jobs = 1;
  if (c.job(l.job[0], x, false, w_in, false, in)) return -1;
  if (is_long(a.dtype, a.cols)) {
    float* pre = a.pre ? a.pre : reinterpret_cast<float*>(c.base() + p.pre);
    const int64_t ld = a.pre ? a.ld_pre : 2 * a.width;
    HeadReduce red[1]{};
    int reds = 0;
    c.target(l.job[0], in, pre, ld, kF32, p.part, red, &reds);
    if (c.products(kHeadBlock, l, in.tile_n, red, reds)) return -1;
    FFN_CUDA(launch_ffn_gate(a, pre, ld, s), "block launch");
  } else {
    gate(l.g, a);
    FFN_CUDA(launch_head(kHeadGate, 2 * in.tile_n, l, s), "block launch");
  }
  ++c.launches;

  if (narrow) {
    FFN_CUDA(launch_ffn_narrow(a, s), "block launch");
    g_kernel_launches.fetch_add(c.launches + 1, std::memory_order_relaxed);
    return 0;
  }
  if (c.pack({&ph}, false)) return -1;
  HeadLaunch q{};
  head_settings(q, a.dtype, a.workspace);
  q.jobs = 1;
  HeadReduce red[1]{};
  int reds = 0;
  if (c.job(q.job[0], h, false, w_out, false, p.y)) return -1;
  c.target(q.job[0], p.y, a.y, a.ld_y, p.part, red, &reds);
  if (c.products(kHeadBlock, q, p.y.tile_n, red, reds)) return -1;
  g_kernel_launches.fetch_add(c.launches, std::memory_order_relaxed);
  return 0;
}

int ffn_grad_device(int device, const FfnArgs& a, cudaStream_t s, std::string& err) {
  if (check(a, true, err)) return -1;
  if (!a.dx && !a.dw_in && !a.dw_out) return 0;
  if (a.rows == 0) {
    if (!a.dw_in && !a.dw_out) return 0;
    if (use_device(device, err)) return -1;
    Guard gd(device);
    const size_t size = size_t(dtype_bytes(a.dtype));
    if (a.dw_in)
      FFN_CUDA(cudaMemset2DAsync(a.dw_in, size_t(a.ld_din) * size, 0, size_t(a.cols) * size, size_t(2 * a.width), s),
               "clearing dw_in");
    if (a.dw_out)
      FFN_CUDA(cudaMemset2DAsync(a.dw_out, size_t(a.ld_dout) * size, 0, size_t(a.width) * size, size_t(a.outs), s),
               "clearing dw_out");
    return 0;
  }
  const Plan p = make_plan(a.dtype, a.rows, a.cols, a.width, a.outs, true, packed(a, true));
  if (check_workspace(a, p.bytes, err)) return -1;
  if (use_device(device, err)) return -1;
  Guard gd(device);
  Call c{a, p, s, err};
  HeadPack px, pin, pout, ph, pdy;
  const Operand x = c.operand(a.x, a.rows, a.cols, a.ld_x, p.x, &px);
  const Operand w_in = c.operand(a.w_in, 2 * a.width, a.cols, a.ld_in, p.w_in, &pin);
  const Operand w_out = c.operand(a.w_out, a.outs, a.width, a.ld_out, p.w_out, &pout);
  const Operand h = c.operand(a.hidden, a.rows, a.width, a.ld_hidden, p.hidden, &ph);
  const Operand dy = c.operand(a.dy, a.rows, a.outs, a.ld_dy, p.dy, &pdy);
  const Operand d{c.base() + p.dpre, a.rows, 2 * p.half, 2 * p.half};
  const bool f32 = a.dtype == kF32, inner = a.dx || a.dw_in;
  // h with the others, unless a launch of its own makes its planes
  const HeadPack none;
  const bool narrow = is_narrow(a.dtype, a.width, a.outs);
  const bool split = inner && (f32 || is_long(a.dtype, a.outs)) && !narrow;
  if (c.pack({narrow ? &none : &pdy, inner && !narrow ? &pout : &none, a.dw_out && !(f32 && split) && !narrow ? &ph : &none,
              inner ? &px : &none, a.dx ? &pin : &none}, false))
    return -1;
  if (narrow) {  // dh, dpre and dw_out at once
    FfnNarrow t{};
    t.act = a.act;
    t.outs = int(a.outs);
    t.rows = a.rows;
    t.per = narrow_rows(a.rows, p.half);
    t.width = int(a.width);
    t.half = int(p.half);
    t.dy = static_cast<const float*>(a.dy);
    t.ld_dy = a.ld_dy;
    t.w = static_cast<const float*>(a.w_out);
    t.ld_w = a.ld_out;
    t.pre = a.pre;
    t.ld_pre = a.ld_pre;
    t.hidden = static_cast<const float*>(a.hidden);
    t.ld_hidden = a.ld_hidden;
    t.dpre = inner ? c.base() + p.dpre : nullptr;
    t.part = a.dw_out ? reinterpret_cast<float*>(c.base() + p.part) : nullptr;
    FFN_CUDA(launch_ffn_narrow_grad(t, s), "block gradient launch");
    ++c.launches;
    if (a.dw_out) {
      const int chunks = int(parts(a.rows, t.per));
      FFN_CUDA(launch_head_reduce(HeadReduce{t.part, chunks, a.outs, a.width, nullptr, 0, 1, a.dw_out, a.ld_dout, 1, 0, 0}, s),
               "block reduce launch");
      ++c.launches;
    }
  }
  // dh = dy w_out; its epilogue (float32, and long sums: a launch) makes the gradients of gates and factors of it
  Shape dh{a.rows, a.width, a.outs, kHeadTileN, 1, 0};
  if (split && !f32) dh.splits = p.dh.splits;
  if (split) {
    HeadLaunch q{};
    head_settings(q, a.dtype, a.workspace);
    q.jobs = 1;
    if (c.job(q.job[0], dy, false, w_out, true, dh)) return -1;
    FfnSplit t{};
    t.dtype = a.dtype;
    t.act = a.act;
    t.rows = a.rows;
    t.width = int(a.width);
    t.half = int(p.half);
    t.ld_h = int(up(a.width, 8));
    t.dh = reinterpret_cast<const float*>(c.base() + p.dh_at);
    t.ld_dh = up(a.width, 4);
    t.pre = a.pre;
    t.ld_pre = a.ld_pre;
    t.hidden = static_cast<const float*>(a.hidden);
    t.ld_hidden = a.ld_hidden;
    t.dpre = c.base() + p.dpre;
    t.h = f32 && a.dw_out ? c.base() + p.hidden : nullptr;
    HeadReduce red[1]{};
    int reds = 0;
    c.target(q.job[0], dh, c.base() + p.dh_at, t.ld_dh, kF32, p.part, red, &reds);
    if (c.products(kHeadBlock, q, kHeadTileN, red, reds)) return -1;
    FFN_CUDA(launch_ffn_split(t, s), "block split launch");
    ++c.launches;
  }
  const bool with = inner && !f32 && !split;
  if ((a.dw_out && !narrow) || with) {
    // dw_out = dy^T h: in bfloat16 in one launch with dh, whose epilogue takes longer than its products
    HeadLaunch q{};
    head_settings(q, a.dtype, a.workspace);
    HeadReduce red[1]{};
    int reds = 0;
    if (a.dw_out) {
      HeadJob& j = q.job[q.jobs++];
      if (c.job(j, dy, true, h, true, p.dw_out)) return -1;
      c.target(j, p.dw_out, a.dw_out, a.ld_dout, p.part, red, &reds);
      j.plain = 1;
    }
    if (with) {
      if (c.job(q.job[q.jobs++], dy, false, w_out, true, dh)) return -1;
      gate(q.g, a);
      q.g.dpre = const_cast<void*>(d.p);
      q.g.ld_d = 2 * p.half;
      q.g.half = int(p.half);
    }
    // tiles of one launch are of one width
    const int tile = with ? kHeadTileN : p.dw_out.tile_n;
    if (a.dw_out && tile != p.dw_out.tile_n) {
      q.job[0].tiles_n = int(parts(p.dw_out.n, tile));
      q.job[0].divide();
    }
    if (c.products(with ? kHeadGateGrad : kHeadBlock, q, tile, red, reds)) return -1;
  }
  if (inner) {
    HeadLaunch q{};
    head_settings(q, a.dtype, a.workspace);
    HeadReduce red[2]{};
    int reds = 0;
    HeadJob dx{}, dw{};
    const int gap = int(p.half - a.width);
    if (a.dx) {  // dx = dpre w_in
      if (c.job(dx, d, false, w_in, true, p.dx)) return -1;
      dx.b_from = int(p.half);
      dx.b_skip = gap;
      c.target(dx, p.dx, a.dx, a.ld_dx, p.part, red, &reds);
    }
    if (a.dw_in) {  // dw_in = dpre^T x
      if (c.job(dw, d, true, x, true, p.dw_in)) return -1;
      dw.m_from = int(a.width);
      dw.m_to = int(p.half);
      c.target(dw, p.dw_in, a.dw_in, a.ld_din, p.part_in, red, &reds);
    }
    // the heavier tiles first
    const bool dw_first = !a.dx || (a.dw_in && dw.kblocks / dw.splits > dx.kblocks / dx.splits);
    q.jobs = a.dx && a.dw_in ? 2 : 1;
    q.job[0] = dw_first ? dw : dx;
    if (q.jobs == 2) q.job[1] = dw_first ? dx : dw;
    if (c.products(kHeadBlock, q, p.dx.tile_n, red, reds)) return -1;
  }
  g_kernel_launches.fetch_add(c.launches, std::memory_order_relaxed);
  return 0;
}

int ffn_check_device(int device, const void* workspace, std::string& err) {
  if (!workspace) return fail(err, "null argument");
  if (use_device(device, err)) return -1;
  Guard gd(device);
  FFN_CUDA(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
  unsigned word = 0;
  FFN_CUDA(cudaMemcpy(&word, workspace, 4, cudaMemcpyDeviceToHost), "reading the block's status word");
  if (word == kHeadExpired)
    return fail(err, "device " + std::to_string(device) +
                         ": feed-forward kernel gave up waiting for a shared-memory transfer");
  return 0;
}

}  // namespace mb
