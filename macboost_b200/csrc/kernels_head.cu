// Kernels of the softmax head (head.h): matrix products on the 5th-generation tensor
// cores whose epilogues reduce, form or store what the head needs.
//
// head_kernel: a persistent kernel, a pair of CTAs a 256 x 256 tile (tcgen05.mma,
// cta_group::2: each CTA holds 128 rows of A and half of B in shared memory and 128 x
// 256 float32 sums in its tensor memory).  Warp 0 fetches 128-byte swizzled tiles with
// TMA into a ring, warp 1 of the first CTA issues the products, warps 4 to 11 take the
// sums out of tensor memory, 32 rows and half the columns each, while the next tile
// fills the second half of it.
//
// A float32 operand is three planes of bfloat16, x = x1 + x2 + x3 with 8 bits each, and
// the product the six terms x_i y_j with i + j <= 4 -- what is dropped is below 2^-24
// of |x||y|.  The tensor core's sums are truncated to 32 bits at every step, so they run
// over one block of 64 of K only, the smallest terms first (they cost little while the sum
// is small), and the epilogue adds the blocks up in registers, rounded to nearest.  With
// whole sums in the tensor core, dh of 26 x 12 x 7,798 was off by 2.5e-6.  A stage of the
// ring holds all three planes of both operands, so a block of K is fetched once for its
// six products.  Logits that infinities took part in are formed again (redo_logits).
// bfloat16 sums stay in the tensor core: logits over all columns, the gradients over parts of
// 2,048 steps (splits_for in head.cpp).
//
// Measured without other load: the loss of 8,192 x 1,024 x 131,072 bfloat16 1,633 us (1.35
// PFLOP/s), g of 16,384 classes 213 us, dh and dw of them 473 us; paced by the copies into
// shared memory (alone they take 88% of the time, three stages are as fast as six; the tensor
// pipe is active for 62, 60 and 55% of the cycles), in a loop by the power cap.  float32, 2,048
// x 1,024 x 32,768: loss 595 us (0.50 ms of bfloat16 products at the measured peak), with
// gradient 2.65 ms.
//
// The gated block's products are tiles of the same kernel: kHeadGate's second CTA holds rows of the
// factors in place of B's second half, so that an epilogue has gates and factors of the same
// columns, kHeadGateGrad forms both gradients of a tile of dh.  Bound by the copies into shared
// memory and by the epilogues' traffic: 8,192 x 1,024 x 4,096 bfloat16 gates 130 us (268 MB of pre and 67
// of h written; tensor pipe 55%), y 69, dh and dw_out 207 (268 MB of pre read; 31%), dx and dw_in 297;
// 2,048 x 1,024 x 4,096 float32 164, 88, 94 and 88, 329 (54 to 66%).
//
// Every wait ends after wait_ns: the CTA then marks itself dead, sets the status word,
// waits (as long again at most) for its copies and products in flight and returns (its
// results are void).
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "activation.cuh"
#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int kEpilogueWarps = 8;
constexpr int kHeadThreads = 128 + kEpilogueWarps * 32;  // three warpgroups

// ---- PTX ------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// Arrive at the barrier of CTA `rank` of the cluster that lies where `bar` does here.
__device__ __forceinline__ void bar_arrive_at(uint32_t bar, uint32_t rank) {
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n"
      " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(bar),
      "r"(rank)
      : "memory");
}
// Without .acquire.cluster, which would make every wait a memory barrier: what the waits
// order is the asynchronous copies, the products and tensor memory, by the rules of
// mbarrier transactions, tcgen05.commit and the tcgen05 fences.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

struct Wait {
  volatile uint32_t* dead;  // shared: some wait of this CTA ran out
  unsigned* status;
  unsigned long long limit;
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    if (bar_try(bar, parity)) return true;
    const uint64_t t0 = now_ns();
    while (!*dead) {
      if (bar_try(bar, parity)) return true;
      if (now_ns() - t0 > limit) {
        *dead = 1;
        atomicExch(status, kHeadExpired);
      }
    }
    return false;
  }
  // Until the barrier's phase is over or `limit` after t0, whatever happened before: for
  // what is in flight when a CTA gives up.
  __device__ __forceinline__ void settle(uint32_t bar, uint32_t parity, uint64_t t0) const {
    while (!bar_try(bar, parity) && now_ns() - t0 <= limit) {
    }
  }
};

// The first CTA's barrier at the same offset: the pair's bit of a cluster address cleared.
constexpr uint32_t kFirstOfPair = 0xFEFFFFFFu;

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar & kFirstOfPair)
      : "memory");
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
// The products issued so far, when done, arrive at this barrier of both CTAs (the multicast
// is of the arrival; no copy is).
__device__ __forceinline__ void commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
__device__ __forceinline__ void commit_here(uint32_t bar) {  // at this CTA's barrier alone
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

// 32 lanes x 32 columns of tensor memory: column c of lane i to v[c] of thread i, which
// are not there before tmem_wait.
__device__ __forceinline__ void tmem_issue(uint32_t addr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
        "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
        "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// 32 lanes x 16 columns, with the wait: one statement, since the values may not be read (or
// moved to other registers) before the wait, and two would leave that to the compiler.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}

// 16 values of each thread to 32 lanes x 16 columns, there after tmem_stored.
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_stored() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle.  K-major: rows of 64 K values,
// groups of 8 rows 1,024 bytes apart.  M/N-major: boxes of 64 (M or N) x 64 (K), 8,192
// bytes apart; inside one, groups of 8 K rows 1,024 bytes apart.
__device__ __forceinline__ uint64_t descriptor(uint32_t addr, bool mn) {
  const uint64_t lead = mn ? 8192 / 16 : 1;
  return uint64_t((addr >> 4) & 0x3FFF) | (lead << 16) | (uint64_t(1024 / 16) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// ---- tiles ----------------------------------------------------------------------

struct Tile {
  int job, m, n, split;
};

// The tiles of a pair, in order.  Two jobs: the first one's tiles go round first; the
// pairs left with one fewer take as many of the second job's as weigh the same, and the
// rest go round again, so that pairs end together.
struct Walk {
  const HeadLaunch& a;
  int pairs, me, step = 0;
  int count[2], extra, light, bonus;
  // a tile's time in steps of one K block
  __device__ int weight(const HeadJob& q) const {
    return (q.kblocks + q.splits - 1) / q.splits * (a.f32 ? 6 : 1) + kHeadEpilogue;
  }
  __device__ Walk(const HeadLaunch& l) : a(l) {
    pairs = int(gridDim.x) / kHeadPair;
    me = int(blockIdx.x) / kHeadPair;
    for (int j = 0; j < 2; ++j)
      count[j] = j < a.jobs ? a.job[j].tiles_m * a.job[j].tiles_n * a.job[j].splits : 0;
    light = count[0] % pairs;  // pairs from here on have one tile of job 0 fewer
    extra = 0;
    if (a.jobs > 1 && light > 0) {
      const int c0 = weight(a.job[0]), c1 = weight(a.job[1]);
      extra = (c0 + c1 / 2) / c1;
      const int most = count[1] / (pairs - light);
      if (extra > most) extra = most;
    }
    bonus = extra * (pairs - light);
  }
  __device__ bool next(Tile* t) {
    int i = me + step * pairs;
    int job = 0;
    if (i >= count[0]) {
      if (a.jobs < 2) return false;
      job = 1;
      int past = step - (count[0] / pairs + (me < light ? 1 : 0));
      if (me >= light && past < extra) {
        i = (me - light) * extra + past;
      } else {
        if (me >= light) past -= extra;
        i = bonus + past * pairs + (me >= light ? me - light : me + pairs - light);
        if (i >= count[1]) return false;
      }
    }
    ++step;
    const HeadJob& q = a.job[job];
    t->job = job;
    t->split = 0;
    if (q.splits > 1) {
      t->split = q.by_split(i);
      i -= t->split * q.tiles_m * q.tiles_n;
    }
    // groups of tile rows, all columns of a group before the next group
    const int g = q.by_group(i);
    i -= g * q.group * q.tiles_n;
    const int rows = min(q.group, q.tiles_m - g * q.group);
    t->n = rows == q.group ? q.by_rows(i) : q.by_last(i);
    t->m = g * q.group + i - t->n * rows;
    return true;
  }
  // K blocks of a tile
  __device__ void blocks(const Tile& t, int* k0, int* k1) const {
    const HeadJob& q = a.job[t.job];
    *k0 = t.split * q.part + min(t.split, q.longer);
    *k1 = *k0 + q.part + (t.split < q.longer ? 1 : 0);
  }
};

// ---- epilogues ------------------------------------------------------------------

// Running maximum and sum of exp(x - max), of 32 more columns of which `n` exist.  Four
// chains each: two warps a scheduler do not hide a chain of 32.
__device__ __forceinline__ void online(const float (&v)[32], int n, float& m, float& s) {
  float t[4] = {m, -INFINITY, -INFINITY, -INFINITY};
  if (n >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) t[i % 4] = fmaxf(t[i % 4], v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) t[i % 4] = fmaxf(t[i % 4], v[i]);
  }
  const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
  // an infinite maximum would make inf - inf of itself: such a row's sum is formed
  // around 0 and comes out inf, or stays 0 for -inf (NaN is kept either way)
  const float base = fabsf(top) == INFINITY ? 0.f : top;
  const float old = fabsf(m) == INFINITY ? 0.f : m;
  float sum[4] = {s == 0.f ? 0.f : s * exp2_approx((old - base) * kLog2e), 0.f, 0.f, 0.f};
  const float b2 = base * kLog2e;
  if (n >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i % 4] += exp2_approx(fmaf(v[i], kLog2e, -b2));
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) sum[i % 4] += exp2_approx(fmaf(v[i], kLog2e, -b2));
  }
  m = top;
  s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// float32 logits that are not finite, formed again from the inputs.  The planes of an
// infinity are (inf, 0, 0), so the products of planes hold 0 x inf and sums of both signs: NaN,
// where a class that is switched off has -inf.  They are never finite, so what to form again
// shows in the result: a sum over the columns for each such logit of this lane's row, one
// class after the other, w read by all lanes at once.  A row of h that holds NaN is left as it
// is.  A function of its own, called once a tile, so that it takes no registers from the
// sums: inline for each 32 columns the loss was 20% slower.
template <int N>
__device__ __noinline__ void redo_logits(float* v, int n, bool mine, const HeadRows& r, int row,
                                         int first) {
  const float* h = r.h + (mine ? row * r.ld_h : 0);
  int row_nan = -1;                      // not yet known
  for (int i = 0; i < N; ++i) {
    const float old = v[i];
    const bool here = mine && i < n && !(fabsf(old) < INFINITY);
    if (here && row_nan < 0) {
      row_nan = 0;
      for (int k = 0; k < r.cols && !row_nan; ++k) row_nan = isnan(h[k]);
    }
    if (!here || row_nan) continue;
    const float* w = r.w + (first + i) * r.ld_w;
    float x = 0.f;
    for (int k0 = 0; k0 < r.cols && !isnan(x); k0 += 32) {
      const int k1 = min(k0 + 32, r.cols);
#pragma unroll 8
      for (int k = k0; k < k1; ++k) x = fmaf(h[k], w[k], x);
    }
    v[i] = x;
  }
}
// N of them, of which `n` exist: those of this lane's row, if it is `mine`.
template <int N>
__device__ __forceinline__ void redo(float (&v)[N], int n, bool mine, const HeadRows& r, int row, int first) {
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) t[i % 4] = fmaf(v[i], 0.f, t[i % 4]);
  const float all = (t[0] + t[1]) + (t[2] + t[3]);
  if (!__any_sync(~0u, mine && all != all)) return;
  float u[N];
#pragma unroll
  for (int i = 0; i < N; ++i) u[i] = v[i];
  redo_logits<N>(u, n, mine, r, row, first);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = u[i];
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// A warp's 32 rows x 32 columns, a row a lane, to four rows at a time with eight lanes a
// row: f(row, column, four values) then reads and writes global memory in whole sectors.
// A row of the 4 KB buffer is eight 16-byte units, at positions permuted by the row, so
// that both directions are free of bank conflicts.
constexpr int kTurnBytes = 32 * 32 * 4;
template <class F>
__device__ __forceinline__ void turn(uint32_t buf, const float (&v)[32], int lane, F f) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 8; ++u)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128 + ((u ^ (lane & 7)) << 4)),
                 "f"(v[4 * u]), "f"(v[4 * u + 1]), "f"(v[4 * u + 2]), "f"(v[4 * u + 3])
                 : "memory");
  __syncwarp();
#pragma unroll 2
  for (int i = 0; i < 8; ++i) {
    const int row = i * 4 + lane / 8, u = lane % 8;
    float4 x;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(buf + row * 128 + ((u ^ (row & 7)) << 4)));
    f(row, 4 * u, x);
  }
}

// The same, a row at a time with a lane a column, f(row, column, value): what does not start on
// 16 bytes is read and written side by side all the same.
template <class F>
__device__ __forceinline__ void turn1(uint32_t buf, const float (&v)[32], int lane, F f) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 8; ++u)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128 + ((u ^ (lane & 7)) << 4)),
                 "f"(v[4 * u]), "f"(v[4 * u + 1]), "f"(v[4 * u + 2]), "f"(v[4 * u + 3])
                 : "memory");
  __syncwarp();
#pragma unroll 4
  for (int row = 0; row < 32; ++row) {
    float x;
    asm volatile("ld.shared.f32 %0, [%1];"
                 : "=f"(x)
                 : "r"(buf + row * 128 + (((lane / 4) ^ (row & 7)) << 4) + lane % 4 * 4));
    f(row, lane, x);
  }
}

// The same in bfloat16: eight rows at a time with four lanes a row, 16 bytes each.
template <class F>
__device__ __forceinline__ void turn_bf16(uint32_t buf, const float (&v)[32], int lane, F f) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 64 +
                                                                  ((u ^ ((lane >> 1) & 3)) << 4)),
                 "r"(pack2(v[8 * u], v[8 * u + 1])), "r"(pack2(v[8 * u + 2], v[8 * u + 3])),
                 "r"(pack2(v[8 * u + 4], v[8 * u + 5])), "r"(pack2(v[8 * u + 6], v[8 * u + 7]))
                 : "memory");
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + lane / 4, u = lane % 4;
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(buf + row * 64 + ((u ^ ((row >> 1) & 3)) << 4)));
    f(row, 8 * u, x);
  }
}

// Four adjacent values to memory; `n` of them exist, `wide`: p is aligned for all four.
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x, int n, bool wide) {
  if (wide && n >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
  } else {
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = __float2bfloat16_rn(v[i]);
  }
}
__device__ __forceinline__ void store4(float* p, float4 x, int n, bool wide) {
  if (wide && n >= 4) {
    *reinterpret_cast<float4*>(p) = x;
  } else {
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}

// Eight adjacent bfloat16.
__device__ __forceinline__ void store8(__nv_bfloat16* p, uint4 x, int n, bool wide) {
  if (wide && n >= 8) {
    *reinterpret_cast<uint4*>(p) = x;
  } else {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = __ushort_as_bfloat16(static_cast<unsigned short>(u[i / 2] >> (16 * (i % 2))));
  }
}
__device__ __forceinline__ float4 load4(const float* p, int n, bool wide) {
  if (wide && n >= 4) return *reinterpret_cast<const float4*>(p);
  return make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
}

// 16 columns of gates and 16 of their factors, a row a lane, to rows of 32 floats (the gates
// first) in the warp's buffer.  A row is eight 16-byte units, at positions permuted so that
// two neighbouring rows' gates, read by eight lanes, have banks of their own.
__device__ __forceinline__ uint32_t pair_unit(uint32_t buf, int row, int unit) {
  return buf + row * 128 + ((unit ^ ((row & 1) << 2 | (row >> 1 & 3))) << 4);
}
__device__ __forceinline__ void put_pairs(uint32_t buf, const float (&v)[16], const float (&w)[16], int lane) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float* x = u < 4 ? v + 4 * u : w + 4 * (u - 4);
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(pair_unit(buf, lane, u)), "f"(x[0]), "f"(x[1]),
                 "f"(x[2]), "f"(x[3])
                 : "memory");
  }
  __syncwarp();
}
__device__ __forceinline__ void read4(uint32_t at, float (&x)[4]) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
               : "r"(at));
}
__device__ __forceinline__ float read1(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at));
  return x;
}
__device__ __forceinline__ float4 four(const float (&x)[4]) { return make_float4(x[0], x[1], x[2], x[3]); }

template <int EPI, int TN, bool F32>
__global__ void __cluster_dims__(kHeadPair, 1, 1) __launch_bounds__(kHeadThreads, 1)
    head_kernel(const __grid_constant__ HeadLaunch a) {
  constexpr int kPlanes = F32 ? 3 : 1;
  constexpr int kBytesA = kHeadTileM * 128;           // of a plane
  constexpr int kBytesB = TN / kHeadPair * 128;
  constexpr int kStage = kPlanes * (kBytesA + kBytesB);
  constexpr int kStages = (192 * 1024) / kStage;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t dead_flag;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages;
  const uint32_t sums_full = empty + 8 * kStages, sums_empty = sums_full + 16;
  const uint32_t settled = sums_empty + 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  const Wait wait{&dead_flag, a.status, a.wait_ns};

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(sums_full + 8 * i, 1);
      bar_init(sums_empty + 8 * i, kHeadPair * kEpilogueWarps);
    }
    bar_init(settled, 1);
    dead_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(2 * TN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  // products of planes, small ones first; a single plane is the last of them
  constexpr int kPlaneA[6] = {2, 1, 0, 1, 0, 0};
  constexpr int kPlaneB[6] = {0, 1, 2, 0, 1, 0};

  // float32: the epilogue keeps 128 sums a thread.  384 threads are launched with 168
  // registers each (64,512); the first warpgroup keeps 56 a thread and the other two get
  // 224: 128 x 56 + 256 x 224 = 64,512.
  if (warp < 4) {
    if constexpr (F32) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0) {
        Walk walk(a);
        Tile t;
        int s = 0, ph = 0;
        bool ok = true;
        while (ok && walk.next(&t)) {
          const HeadJob& q = a.job[t.job];
          int k0, k1;
          walk.blocks(t, &k0, &k1);
          const int am = (t.m * kHeadPair + int(rank)) * kHeadTileM;
          // a gated product: the first CTA's half of B are gate rows, the second's the rows
          // `width` below, so the tile's columns are 128 gates and their 128 factors
          const int bn = EPI == kHeadGate ? t.n * (TN / 2) + int(rank) * a.g.width
                                          : t.n * TN + int(rank) * (TN / kHeadPair);
          // Boxes that lie outside the matrix are not fetched (what the shared memory holds
          // there only reaches sums that are not used): a box that TMA has to fill with
          // zeros is slower than one it reads.
          auto bytes_a = [&](int m0) {
            return q.a_mn ? min(kHeadTileM / 64, max(0, (q.M - m0 + 63) / 64)) * 8192
                          : m0 < q.M ? q.a_box * 128 : 0;
          };
          auto bytes_b = [&](int n0) {
            return q.b_mn ? min(TN / kHeadPair / 64, max(0, (q.N - n0 + 63) / 64)) * 8192
                          : EPI == kHeadGate || n0 < q.N ? q.b_box * 128 : 0;
          };
          // (read from the job at every block, and in every form of the kernel, the gap cost the head's tiles 2 to 4%)
          const int b_k0 = q.b_k0, gap = q.b_from / kHeadTileK, skip = q.b_skip;
          const int m0 = t.m * kHeadPair * kHeadTileM, n0 = t.n * TN;
          const uint32_t bytes = kPlanes * uint32_t(bytes_a(m0) + bytes_a(m0 + kHeadTileM) + bytes_b(n0) +
                                          bytes_b(n0 + TN / kHeadPair));
          for (int kb = k0; kb < k1; ++kb) {
            ok = wait(empty + 8 * s, ph ^ 1);
            if (!ok) break;
            if (rank == 0) bar_expect(full + 8 * s, bytes);
            const uint32_t bar = full + 8 * s;
            uint32_t sa = ring + s * kStage, sb = sa + kPlanes * kBytesA;
            if (++s == kStages) {
              s = 0;
              ph ^= 1;
            }
            if (a.stall) continue;
            const int ka = q.a_k0 + kb * kHeadTileK;
            const int kk = b_k0 + kb * kHeadTileK - (EPI == kHeadBlock && kb >= gap ? skip : 0);
            for (int z = 0; z < kPlanes; ++z, sa += kBytesA, sb += kBytesB) {
              if (q.a_mn) {
#pragma unroll
                for (int j = 0; j < kHeadTileM / 64; ++j)
                  if (am + 64 * j < q.M) tma_load(sa + j * 8192, &q.a, q.a_row0 + am + 64 * j, ka, z, bar);
              } else if (am < q.M) {
                tma_load(sa, &q.a, ka, q.a_row0 + am, z, bar);
              }
              if (q.b_mn) {
#pragma unroll
                for (int j = 0; j < TN / kHeadPair / 64; ++j)
                  if (bn + 64 * j < q.N) tma_load(sb + j * 8192, &q.b, q.b_row0 + bn + 64 * j, kk, z, bar);
              } else if (EPI == kHeadGate || bn < q.N) {
                tma_load(sb, &q.b, kk, q.b_row0 + bn, z, bar);
              }
            }
          }
        }
        // The copies in flight land before the shared memory is given up: every stage's last
        // copies, of both CTAs, complete the first CTA's barrier, and the second leaves with
        // the first.  Without an expired wait that is a matter of a microsecond.  A step
        // that the second CTA alone had begun when the first gave up has no barrier of its
        // own; it gets 2 ms.
        const uint64_t t0 = now_ns();
        if (rank == 0)
          for (int i = 0; i < kStages; ++i) wait.settle(full + 8 * i, i < s ? ph : ph ^ 1, t0);
        if (!ok)
          while (now_ns() - t0 < 2000000) {
          }
      }
    } else if (warp == 1) {
      if (rank == 0 && lane == 0) {
        Walk walk(a);
        Tile t;
        int s = 0, ph = 0, as = 0, aph = 0;
        bool ok = true;
        while (ok && walk.next(&t)) {
          const HeadJob& q = a.job[t.job];
          int k0, k1;
          walk.blocks(t, &k0, &k1);
          // float32 sums of bfloat16, M 256 (both CTAs), N TN
          const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(q.a_mn) << 15) |
                                 (uint32_t(q.b_mn) << 16) | (uint32_t(TN / 8) << 17) |
                                 (uint32_t(kHeadPair * kHeadTileM / 16) << 24);
          const uint32_t step_a = q.a_mn ? 2048 / 16 : 32 / 16, step_b = q.b_mn ? 2048 / 16 : 32 / 16;
          for (int c0 = k0; ok && c0 < k1; c0 += F32 ? 1 : k1 - k0) {
            ok = wait(sums_empty + 8 * as, aph ^ 1);
            if (!ok) break;
            fence_after();
            bool add = false;
            for (int i = 0; i < (F32 ? 1 : k1 - k0); ++i) {
              ok = wait(full + 8 * s, ph);
              if (!ok) break;
              fence_after();
              const uint32_t sa = ring + s * kStage, sb = sa + kPlanes * kBytesA;
#pragma unroll
              for (int p = F32 ? 0 : 5; p < 6; ++p) {
                const uint64_t da = descriptor(sa + (F32 ? kPlaneA[p] : 0) * kBytesA, q.a_mn);
                const uint64_t db = descriptor(sb + (F32 ? kPlaneB[p] : 0) * kBytesB, q.b_mn);
#pragma unroll
                for (int k = 0; k < kHeadTileK / 16; ++k) {
                  mma(tmem + as * TN, da + k * step_a, db + k * step_b, idesc, add);
                  add = true;
                }
              }
              commit_both(empty + 8 * s);
              if (++s == kStages) {
                s = 0;
                ph ^= 1;
              }
            }
            if (ok) commit_both(sums_full + 8 * as);
            as ^= 1;
            if (as == 0) aph ^= 1;
          }
        }
        if (!ok) {  // the products in flight read the shared memory of both CTAs
          commit_here(settled);
          wait.settle(settled, 0, now_ns());
        }
      }
    }
  } else {
    if constexpr (F32) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    Walk walk(a);
    Tile t;
    int as = 0, aph = 0;
    const int quarter = warp % 4, half = warp / 4 - 1;
    const HeadRows& r = a.r;
    const uint32_t stage = ring + kStages * kStage + (warp - 4) * kTurnBytes;
    // this thread's row of the tile's half: chunks of sums added up (float32)
    float sums[F32 ? TN / 2 : 1];
    // float32 sums go back to tensor memory, and from there the way of bfloat16's: an epilogue
    // unrolled over 128 registers runs at the speed of instruction fetches (25 us a tile)
    constexpr bool kBack = F32 && (EPI == kHeadOut || EPI == kHeadBlock || EPI == kHeadGate);
    // A gated block's products: rows that move up, and rows side by side whatever their alignment.  The head's
    // are a form of their own without that: in one form with it they took 1.5 to 2 us longer a launch
    // (2,048 x 512 x 1,000 dh and dw 15.6, in one form 18.0, now 16.2; 1,000 x 100 x 403 11.9, 13.4, 12.2).
    constexpr bool kBlock = EPI != kHeadOut;
    while (walk.next(&t)) {
      const HeadJob& q = a.job[t.job];
      int k0, k1;
      walk.blocks(t, &k0, &k1);
      const int row = (t.m * kHeadPair + int(rank)) * kHeadTileM + quarter * 32 + lane;
      const int col0 = EPI == kHeadGate ? t.n * (TN / 2) + half * (TN / 4) : t.n * TN + half * (TN / 2);
      // what the epilogue knows of the row is fetched while the products run
      const bool there = (EPI == kHeadLse || EPI == kHeadG) && row < r.rows;
      const int y = there ? r.labels[row] : -1;
      const bool known = unsigned(y) < unsigned(r.classes);
      const float lse = EPI == kHeadG && there ? r.lse[row] : 0.f;
      const float up = EPI == kHeadG && known ? r.dloss[row] : 0.f;
      // a gated block's gradient: what the forward call kept, four rows of 32 columns a step
      // (32 steps a tile), eight steps on their way
      constexpr int kAhead = 8;
      float px[kAhead][4], py[kAhead][4];
      auto fetch = [&](int step, float (&x)[4], float (&y)[4]) {
        const int rr = step % 8 * 4 + lane / 8, cc = step / 8 * 32 + lane % 8 * 4;
        const int n = a.g.width - (col0 + cc);
        if (step >= TN / 8 || row - lane + rr >= a.g.rows || n <= 0) return;
        const float* p = a.g.pre + (long long)(row - lane + rr) * a.g.ld_pre + col0 + cc;
        const float4 f = load4(p, n, a.g.wide_pre), h = load4(p + a.g.width, n, a.g.wide_pre);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        y[0] = h.x, y[1] = h.y, y[2] = h.z, y[3] = h.w;
      };
      if constexpr (EPI == kHeadGateGrad) {
        if (!q.plain) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) fetch(i, px[i], py[i]);
        }
      }
      bool ok = true;
      uint32_t src = 0;
      for (int c0 = k0; c0 < k1; c0 += F32 ? 1 : k1 - k0) {
        ok = __all_sync(~0u, wait(sums_full + 8 * as, aph));
        if (!ok) break;
        fence_after();
        src = tmem + as * TN + (uint32_t(quarter * 32) << 16) + half * (EPI == kHeadGate ? TN / 4 : TN / 2);
        if constexpr (F32) {
#pragma unroll
          for (int c = 0; c < TN / 2; c += 16) {
            float v[16];
            // a gated product: 64 gates, and their factors 128 columns on
            tmem_load16(src + c + (EPI == kHeadGate && c >= TN / 4 ? TN / 4 : 0), v);
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[c + i] = c0 == k0 ? v[i] : sums[c + i] + v[i];
          }
          if (kBack && c0 + 1 == k1) {
#pragma unroll
            for (int c = 0; c < TN / 2; c += 16)
              tmem_store16(src + c + (EPI == kHeadGate && c >= TN / 4 ? TN / 4 : 0), sums + c);
            tmem_stored();
            break;
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_at(sums_empty + 8 * as, 0);
          as ^= 1;
          if (as == 0) aph ^= 1;
        }
      }
      if (!ok) break;
      // the tile's tensor memory may be written again
      auto release = [&] {
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_at(sums_empty + 8 * as, 0);
        as ^= 1;
        if (as == 0) aph ^= 1;
      };
      // f(column, values) for each 32 columns: the sums in registers (their place has to be
      // known to the compiler), or from tensor memory, the next ones on their way
      auto each_part = [&](auto f) {
        if constexpr (F32 && !kBack) {
#pragma unroll
          for (int c = 0; c < TN / 2; c += 32) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = sums[c + i];
            f(c, v);
          }
        } else if constexpr (EPI != kHeadLse && EPI != kHeadG && EPI != kHeadOut) {
          // one copy of an epilogue that is long: its instructions come from far
          float v[32];
#pragma unroll 1
          for (int c = 0; c < TN / 2; c += 32) {
            tmem_issue(src + c, v);
            tmem_wait(v);
            if (c + 32 == TN / 2) release();  // all of it has been read
            f(c, v);
          }
        } else {
          float v[32], w[32];
          tmem_issue(src, v);
#pragma unroll 1
          for (int c = 0; c < TN / 2; c += 64) {
            tmem_wait(v);
            tmem_issue(src + c + 32, w);
            f(c, v);
            tmem_wait(w);
            if (c + 64 < TN / 2)
              tmem_issue(src + c + 64, v);
            else
              release();  // all of it has been read
            f(c + 32, w);
          }
        }
      };
      auto store_out = [&] {
        const int row0 = row - lane, rows = q.M - row0;
        float* acc = q.acc ? q.acc + ((long long)t.split * q.M + row0) * q.N + col0 : nullptr;
        const bool wide_acc = q.N % 4 == 0;  // its base is aligned
        // where row r of the product goes, -1: nowhere
        auto place = [&](int r) {
          return r < q.m_from ? r : r < q.m_to ? -1 : r - (q.m_to - q.m_from);
        };
        each_part([&](int c, float (&v)[32]) {
          if (kBlock && q.final && !q.acc_in && q.wide != 1) {
            // rows that start on 16 bytes of bfloat16, or off four values
            if (q.wide) {
              turn_bf16(stage, v, lane, [&](int rr, int cc, uint4 x) {
                const int n = q.N - (col0 + c + cc), to = place(row0 + rr);
                if (rr >= rows || n <= 0 || to < 0) return;
                store8(static_cast<__nv_bfloat16*>(q.out) + (long long)to * q.ld_out + col0 + c + cc, x, n, true);
              });
              return;
            }
            turn1(stage, v, lane, [&](int rr, int cc, float x) {
              const int to = place(row0 + rr);
              if (rr >= rows || col0 + c + cc >= q.N || to < 0) return;
              const long long at = (long long)to * q.ld_out + col0 + c + cc;
              if (q.out_f32)
                static_cast<float*>(q.out)[at] = x;
              else
                static_cast<__nv_bfloat16*>(q.out)[at] = __float2bfloat16_rn(x);
            });
            return;
          }
          turn(stage, v, lane, [&](int rr, int cc, float4 x) {
            const int n = q.N - (col0 + c + cc);
            if (rr >= rows || n <= 0) return;
            float* sum = acc + (long long)rr * q.N + c + cc;
            if (q.acc_in) {
              if (wide_acc) {
                const float4 o = *reinterpret_cast<const float4*>(sum);
                x = make_float4(x.x + o.x, x.y + o.y, x.z + o.z, x.w + o.w);
              } else {
                x.x += sum[0];
                if (n > 1) x.y += sum[1];
                if (n > 2) x.z += sum[2];
                if (n > 3) x.w += sum[3];
              }
            }
            const int to = kBlock ? place(row0 + rr) : row0 + rr;
            if (q.final && to < 0) return;
            const long long at = (long long)to * q.ld_out + col0 + c + cc;
            if (!q.final)
              store4(sum, x, n, wide_acc);
            else if (q.out_f32)
              store4(static_cast<float*>(q.out) + at, x, n, q.wide);
            else
              store4(static_cast<__nv_bfloat16*>(q.out) + at, x, n, q.wide);
          });
        });
      };
      if constexpr (F32 && (EPI == kHeadLse || EPI == kHeadG)) {
        const int v0 = (EPI == kHeadG ? r.v0 : 0) + col0;
        redo(sums, r.classes - v0, EPI == kHeadG ? known : there, r, row, v0);
      }
      if (EPI == kHeadLse) {
        float m = -INFINITY, sum = 0.f;
        each_part([&](int c, float (&v)[32]) {
          const int n = r.classes - (col0 + c);
          online(v, n, m, sum);
          if (unsigned(y - (col0 + c)) < 32u && y < r.classes) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col0 + c + i == y) x = v[i];
            r.target[row] = x;
          }
        });
        if (there) r.part[(long long)(t.n * 2 + half) * r.rows + row] = make_float2(m, sum);
      } else if (EPI == kHeadG) {
        // lanes past the last row hold zeros, which are not stored
        __nv_bfloat16* g = static_cast<__nv_bfloat16*>(r.g) + (long long)(row - lane) * r.ld_g + col0;
        const int rows = r.rows - (row - lane);
        each_part([&](int c, float (&v)[32]) {
          const int v0 = r.v0 + col0 + c;
          const int n = int(r.ld_g) - (col0 + c);  // a multiple of 32
          if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float p = exp2_approx((v[i] - lse) * kLog2e);
              if (v0 + i == y) p -= 1.f;
              v[i] = known && v0 + i < r.classes ? up * p : 0.f;
            }
            turn(stage, v, lane, [&](int rr, int cc, float4 x) {
              if (rr >= rows || n <= 0) return;
              __nv_bfloat16* p = g + rr * r.ld_g + c + cc;
              store4(p, x, 4, true);
              auto rest = [](float f) { return f - __bfloat162float(__float2bfloat16_rn(f)); };
#pragma unroll
              for (int z = 1; z < 3; ++z) {
                x = make_float4(rest(x.x), rest(x.y), rest(x.z), rest(x.w));
                store4(p + z * r.plane_g, x, 4, true);
              }
            });
          } else {
            // one product and sum, one exponential, one product a value; what only few
            // columns or rows need is done apart
            const float lse2 = lse * kLog2e;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = up * exp2_approx(fmaf(v[i], kLog2e, -lse2));
            if (unsigned(y - v0) < 32u) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (v0 + i == y) v[i] -= up;
            }
            if (!known || v0 + 32 > r.classes) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!known || v0 + i >= r.classes) v[i] = 0.f;
            }
            turn_bf16(stage, v, lane, [&](int rr, int cc, uint4 x) {
              if (rr < rows && n > 0) *reinterpret_cast<uint4*>(g + rr * r.ld_g + c + cc) = x;
            });
          }
        });
      } else if constexpr (EPI == kHeadGate) {
        const HeadGate& g = a.g;
        const int rows = g.rows - (row - lane);
        const long long r0 = row - lane;
        const bool wide = g.wide && (g.wide_pre || !g.pre);
        float* pre = g.pre ? g.pre + r0 * g.ld_pre + col0 : nullptr;
        // 16 gates and their factors at a time.  The product act(a) b is rounded once, to the type of h, which is the
        // caller's and the next product's operand: bfloat16 puts y 0.23% off where y's own rounding costs 0.17%.
#pragma unroll 1
        for (int c = 0; c < TN / 4; c += 16) {
          const int n0 = g.width - (col0 + c);
          {
            float v[16], w[16];
            tmem_load16(src + c, v);
            tmem_load16(src + TN / 2 + c, w);
            if (c + 16 == TN / 4) release();
            put_pairs(stage, v, w, lane);
          }
          if (wide) {
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {  // eight rows, four columns a lane
              const int rr = i * 8 + lane / 4, cc = lane % 4 * 4, n = n0 - cc;
              float x[4], y[4];
              read4(pair_unit(stage, rr, lane % 4), x);
              read4(pair_unit(stage, rr, 4 + lane % 4), y);
              if (rr >= rows || n <= 0) continue;
              if (pre) {
                store4(pre + rr * g.ld_pre + c + cc, four(x), n, true);
                store4(pre + rr * g.ld_pre + g.width + c + cc, four(y), n, true);
              }
              activate<!F32>(g.act, x, y);
              const long long at = (r0 + rr) * g.ld_hidden + col0 + c + cc;
              if (F32)
                store4(static_cast<float*>(g.hidden) + at, four(x), n, true);
              else
                store4(static_cast<__nv_bfloat16*>(g.hidden) + at, four(x), n, true);
            }
          } else {
#pragma unroll 2
            for (int i = 0; i < 16; ++i) {  // two rows, a column a lane
              const int rr = i * 2 + lane / 16, cc = lane % 16;
              float x[1] = {read1(pair_unit(stage, rr, cc / 4) + cc % 4 * 4)};
              const float y[1] = {read1(pair_unit(stage, rr, 4 + cc / 4) + cc % 4 * 4)};
              if (rr >= rows || cc >= n0) continue;
              if (pre) {
                pre[rr * g.ld_pre + c + cc] = x[0];
                pre[rr * g.ld_pre + g.width + c + cc] = y[0];
              }
              activate<!F32>(g.act, x, y);
              const long long at = (r0 + rr) * g.ld_hidden + col0 + c + cc;
              if (F32)
                static_cast<float*>(g.hidden)[at] = x[0];
              else
                static_cast<__nv_bfloat16*>(g.hidden)[at] = __float2bfloat16_rn(x[0]);
            }
          }
        }
      } else if constexpr (EPI == kHeadGateGrad) {
        if (q.plain) {
          store_out();
          continue;
        }
        // up to `half` columns a half, zeros from `width` on: whole units of four.  Rounded to bfloat16, as operands
        // of dx and dW: three planes, as float32 has them, would be six products in place of one.
        const HeadGate& g = a.g;
        const int rows = g.rows - (row - lane), n0 = g.width - col0, n1 = g.half - col0;
        __nv_bfloat16* d = static_cast<__nv_bfloat16*>(g.dpre) + (long long)(row - lane) * g.ld_d + col0;
        each_part([&](int c, float (&v)[32]) {
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((u ^ (lane & 7)) << 4)),
                         "f"(v[4 * u]), "f"(v[4 * u + 1]), "f"(v[4 * u + 2]), "f"(v[4 * u + 3])
                         : "memory");
          __syncwarp();
#pragma unroll 1
          for (int i0 = 0; i0 < 8; i0 += kAhead)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {  // four rows, four columns a lane
              const int rr = (i0 + k) * 4 + lane / 8, u = lane % 8, cc = c + 4 * u;
              float dh[4], dx[4], dy[4];
              read4(stage + rr * 128 + ((u ^ (rr & 7)) << 4), dh);
              gate_grad4(g.act, px[k], py[k], dh, dx, dy);
              fetch(c / 4 + i0 + k + kAhead, px[k], py[k]);
              if (rr >= rows || cc >= n1) continue;
              if (cc + 4 > n0)
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (cc + z >= n0) dx[z] = dy[z] = 0.f;
              __nv_bfloat16* to = d + rr * g.ld_d + cc;
              store4(to, four(dx), 4, true);
              store4(to + g.half, four(dy), 4, true);
            }
        });
      } else {
        store_out();
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still reach its barriers
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TN));
  }
}

// ---- the kernels around it ------------------------------------------------------

// Planes of bfloat16 with 16-byte aligned rows: the terms of a float32, or a copy.  A
// warp a row, eight values a lane; the rows of several matrices one after the other.
// It also clears the status word, unless null.
constexpr float kLargest = 3.3895313892515355e38f;  // of bfloat16
struct HeadPackList {
  HeadPack m[kHeadPacks];
  int count;
};
template <class T>
__global__ void __launch_bounds__(256) head_pack_kernel(const __grid_constant__ HeadPackList list, unsigned* status) {
  if (status && blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
  const int lane = threadIdx.x % 32;
  long long r = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  int at = 0;
  while (at < list.count && r >= list.m[at].rows) r -= list.m[at++].rows;
  if (at == list.count) return;
  const HeadPack& m = list.m[at];
  // a row without a label becomes zeros
  const int cols = m.labels && unsigned(m.labels[r]) >= unsigned(m.classes) ? 0 : int(m.cols);
  const T* from = static_cast<const T*>(m.src) + r * m.ld;
  __nv_bfloat16* to = static_cast<__nv_bfloat16*>(m.dst) + r * m.ldp;
  const long long plane = m.rows * m.ldp;
#pragma unroll 2
  for (int c = lane * 8; c < int(m.ldp); c += 256) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? float(from[c + i]) : 0.f;
#pragma unroll
    for (int z = 0; z < (sizeof(T) == 4 ? 3 : 1); ++z) {
      __nv_bfloat16 t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // finite values that would round to infinity: bfloat16's largest, and a rest
        const float u = sizeof(T) == 4 && isfinite(v[i]) ? fminf(fmaxf(v[i], -kLargest), kLargest) : v[i];
        t[i] = __float2bfloat16_rn(u);
        v[i] = z == 0 && !isfinite(v[i]) ? 0.f : v[i] - __bfloat162float(t[i]);
      }
      *reinterpret_cast<uint4*>(to + z * plane + c) = *reinterpret_cast<const uint4*>(t);
    }
  }
}

// The (max, sum) parts of a row to its log-sum-exp and loss.  A block takes `per` rows
// (a power of two, at most 32) with 256 / per threads each, eight parts at a time.
__global__ void __launch_bounds__(256)
    head_finish_kernel(const float2* part, const float* target, const int* labels, long long rows,
                       int classes, int parts, float* loss, float* lse, int per) {
  constexpr int BATCH = 8;
  __shared__ float2 mine[256];
  const int x = threadIdx.x % per, t = threadIdx.x / per, threads = 256 / per;
  const long long n = (long long)blockIdx.x * per + x;
  float m = -INFINITY, s = 0.f;
  // s exp(m - base), with an infinite m standing for 0 as in online()
  auto term = [](float m, float s, float base) {
    return s == 0.f ? 0.f : s * expf((fabsf(m) == INFINITY ? 0.f : m) - base);
  };
  if (n < rows)
    for (int i = t; i < parts; i += threads * BATCH) {
      float2 p[BATCH];
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        const int at = i + q * threads;
        p[q] = at < parts ? part[at * rows + n] : make_float2(-INFINITY, 0.f);
      }
      float top = m;
#pragma unroll
      for (int q = 0; q < BATCH; ++q) top = fmaxf(top, p[q].x);
      const float base = fabsf(top) == INFINITY ? 0.f : top;
      s = term(m, s, base);
#pragma unroll
      for (int q = 0; q < BATCH; ++q) s += term(p[q].x, p[q].y, base);
      m = top;
    }
  mine[threadIdx.x] = make_float2(m, s);
  __syncthreads();
  for (int o = threads / 2; o > 0; o /= 2) {
    if (t < o) {
      const float2 p = mine[threadIdx.x + o * per];
      const float top = fmaxf(m, p.x), base = fabsf(top) == INFINITY ? 0.f : top;
      s = term(m, s, base) + term(p.x, p.y, base);
      m = top;
      mine[threadIdx.x] = make_float2(m, s);
    }
    __syncthreads();
  }
  if (t == 0 && n < rows) {
    const float v = (fabsf(m) == INFINITY ? 0.f : m) + logf(s);
    const int y = labels[n];
    lse[n] = v;
    loss[n] = unsigned(y) < unsigned(classes) ? v - target[n] : 0.f;
  }
}

// Y threads a value, each every Y-th part.
template <int Y>
__global__ void __launch_bounds__(256) head_reduce_kernel(const HeadReduce a) {
  __shared__ float sums[256];
  constexpr int X = 256 / Y;
  const int x = threadIdx.x % X, y = threadIdx.x / X;
  const long long i = (long long)blockIdx.x * X + x, all = a.M * a.N;
  float v = 0.f;
  if (i < all) {
    if (y == 0 && a.acc_in) v = a.acc[i];
#pragma unroll 8
    for (int s = y; s < a.splits; s += Y) v += a.part[s * all + i];
  }
  if (Y > 1) {
    sums[threadIdx.x] = v;
    __syncthreads();
    if (y > 0) return;
#pragma unroll
    for (int q = 1; q < Y; ++q) v += sums[q * X + x];
  }
  if (i >= all) return;
  if (!a.final) {
    a.acc[i] = v;
    return;
  }
  const long long r = i / a.N;
  long long to = r;
  if (to >= a.m_from) {
    if (to < a.m_to) return;
    to -= a.m_to - a.m_from;
  }
  const long long o = to * a.ld_out + (i - r * a.N);
  if (a.out_f32)
    static_cast<float*>(a.out)[o] = v;
  else
    static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(v);
}

// ---- a narrow head --------------------------------------------------------------
//
// At most 64 columns and 32 classes (a calibration of class margins): the tensor
// cores' tiles of 256 x 256 would be padding, and the bytes of h and dh bound the work.
// A lane has a row in registers, the weights are 16-byte broadcasts from shared memory,
// all in float32.  dw: lane c of a warp sums the products of class and four columns
// number c (and c + 32 ...) over the warp's rows, block after block of rows, in
// registers; blocks leave their sums for a last small kernel.  500k x 10 x 10 float32: loss
// 15 us, gradient 35, last sums 5, bound by instructions and shared-memory reads (the
// tensor-core form took 956 for the step).

constexpr int kNarrowWarps = 4;

struct Narrow {
  const void *h, *w;
  long long rows, ld_h, ld_w;
  int cols, classes;
  const int* labels;
  float *loss, *lse_out;
  const float *lse, *dloss;
  void* dh;
  long long ld_dh;
  float* part;             // gridDim.x x classes x cols, or null
  unsigned* status;
};

template <class T>
__device__ __forceinline__ float load_f(const T* p) {
  return float(*p);
}

// Two float32 products and sums in one instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pair(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
struct alignas(16) F4 {  // four adjacent floats of shared memory
  F2 lo, hi;
};

template <class T, int DP, int VP, bool GRAD>
__global__ void __launch_bounds__(kNarrowWarps * 32) head_narrow_kernel(const Narrow a) {
  constexpr int Q = DP / 4;              // quads of columns
  constexpr int PITCH = DP + 4;          // an odd number of 16 bytes: no bank conflicts
  constexpr int GP = VP + 1;
  constexpr int NC = (VP * Q + 31) / 32; // (class, quad) pairs a lane
  extern __shared__ float4 shared4[];
  float* w = reinterpret_cast<float*>(shared4);                      // VP x DP, zeros beyond
  float* tiles = w + VP * DP;                                        // warps x 32 x PITCH
  float* gs = tiles + kNarrowWarps * 32 * PITCH;                     // warps x 32 x GP
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float* tile = tiles + warp * 32 * PITCH;
  float* gt = gs + warp * 32 * GP;
  const int D = a.cols, V = a.classes, nq = (D + 3) / 4;
  const T* W = static_cast<const T*>(a.w);
  for (int i = threadIdx.x; i < VP * DP; i += kNarrowWarps * 32) {
    const int v = i / DP, d = i % DP;
    w[i] = v < V && d < D ? load_f(W + v * a.ld_w + d) : 0.f;
  }
  for (int i = lane; i < 32 * PITCH; i += 32) tile[i] = 0.f;  // columns D .. stay zero
  // there is no wait to run out
  if (!GRAD && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  __syncthreads();
  const unsigned inv = ((1u << 20) + unsigned(D) - 1u) / unsigned(D);  // exact for i < 2,048
  F4 acc[GRAD ? NC : 1];
  int acc_v[GRAD ? NC : 1], acc_q[GRAD ? NC : 1];
#pragma unroll
  for (int c = 0; c < (GRAD ? NC : 1); ++c) {
    acc[c].lo = acc[c].hi = pair(0.f, 0.f);
    const int i = lane + 32 * c;
    acc_v[c] = i < V * nq ? i / nq : 0;
    acc_q[c] = i < V * nq ? i % nq : 0;
  }
  const long long step = (long long)gridDim.x * kNarrowWarps * 32;
  // adjacent rows on 16 bytes: a warp's 32 are fetched ahead, while the ones before are
  // worked on
  constexpr int PER = 16 / int(sizeof(T)), AHEAD = DP / PER;
  const bool dense = a.ld_h == D && (reinterpret_cast<uintptr_t>(a.h) & 15) == 0;
  uint4 ahead[AHEAD];
  auto fetch = [&](long long row0) {
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(a.h) + row0 * D);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (32 * j + lane < 32 / PER * D) ahead[j] = from[32 * j + lane];
  };
  {
    const long long row0 = ((long long)blockIdx.x * kNarrowWarps + warp) * 32;
    if (dense && row0 + 32 <= a.rows) fetch(row0);
  }
  for (long long row0 = ((long long)blockIdx.x * kNarrowWarps + warp) * 32; row0 < a.rows; row0 += step) {
    const int nr = int(a.rows - row0 < 32 ? a.rows - row0 : 32);
    const T* H = static_cast<const T*>(a.h) + row0 * a.ld_h;
    const long long row = row0 + lane;
    const bool there = lane < nr;
    const int y = there ? a.labels[row] : -1;
    const bool known = unsigned(y) < unsigned(V);
    const float lse_in = GRAD && there ? a.lse[row] : 0.f, up = GRAD && known ? a.dloss[row] : 0.f;
    __syncwarp();
    if (dense && nr == 32) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (32 * j + lane < 32 / PER * D) {
          const T* x = reinterpret_cast<const T*>(&ahead[j]);
          const int i0 = (32 * j + lane) * PER;
          int r = int((unsigned(i0) * inv) >> 20), c = i0 - r * D;
#pragma unroll
          for (int z = 0; z < PER; ++z) {
            tile[r * PITCH + c] = load_f(x + z);
            if (++c == D) {
              c = 0;
              ++r;
            }
          }
        }
      if (row0 + step + 32 <= a.rows) fetch(row0 + step);
    } else {
      for (int i = lane; i < nr * D; i += 32) {
        const int r = int((unsigned(i) * inv) >> 20), c = i - r * D;
        tile[r * PITCH + c] = load_f(H + r * a.ld_h + c);
      }
    }
    __syncwarp();
    // logits: VP independent chains, a quad of columns after the other
    F2 x[VP];
#pragma unroll
    for (int v = 0; v < VP; ++v) x[v] = pair(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (q < nq) {
        const F4 h = *reinterpret_cast<const F4*>(tile + lane * PITCH + 4 * q);
#pragma unroll
        for (int v = 0; v < VP; ++v) {
          const F4 t = *reinterpret_cast<const F4*>(w + v * DP + 4 * q);
          x[v] = fma2(h.hi, t.hi, fma2(h.lo, t.lo, x[v]));
        }
      }
    float l[VP], m = -INFINITY, target = 0.f;
#pragma unroll
    for (int v = 0; v < VP; ++v) {
      const float2 p = split(x[v]);
      l[v] = v < V ? p.x + p.y : -INFINITY;
      m = fmaxf(m, l[v]);
      if (v == y) target = l[v];
    }
    if constexpr (!GRAD) {
      const float base = fabsf(m) == INFINITY ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < VP; ++v) s += exp2_approx((l[v] - base) * kLog2e);
      const float lse = base + logf(s);
      if (there) {
        a.lse_out[row] = lse;
        a.loss[row] = known ? lse - target : 0.f;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VP; ++v) {
        const float p = exp2_approx((l[v] - lse_in) * kLog2e);
        l[v] = known && v < V ? up * (v == y ? p - 1.f : p) : 0.f;
        gt[lane * GP + v] = l[v];
      }
      if (a.part) {
        // a row without a label adds nothing, whatever its h
        if (!known)
#pragma unroll
          for (int q = 0; q < Q; ++q)
            *reinterpret_cast<float4*>(tile + lane * PITCH + 4 * q) = make_float4(0.f, 0.f, 0.f, 0.f);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (32 * c < V * nq) {
            const float *pg = gt + acc_v[c], *ph = tile + 4 * acc_q[c];
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
              const float g = pg[r * GP];
              const F4 h = *reinterpret_cast<const F4*>(ph + r * PITCH);
              const F2 gg = pair(g, g);
              acc[c].lo = fma2(gg, h.lo, acc[c].lo);
              acc[c].hi = fma2(gg, h.hi, acc[c].hi);
            }
          }
        __syncwarp();
      }
      if (a.dh) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (q < nq) {
            F4 s;
            s.lo = s.hi = pair(0.f, 0.f);
#pragma unroll
            for (int v = 0; v < VP; ++v) {
              const F4 t = *reinterpret_cast<const F4*>(w + v * DP + 4 * q);
              const F2 gg = pair(l[v], l[v]);
              s.lo = fma2(gg, t.lo, s.lo);
              s.hi = fma2(gg, t.hi, s.hi);
            }
            // columns D .. stay zero: there g times w's zeros is NaN for a g that is not
            // finite, and the next row's logits read them
            if (4 * q + 4 > D) {
              const float2 lo = split(s.lo), hi = split(s.hi);
              s.lo = pair(lo.x, 4 * q + 1 < D ? lo.y : 0.f);
              s.hi = pair(4 * q + 2 < D ? hi.x : 0.f, 0.f);
            }
            *reinterpret_cast<F4*>(tile + lane * PITCH + 4 * q) = s;
          }
        __syncwarp();
        T* to = static_cast<T*>(a.dh) + row0 * a.ld_dh;
#pragma unroll 4
        for (int i = lane; i < nr * D; i += 32) {
          const int r = int((unsigned(i) * inv) >> 20), c = i - r * D;
          to[r * a.ld_dh + c] = T(tile[r * PITCH + c]);
        }
      }
    }
  }
  if (GRAD && a.part) {
    // the warps' sums, one after the other, in the tiles' place
    float4* sums = reinterpret_cast<float4*>(tiles);
    for (int k = 0; k < kNarrowWarps; ++k) {
      __syncthreads();
      if (warp == k) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float2 lo = split(acc[c].lo), hi = split(acc[c].hi);
          float4 x = make_float4(lo.x, lo.y, hi.x, hi.y);
          if (k > 0) {
            const float4 o = sums[lane + 32 * c];
            x = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
          }
          sums[lane + 32 * c] = x;
        }
      }
    }
    __syncthreads();
    const float* flat = reinterpret_cast<const float*>(sums);
    for (int i = threadIdx.x; i < V * D; i += kNarrowWarps * 32)
      a.part[(long long)blockIdx.x * V * D + i] = flat[i / D * (4 * nq) + i % D];
  }
}

// dw from the blocks' sums, a block a value: every thread has its few loads in flight.
constexpr int kNarrowReduce = 128;
template <class T>
__global__ void __launch_bounds__(kNarrowReduce)
    head_narrow_reduce_kernel(const float* part, int blocks, int cols, int values, T* dw, long long ld) {
  __shared__ float sums[kNarrowReduce / 32];
  const int i = int(blockIdx.x);
  float v = 0.f;
#pragma unroll 5
  for (int b = threadIdx.x; b < blocks; b += kNarrowReduce) v += part[(long long)b * values + i];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kNarrowReduce / 32; ++w) v += sums[w];
    dw[i / cols * ld + i % cols] = T(v);
  }
}

template <class T, int DP, int VP>
cudaError_t narrow_of(const Narrow& a, bool grad, int blocks, cudaStream_t s) {
  constexpr size_t smem = (VP * DP + kNarrowWarps * 32 * (DP + 4 + VP + 1)) * sizeof(float);
  const auto k = grad ? head_narrow_kernel<T, DP, VP, true> : head_narrow_kernel<T, DP, VP, false>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  k<<<blocks, kNarrowWarps * 32, smem, s>>>(a);
  return cudaGetLastError();
}

template <class T, int DP>
cudaError_t narrow_cols(const Narrow& a, bool grad, int blocks, cudaStream_t s) {
  if (a.classes <= 4) return narrow_of<T, DP, 4>(a, grad, blocks, s);
  if (a.classes <= 8) return narrow_of<T, DP, 8>(a, grad, blocks, s);
  if (a.classes <= 12) return narrow_of<T, DP, 12>(a, grad, blocks, s);
  if (a.classes <= 16) return narrow_of<T, DP, 16>(a, grad, blocks, s);
  return narrow_of<T, DP, 32>(a, grad, blocks, s);
}

template <class T>
cudaError_t narrow_type(const Narrow& a, bool grad, int blocks, cudaStream_t s) {
  if (a.cols <= 16) return narrow_cols<T, 16>(a, grad, blocks, s);
  if (a.cols <= 32) return narrow_cols<T, 32>(a, grad, blocks, s);
  return narrow_cols<T, 64>(a, grad, blocks, s);
}

// ---- few rows -------------------------------------------------------------------
//
// A handful of rows against many classes: reading the weights bounds the work, so the
// CUDA cores take them as they stream by, in float32 (the tensor cores would want 256
// rows, and three planes of float32 weights written first).  The rows lie in shared
// memory.  A warp takes C classes at once -- each 16 bytes of a row of h it reads serve C
// classes -- and its C x NR <= 32 sums meet in 31 shuffles, one sum a lane.
//
// loss   lane (c, n) keeps the running maximum and sum of its classes' logits
// grad   g goes to the workspace, dw's C rows are formed at once from g and h; a second
//        kernel reads the weights again for dh = g w, a thread a few columns
//
// One row x 1,024 x 131,072 bfloat16: loss 43 us (6.2 TB/s).  Four rows with gradient: 56 +
// 99 + 86 us.

constexpr int kFewThreads = 256;

struct Few {
  const void *h, *w;
  int rows, cols, classes;
  long long ld_h, ld_w;
  const int* labels;
  const float *lse, *dloss;
  float2* part;            // loss: blocks x rows
  float* target;
  float* g;                // grad: classes x NR
  void* dw;                // or null
  long long ld_dw;
  float* dh_part;          // grad: chunks x rows x cols
  unsigned* status;
};

// PER adjacent values of a row, as pairs of floats; PER = 1: two values `apart` columns
// from each other, the second one if there are `left` > apart columns.
template <class T, int PER>
__device__ __forceinline__ void load_pairs(const T* p, int apart, int left, F2 (&v)[(PER + 1) / 2]) {
  if constexpr (PER == 1) {
    v[0] = pair(float(p[0]), left > apart ? float(p[apart]) : 0.f);
  } else if constexpr (sizeof(T) == 4) {
    const float4 q = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = pair(q.x, q.y);
    v[1] = pair(q.z, q.w);
  } else {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = pair(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
  }
}
template <int PER>
__device__ __forceinline__ void load_shared(const float* p, F2 (&v)[(PER + 1) / 2]) {
  if constexpr (PER == 1) {
    v[0] = pair(p[0], p[32]);
  } else {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      const F4 q = *reinterpret_cast<const F4*>(p + 4 * i);
      v[2 * i] = q.lo;
      v[2 * i + 1] = q.hi;
    }
  }
}
template <class T, int PER>
__device__ __forceinline__ void store_pairs(T* p, int left, const F2 (&v)[(PER + 1) / 2]) {
  if constexpr (PER == 1) {
    const float2 x = split(v[0]);
    p[0] = T(x.x);
    if (left > 32) p[32] = T(x.y);
  } else if constexpr (sizeof(T) == 4) {
    const float2 x = split(v[0]), y = split(v[1]);
    *reinterpret_cast<float4*>(p) = make_float4(x.x, x.y, y.x, y.y);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = split(v[i]);
      u[i] = pack2(x.x, x.y);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

template <class T, int NR, int PER, bool GRAD>
__global__ void __launch_bounds__(kFewThreads, 2) head_few_kernel(const Few a) {
  constexpr int C = NR > 4 ? 32 / NR : NR == 4 && PER == 8 ? 4 : 8;  // classes a warp
  constexpr int S = C * NR;                 // sums: 8, 16 or 32
  constexpr int P = (PER + 1) / 2;
  extern __shared__ float4 few_shared[];
  float* hs = reinterpret_cast<float*>(few_shared);  // NR x pitch
  __shared__ float2 sums[kFewThreads / 32][NR];
  constexpr int STEP = PER == 1 ? 64 : 32 * PER;  // columns a warp takes at once
  const int pitch = few_pitch(a.cols);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // there is no wait to run out
  if (!GRAD && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  for (int n = 0; n < NR; ++n) {
    // rows that do not exist, and in the gradient rows without a label, are zeros
    const bool there = n < a.rows && (!GRAD || unsigned(a.labels[n]) < unsigned(a.classes));
    for (int d = threadIdx.x; d < pitch; d += kFewThreads)
      hs[n * pitch + d] = there && d < a.cols ? float(static_cast<const T*>(a.h)[n * a.ld_h + d]) : 0.f;
  }
  __syncthreads();
  const T* W = static_cast<const T*>(a.w);
  // after the shuffles lane i has sum i / (32 / S)
  const int mine = lane / (32 / S), mc = mine / NR, mn = mine % NR;
  const bool there = mn < a.rows;
  const int y = there ? a.labels[mn] : -1;
  const bool known = unsigned(y) < unsigned(a.classes);
  const float lse = GRAD && there ? a.lse[mn] : 0.f, up = GRAD && known ? a.dloss[mn] : 0.f;
  float m = -INFINITY, sum = 0.f;
  const int stride = int(gridDim.x) * (kFewThreads / 32) * C;
  for (int v0 = (int(blockIdx.x) * (kFewThreads / 32) + warp) * C; v0 < a.classes; v0 += stride) {
    F2 acc[C][NR];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[c][n] = pair(0.f, 0.f);
#pragma unroll 2
    for (int d = lane * PER; d < a.cols; d += STEP) {
      F2 w[C][P];
#pragma unroll
      for (int c = 0; c < C; ++c)
        load_pairs<T, PER>(W + min(v0 + c, a.classes - 1) * a.ld_w + d, 32, a.cols - d, w[c]);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        F2 h[P];
        load_shared<PER>(hs + n * pitch + d, h);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) acc[c][n] = fma2(w[c][i], h[i], acc[c][n]);
      }
    }
    float s[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const float2 x = split(acc[i / NR][i % NR]);
      s[i] = x.x + x.y;
    }
    int o = 16;
#pragma unroll
    for (int k = S / 2; k > 0; k /= 2) {
      const bool high = lane & o;
#pragma unroll
      for (int i = 0; i < k; ++i) {
        const float give = high ? s[i] : s[i + k], keep = high ? s[i + k] : s[i];
        s[i] = keep + __shfl_xor_sync(~0u, give, o);
      }
      o /= 2;
    }
    float l = s[0];
    for (; o > 0; o /= 2) l += __shfl_xor_sync(~0u, l, o);
    const int v = v0 + mc;
    if (!GRAD) {
      if (v < a.classes) {
        const float top = fmaxf(m, l), base = fabsf(top) == INFINITY ? 0.f : top;
        const float old = fabsf(m) == INFINITY ? 0.f : m;
        sum = (sum == 0.f ? 0.f : sum * exp2_approx((old - base) * kLog2e)) +
              exp2_approx((l - base) * kLog2e);
        m = top;
        if (v == y && lane % (32 / S) == 0) a.target[mn] = l;
      }
    } else {
      float g = 0.f;
      if (known && v < a.classes) {
        const float p = exp2_approx((l - lse) * kLog2e);
        g = up * (v == y ? p - 1.f : p);
      }
      if (lane % (32 / S) == 0 && v < a.classes) a.g[(long long)v * NR + mn] = g;
      if (a.dw) {
        float gs[S];
#pragma unroll
        for (int i = 0; i < S; ++i) gs[i] = __shfl_sync(~0u, g, i * (32 / S));
        T* to = static_cast<T*>(a.dw) + v0 * a.ld_dw;
        for (int d = lane * PER; d < a.cols; d += STEP) {
          F2 x[C][P];
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i) x[c][i] = pair(0.f, 0.f);
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            F2 h[P];
            load_shared<PER>(hs + n * pitch + d, h);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const F2 gg = pair(gs[c * NR + n], gs[c * NR + n]);
#pragma unroll
              for (int i = 0; i < P; ++i) x[c][i] = fma2(gg, h[i], x[c][i]);
            }
          }
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (v0 + c < a.classes) store_pairs<T, PER>(to + c * a.ld_dw + d, a.cols - d, x[c]);
        }
      }
    }
  }
  if (!GRAD) {
    // lanes of one row, then the warps
    auto join = [&](float m2, float s2) {
      const float top = fmaxf(m, m2), base = fabsf(top) == INFINITY ? 0.f : top;
      auto term = [&](float mm, float ss) {
        return ss == 0.f ? 0.f : ss * exp2_approx(((fabsf(mm) == INFINITY ? 0.f : mm) - base) * kLog2e);
      };
      sum = term(m, sum) + term(m2, s2);
      m = top;
    };
#pragma unroll
    for (int o = NR * (32 / S); o < 32; o *= 2) {
      const float m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, sum, o);
      join(m2, s2);
    }
    if (lane % (32 / S) == 0 && mc == 0) sums[warp][mn] = make_float2(m, sum);
    __syncthreads();
    if (threadIdx.x < NR && int(threadIdx.x) < a.rows) {
      m = sums[0][threadIdx.x].x;
      sum = sums[0][threadIdx.x].y;
      for (int q = 1; q < kFewThreads / 32; ++q) join(sums[q][threadIdx.x].x, sums[q][threadIdx.x].y);
      a.part[(long long)blockIdx.x * a.rows + threadIdx.x] = make_float2(m, sum);
    }
  }
}

// dh_part[chunk] = g w over the chunk's classes: `tx` threads for PER columns each,
// 256 / tx classes at once.
template <class T, int NR, int PER>
__global__ void __launch_bounds__(kFewThreads) head_few_dh_kernel(const Few a, int tx, int chunk) {
  constexpr int P = (PER + 1) / 2;
  __shared__ F2 meet[kFewThreads];
  const int ty = kFewThreads / tx, x = threadIdx.x % tx, yy = threadIdx.x / tx;
  // PER columns from d on, or d and d + tx
  const int d = PER == 1 ? int(blockIdx.x) * 2 * tx + x : (int(blockIdx.x) * tx + x) * PER;
  const int v0 = int(blockIdx.y) * chunk, v1 = min(v0 + chunk, a.classes);
  F2 acc[NR][P];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < P; ++i) acc[n][i] = pair(0.f, 0.f);
  if (d < a.cols) {
    const T* w = static_cast<const T*>(a.w) + d;
#pragma unroll 4
    for (int v = v0 + yy; v < v1; v += ty) {
      F2 q[P];
      load_pairs<T, PER>(w + v * a.ld_w, tx, a.cols - d, q);
      float g[NR];
      if constexpr (NR >= 4) {
#pragma unroll
        for (int n = 0; n < NR; n += 4) {
          const float4 t = __ldg(reinterpret_cast<const float4*>(a.g + (long long)v * NR + n));
          g[n] = t.x, g[n + 1] = t.y, g[n + 2] = t.z, g[n + 3] = t.w;
        }
      } else {
#pragma unroll
        for (int n = 0; n < NR; ++n) g[n] = __ldg(a.g + (long long)v * NR + n);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const F2 gg = pair(g[n], g[n]);
#pragma unroll
        for (int i = 0; i < P; ++i) acc[n][i] = fma2(gg, q[i], acc[n][i]);
      }
    }
  }
  for (int n = 0; n < NR; ++n) {
    if (n >= a.rows) break;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      F2 v = acc[0][i];
#pragma unroll
      for (int k = 1; k < NR; ++k)
        if (k == n) v = acc[k][i];
      if (ty > 1) {
        __syncthreads();
        meet[threadIdx.x] = v;
        __syncthreads();
      }
      if (yy == 0 && d < a.cols) {
        float2 s = split(v);
        for (int k = 1; k < ty; ++k) {
          const float2 o = split(meet[k * tx + x]);
          s.x += o.x;
          s.y += o.y;
        }
        float* to = a.dh_part + ((long long)blockIdx.y * a.rows + n) * a.cols + d + 2 * i;
        to[0] = s.x;
        if (PER > 1)
          to[1] = s.y;
        else if (d + tx < a.cols)
          to[tx] = s.y;
      }
    }
  }
}

template <class T, int NR, int PER>
cudaError_t few_of(const Few& a, bool grad, int blocks, int chunks, cudaStream_t s) {
  const size_t smem = size_t(NR) * few_pitch(a.cols) * sizeof(float);
  const auto k = grad ? head_few_kernel<T, NR, PER, true> : head_few_kernel<T, NR, PER, false>;
  // the limit of the largest call, not this one's: it is the kernel's, and another thread may
  // launch between this thread's two calls
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kFewSmem));
  if (e != cudaSuccess) return e;
  k<<<blocks, kFewThreads, smem, s>>>(a);
  if (grad && a.dh_part) {
    int tx = 32;
    constexpr int PER2 = PER == 1 ? 2 : PER;  // columns a thread
    while (tx < kFewThreads && tx * PER2 < a.cols) tx *= 2;
    const int chunk = (a.classes + chunks - 1) / chunks;
    head_few_dh_kernel<T, NR, PER>
        <<<dim3((a.cols + tx * PER2 - 1) / (tx * PER2), chunks), kFewThreads, 0, s>>>(a, tx, chunk);
  }
  return cudaGetLastError();
}

template <class T, int PER>
cudaError_t few_rows(const Few& a, bool grad, int blocks, int chunks, cudaStream_t s) {
  if (a.rows <= 1) return few_of<T, 1, PER>(a, grad, blocks, chunks, s);
  if (a.rows <= 2) return few_of<T, 2, PER>(a, grad, blocks, chunks, s);
  if (a.rows <= 4) return few_of<T, 4, PER>(a, grad, blocks, chunks, s);
  if constexpr (sizeof(T) == 4) {
    if (a.rows <= 8) return few_of<T, 8, PER>(a, grad, blocks, chunks, s);
    return few_of<T, 16, PER>(a, grad, blocks, chunks, s);
  }
  return cudaErrorInvalidValue;
}

template <int EPI, int TN, bool F32>
cudaError_t go_type(const HeadLaunch& a, cudaStream_t s) {
  constexpr int kStage = (F32 ? 3 : 1) * (kHeadTileM * 128 + TN / kHeadPair * 128);
  constexpr size_t smem = size_t((192 * 1024) / kStage) * kStage + 1024 +
                          (EPI == kHeadLse ? 0 : kEpilogueWarps * kTurnBytes);
  const auto k = head_kernel<EPI, TN, F32>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  if (F32) {
    // the warpgroups' registers are shared out of what the block is launched with
    static const bool enough = [] {
      cudaFuncAttributes f{};
      return cudaFuncGetAttributes(&f, head_kernel<EPI, TN, F32>) == cudaSuccess &&
             f.numRegs * kHeadThreads >= 128 * 56 + 256 * 224;
    }();
    if (!enough) return cudaErrorInvalidConfiguration;
  }
  long long tiles = 0;
  for (int j = 0; j < a.jobs; ++j)
    tiles += (long long)a.job[j].tiles_m * a.job[j].tiles_n * a.job[j].splits;
  if (tiles <= 0) return cudaSuccess;
  const int pairs = int(std::min<long long>(tiles, device_sms() / kHeadPair));
  k<<<pairs * kHeadPair, kHeadThreads, smem, s>>>(a);
  return cudaGetLastError();
}

template <int EPI, int TN>
cudaError_t go(const HeadLaunch& a, cudaStream_t s) {
  return a.f32 ? go_type<EPI, TN, true>(a, s) : go_type<EPI, TN, false>(a, s);
}

}  // namespace

cudaError_t launch_head(int epilogue, int tile_n, const HeadLaunch& a, cudaStream_t s) {
  if (epilogue == kHeadLse) return go<kHeadLse, 256>(a, s);
  if (epilogue == kHeadG) return go<kHeadG, 256>(a, s);
  if (epilogue == kHeadGate) return tile_n == 128 ? go<kHeadGate, 128>(a, s) : go<kHeadGate, 256>(a, s);
  if (epilogue == kHeadGateGrad)  // float32: a launch of its own (launch_ffn_split)
    return a.f32 ? cudaErrorInvalidValue : go_type<kHeadGateGrad, 256, false>(a, s);
  if (epilogue == kHeadBlock) return tile_n == 128 ? go<kHeadBlock, 128>(a, s) : go<kHeadBlock, 256>(a, s);
  return tile_n == 128 ? go<kHeadOut, 128>(a, s) : go<kHeadOut, 256>(a, s);
}

cudaError_t launch_head_narrow(const HeadArgs& h, bool grad, float* part, int blocks, cudaStream_t s) {
  Narrow a{};
  a.h = h.h;
  a.w = h.w;
  a.rows = h.rows;
  a.ld_h = h.ld_h;
  a.ld_w = h.ld_w;
  a.cols = int(h.cols);
  a.classes = int(h.classes);
  a.labels = h.labels;
  a.loss = h.loss;
  a.lse_out = h.lse_out;
  a.lse = h.lse;
  a.dloss = h.dloss;
  a.dh = h.dh;
  a.ld_dh = h.ld_dh;
  a.part = h.dw ? part : nullptr;
  a.status = static_cast<unsigned*>(h.workspace);
  cudaError_t e = h.dtype == kF32 ? narrow_type<float>(a, grad, blocks, s)
                                  : narrow_type<__nv_bfloat16>(a, grad, blocks, s);
  if (e != cudaSuccess || !grad || !h.dw) return e;
  const int values = a.classes * a.cols;
  if (h.dtype == kF32)
    head_narrow_reduce_kernel<float><<<values, kNarrowReduce, 0, s>>>(
        part, blocks, a.cols, values, static_cast<float*>(h.dw), h.ld_dw);
  else
    head_narrow_reduce_kernel<__nv_bfloat16><<<values, kNarrowReduce, 0, s>>>(
        part, blocks, a.cols, values, static_cast<__nv_bfloat16*>(h.dw), h.ld_dw);
  return cudaGetLastError();
}

cudaError_t launch_head_few(const HeadArgs& h, bool grad, const HeadFew& f, cudaStream_t s) {
  Few a{};
  a.h = h.h;
  a.w = h.w;
  a.rows = int(h.rows);
  a.cols = int(h.cols);
  a.classes = int(h.classes);
  a.ld_h = h.ld_h;
  a.ld_w = h.ld_w;
  a.labels = h.labels;
  a.lse = h.lse;
  a.dloss = h.dloss;
  a.part = f.part;
  a.target = f.target;
  a.g = f.g;
  a.dw = h.dw;
  a.ld_dw = h.ld_dw;
  a.dh_part = h.dh ? f.dh_part : nullptr;
  a.status = static_cast<unsigned*>(h.workspace);
  // 16 bytes at a time where the rows of w (and dw) start on them
  const long long size = h.dtype == kF32 ? 4 : 2, per = 16 / size;
  const uintptr_t at = reinterpret_cast<uintptr_t>(h.w) | uintptr_t(h.ld_w * size) |
                       uintptr_t(h.cols * size) |
                       (grad && h.dw ? reinterpret_cast<uintptr_t>(h.dw) | uintptr_t(h.ld_dw * size) : 0);
  const bool wide = at % 16 == 0 && h.cols % per == 0;
  if (h.dtype == kF32)
    return wide ? few_rows<float, 4>(a, grad, f.blocks, f.chunks, s)
                : few_rows<float, 1>(a, grad, f.blocks, f.chunks, s);
  return wide ? few_rows<__nv_bfloat16, 8>(a, grad, f.blocks, f.chunks, s)
              : few_rows<__nv_bfloat16, 1>(a, grad, f.blocks, f.chunks, s);
}

cudaError_t launch_head_pack(int dtype, const HeadPack* list, int count, unsigned* status, cudaStream_t s) {
  HeadPackList all{};
  long long rows = 0;
  for (; all.count < count; ++all.count) {
    all.m[all.count] = list[all.count];
    rows += list[all.count].rows;
  }
  const long long blocks = (rows + 7) / 8;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (dtype == kF32)
    head_pack_kernel<float><<<unsigned(blocks), 256, 0, s>>>(all, status);
  else
    head_pack_kernel<__nv_bfloat16><<<unsigned(blocks), 256, 0, s>>>(all, status);
  return cudaGetLastError();
}

cudaError_t launch_head_finish(const float2* part, const float* target, const int* labels,
                               int64_t rows, int64_t classes, int64_t parts, float* loss,
                               float* lse, cudaStream_t s) {
  // rows a block: fewer when that leaves multiprocessors without one
  int per = 1;
  while (per < 32 && rows / (2 * per) >= 2 * device_sms()) per *= 2;
  const long long blocks = (rows + per - 1) / per;
  head_finish_kernel<<<unsigned(blocks), 256, 0, s>>>(part, target, labels, rows, int(classes),
                                                      int(parts), loss, lse, per);
  return cudaGetLastError();
}

cudaError_t launch_head_reduce(const HeadReduce& a, cudaStream_t s) {
  const int x = a.splits >= 16 ? 32 : 256;
  const long long blocks = (a.M * a.N + x - 1) / x;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (x == 32)
    head_reduce_kernel<8><<<unsigned(blocks), 256, 0, s>>>(a);
  else
    head_reduce_kernel<1><<<unsigned(blocks), 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mb
