// Kernels of the softmax head (head.h): matrix products on the 5th-generation tensor
// cores whose epilogues reduce, form or store what the head needs.
//
// head_kernel: a persistent kernel, a pair of CTAs a 256 x 256 tile (tcgen05.mma,
// cta_group::2: each CTA holds 128 rows of A and half of B in shared memory and 128 x
// 256 float32 sums in its tensor memory).  Warp 0 fetches 128-byte swizzled tiles with
// TMA into a ring, warp 1 of the first CTA issues the products, warps 2 to 9 take the
// sums out of tensor memory, 32 rows and half the columns each, while the next tile
// fills the second half of it.
//
// A float32 operand is three planes of bfloat16, x = x1 + x2 + x3 with 8 bits each, and
// the product the six terms x_i y_j with i + j <= 4 -- what is dropped is below 2^-24
// of |x||y| -- the smallest terms first: the tensor core's sums are truncated to 32
// bits, and a small term costs little while the sum is small.
//
// Every wait ends after wait_ns: the CTA then marks itself dead, sets the status word,
// lets its copies land and returns (its results are void).
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "head.h"
#include "mixture.h"

namespace mb {

namespace {

constexpr int kEpilogueWarps = 8;
constexpr int kHeadThreads = 64 + kEpilogueWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

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
      " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}\n" ::"r"(bar),
      "r"(rank)
      : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
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
        atomicOr(status, 1u);
      }
    }
    return false;
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
// The products issued so far, when done, arrive at this barrier of both CTAs.
__device__ __forceinline__ void commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

// 32 lanes x 32 columns of tensor memory: column c of lane i to v[c] of thread i.
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
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
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  __device__ Walk(const HeadLaunch& l) : a(l) {
    pairs = int(gridDim.x) / kHeadPair;
    me = int(blockIdx.x) / kHeadPair;
    for (int j = 0; j < 2; ++j)
      count[j] = j < a.jobs ? a.job[j].tiles_m * a.job[j].tiles_n * a.job[j].splits : 0;
    light = count[0] % pairs;  // pairs from here on have one tile of job 0 fewer
    extra = 0;
    if (a.jobs > 1 && light > 0) {
      const int c0 = (a.job[0].kblocks + a.job[0].splits - 1) / a.job[0].splits;
      const int c1 = (a.job[1].kblocks + a.job[1].splits - 1) / a.job[1].splits;
      extra = c1 > 0 ? (c0 + c1 / 2) / c1 : 0;
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
    const int tiles = q.tiles_m * q.tiles_n;
    t->split = i / tiles;
    i -= t->split * tiles;
    // groups of tile rows, all columns of a group before the next group
    const int per = q.group * q.tiles_n;
    const int g = i / per;
    const int rows = min(q.group, q.tiles_m - g * q.group);
    i -= g * per;
    t->m = g * q.group + i % rows;
    t->n = i / rows;
    return true;
  }
  __device__ void blocks(const Tile& t, int* k0, int* k1) const {
    const HeadJob& q = a.job[t.job];
    *k0 = int((long long)q.kblocks * t.split / q.splits);
    *k1 = int((long long)q.kblocks * (t.split + 1) / q.splits);
  }
};

// ---- epilogues ------------------------------------------------------------------

// Running maximum and sum of exp(x - max), of 32 more columns of which `n` exist.
__device__ __forceinline__ void online(const float (&v)[32], int n, float& m, float& s) {
  float top = m;
  if (n >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) top = fmaxf(top, v[i]);
  }
  // an infinite maximum would make inf - inf of itself: such a row's sum is formed
  // around 0 and comes out inf, or stays 0 for -inf (NaN is kept either way)
  const float base = fabsf(top) == INFINITY ? 0.f : top;
  const float old = fabsf(m) == INFINITY ? 0.f : m;
  float sum = s == 0.f ? 0.f : s * exp2_approx((old - base) * kLog2e);
  const float b2 = base * kLog2e;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < n) sum += exp2_approx(fmaf(v[i], kLog2e, -b2));
  m = top;
  s = sum;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// 32 values of one row to bfloat16, n of them (16-byte stores when the row allows it).
__device__ __forceinline__ void store_bf16(__nv_bfloat16* p, const float (&v)[32], int n) {
  if (n >= 32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      *reinterpret_cast<uint4*>(p + i) = make_uint4(pack2(v[i], v[i + 1]), pack2(v[i + 2], v[i + 3]),
                                                    pack2(v[i + 4], v[i + 5]), pack2(v[i + 6], v[i + 7]));
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) p[i] = __float2bfloat16_rn(v[i]);
  }
}
__device__ __forceinline__ void store_f32(float* p, const float (&v)[32], int n) {
  if (n >= 32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) p[i] = v[i];
  }
}

template <int EPI, int TN>
__global__ void __cluster_dims__(kHeadPair, 1, 1) __launch_bounds__(kHeadThreads, 1)
    head_kernel(const __grid_constant__ HeadLaunch a) {
  constexpr int kBytesA = kHeadTileM * 128;
  constexpr int kBytesB = TN / kHeadPair * 128;
  constexpr int kStage = kBytesA + kBytesB;
  constexpr int kStages = (192 * 1024) / kStage;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t dead_flag;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages;
  const uint32_t sums_full = empty + 8 * kStages, sums_empty = sums_full + 16;
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
  const int kPlaneA[6] = {2, 1, 0, 1, 0, 0};
  const int kPlaneB[6] = {0, 1, 2, 0, 1, 0};

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
        const int bn = t.n * TN + int(rank) * (TN / kHeadPair);
        for (int p = 6 - a.pairs; ok && p < 6; ++p)
          for (int kb = k0; kb < k1; ++kb) {
            ok = wait(empty + 8 * s, ph ^ 1);
            if (!ok) break;
            if (rank == 0) bar_expect(full + 8 * s, kHeadPair * kStage);
            const uint32_t sa = ring + s * kStage, sb = sa + kBytesA, bar = full + 8 * s;
            if (++s == kStages) {
              s = 0;
              ph ^= 1;
            }
            if (a.stall) continue;
            const int ka = q.a_k0 + kb * kHeadTileK, kk = q.b_k0 + kb * kHeadTileK;
            int pa = 0, pb = 0;
#pragma unroll
            for (int i = 0; i < 6; ++i)
              if (i == p) {
                pa = kPlaneA[i];
                pb = kPlaneB[i];
              }
            if (q.a_mn) {
#pragma unroll
              for (int i = 0; i < kHeadTileM / 64; ++i)
                tma_load(sa + i * 8192, &q.a, q.a_row0 + am + 64 * i, ka, pa, bar);
            } else {
              tma_load(sa, &q.a, ka, q.a_row0 + am, pa, bar);
            }
            if (q.b_mn) {
#pragma unroll
              for (int i = 0; i < TN / kHeadPair / 64; ++i)
                tma_load(sb + i * 8192, &q.b, q.b_row0 + bn + 64 * i, kk, pb, bar);
            } else {
              tma_load(sb, &q.b, kk, q.b_row0 + bn, pb, bar);
            }
          }
      }
      if (!ok) {  // copies in flight land before the shared memory is given up
        const uint64_t t0 = now_ns();
        while (now_ns() - t0 < 2000000) {
        }
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
        ok = wait(sums_empty + 8 * as, aph ^ 1);
        if (!ok) break;
        fence_after();
        // float32 sums of bfloat16, M 256 (both CTAs), N TN
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(q.a_mn) << 15) |
                               (uint32_t(q.b_mn) << 16) | (uint32_t(TN / 8) << 17) |
                               (uint32_t(kHeadPair * kHeadTileM / 16) << 24);
        const uint32_t step_a = q.a_mn ? 2048 / 16 : 32 / 16, step_b = q.b_mn ? 2048 / 16 : 32 / 16;
        bool add = false;
        const int steps = a.pairs * (k1 - k0);
        for (int i = 0; i < steps; ++i) {
          ok = wait(full + 8 * s, ph);
          if (!ok) break;
          fence_after();
          const uint64_t da = descriptor(ring + s * kStage, q.a_mn);
          const uint64_t db = descriptor(ring + s * kStage + kBytesA, q.b_mn);
#pragma unroll
          for (int k = 0; k < kHeadTileK / 16; ++k) {
            mma(tmem + as * TN, da + k * step_a, db + k * step_b, idesc, add);
            add = true;
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
  } else {
    Walk walk(a);
    Tile t;
    int as = 0, aph = 0;
    const int quarter = warp % 4, half = (warp - 2) / 4;
    const HeadRows& r = a.r;
    while (walk.next(&t)) {
      const HeadJob& q = a.job[t.job];
      bool ok = wait(sums_full + 8 * as, aph);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      fence_after();
      const uint32_t src = tmem + as * TN + (uint32_t(quarter * 32) << 16) + half * (TN / 2);
      const int row = (t.m * kHeadPair + int(rank)) * kHeadTileM + quarter * 32 + lane;
      const int col0 = t.n * TN + half * (TN / 2);
      if (EPI == kHeadLse) {
        const bool there = row < r.rows;
        const int y = there ? r.labels[row] : -1;
        float m = -INFINITY, sum = 0.f;
#pragma unroll 1
        for (int c = 0; c < TN / 2; c += 32) {
          float v[32];
          tmem_load(src + c, v);
          const int n = r.classes - (col0 + c);
          online(v, n, m, sum);
          if (unsigned(y - (col0 + c)) < 32u && y < r.classes) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col0 + c + i == y) x = v[i];
            r.target[row] = x;
          }
        }
        if (there) r.part[(long long)(t.n * 2 + half) * r.rows + row] = make_float2(m, sum);
      } else if (EPI == kHeadG) {
        const bool there = row < r.rows;
        const int y = there ? r.labels[row] : -1;
        const bool known = unsigned(y) < unsigned(r.classes);
        const float lse = there ? r.lse[row] : 0.f;
        const float up = known ? r.dloss[row] : 0.f;
        __nv_bfloat16* g = static_cast<__nv_bfloat16*>(r.g) + (long long)row * r.ld_g + col0;
#pragma unroll 1
        for (int c = 0; c < TN / 2; c += 32) {
          float v[32];
          tmem_load(src + c, v);
          const int v0 = r.v0 + col0 + c;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float p = exp2_approx((v[i] - lse) * kLog2e);
            if (v0 + i == y) p -= 1.f;
            v[i] = known && v0 + i < r.classes ? up * p : 0.f;
          }
          const int n = int(r.ld_g) - (col0 + c);
          if (there && n > 0) {
            store_bf16(g + c, v, n);
            if (a.pairs > 1) {
#pragma unroll
              for (int z = 1; z < 3; ++z) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
                store_bf16(g + c + z * r.plane_g, v, n);
              }
            }
          }
        }
      } else {
        const bool there = row < q.M;
        float* acc = q.acc ? q.acc + ((long long)t.split * q.M + row) * q.N + col0 : nullptr;
#pragma unroll 1
        for (int c = 0; c < TN / 2; c += 32) {
          float v[32];
          tmem_load(src + c, v);
          const int n = q.N - (col0 + c);
          if (!there || n <= 0) continue;
          if (q.acc_in) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < n) v[i] += acc[c + i];
          }
          if (!q.final) {
            store_f32(acc + c, v, n);
          } else if (q.out_f32) {
            store_f32(static_cast<float*>(q.out) + (long long)row * q.ld_out + col0 + c, v, n);
          } else {
            store_bf16(static_cast<__nv_bfloat16*>(q.out) + (long long)row * q.ld_out + col0 + c, v, n);
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_at(sums_empty + 8 * as, 0);
      as ^= 1;
      if (as == 0) aph ^= 1;
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

// Planes of bfloat16 with 16-byte aligned rows: the terms of a float32, or a copy.
template <class T>
__global__ void __launch_bounds__(256)
    head_pack_kernel(const T* src, long long rows, int cols, long long ld, const int* labels,
                     int classes, __nv_bfloat16* dst, int ldp) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * ldp) return;
  const long long r = i / ldp;
  int c = int(i - r * ldp);
  if (labels && unsigned(labels[r]) >= unsigned(classes)) c = cols;  // zeros
  if (sizeof(T) == 2) {
    const unsigned short v = c < cols ? reinterpret_cast<const unsigned short*>(src)[r * ld + c] : 0;
    reinterpret_cast<unsigned short*>(dst)[i] = v;
    return;
  }
  float v = c < cols ? reinterpret_cast<const float*>(src)[r * ld + c] : 0.f;
#pragma unroll
  for (int z = 0; z < 3; ++z) {
    const __nv_bfloat16 t = __float2bfloat16_rn(v);
    dst[z * rows * ldp + i] = t;
    v = z == 0 && !isfinite(v) ? 0.f : v - __bfloat162float(t);
  }
}

// The (max, sum) parts of a row to its log-sum-exp and loss.  A block takes `per` rows
// (a power of two, at most 32) with 256 / per threads each.
__global__ void __launch_bounds__(256)
    head_finish_kernel(const float2* part, const float* target, const int* labels, long long rows,
                       int classes, int parts, float* loss, float* lse, int per) {
  __shared__ float2 mine[256];
  const int x = threadIdx.x % per, t = threadIdx.x / per, threads = 256 / per;
  const long long n = (long long)blockIdx.x * per + x;
  float m = -INFINITY, s = 0.f;
  // s exp(m - base), with an infinite m standing for 0 as in online()
  auto term = [](float2 p, float base) {
    return p.y == 0.f ? 0.f : p.y * expf((fabsf(p.x) == INFINITY ? 0.f : p.x) - base);
  };
  auto join = [&](float2 p) {
    const float top = fmaxf(m, p.x), base = fabsf(top) == INFINITY ? 0.f : top;
    s = term(make_float2(m, s), base) + term(p, base);
    m = top;
  };
  if (n < rows)
    for (int i = t; i < parts; i += threads) join(part[i * rows + n]);
  mine[threadIdx.x] = make_float2(m, s);
  __syncthreads();
  for (int o = threads / 2; o > 0; o /= 2) {
    if (t < o) {
      join(mine[threadIdx.x + o * per]);
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

__global__ void __launch_bounds__(256) head_reduce_kernel(const HeadReduce a) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.M * a.N) return;
  float v = a.acc_in ? a.acc[i] : 0.f;
  for (int s = 0; s < a.splits; ++s) v += a.part[s * a.M * a.N + i];
  if (!a.final) {
    a.acc[i] = v;
    return;
  }
  const long long r = i / a.N, o = r * a.ld_out + (i - r * a.N);
  if (a.out_f32)
    static_cast<float*>(a.out)[o] = v;
  else
    static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(v);
}

template <int EPI, int TN>
cudaError_t go(const HeadLaunch& a, cudaStream_t s) {
  constexpr int kStage = kHeadTileM * 128 + TN / kHeadPair * 128;
  constexpr size_t smem = size_t((192 * 1024) / kStage) * kStage + 1024;
  const cudaError_t e = cudaFuncSetAttribute(head_kernel<EPI, TN>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  long long tiles = 0;
  for (int j = 0; j < a.jobs; ++j)
    tiles += (long long)a.job[j].tiles_m * a.job[j].tiles_n * a.job[j].splits;
  if (tiles <= 0) return cudaSuccess;
  const int pairs = int(std::min<long long>(tiles, device_sms() / kHeadPair));
  head_kernel<EPI, TN><<<pairs * kHeadPair, kHeadThreads, smem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_head(int epilogue, int tile_n, const HeadLaunch& a, cudaStream_t s) {
  if (epilogue == kHeadLse) return go<kHeadLse, 256>(a, s);
  if (epilogue == kHeadG) return go<kHeadG, 256>(a, s);
  return tile_n == 128 ? go<kHeadOut, 128>(a, s) : go<kHeadOut, 256>(a, s);
}

cudaError_t launch_head_pack(int dtype, const void* src, int64_t rows, int64_t cols, int64_t ld,
                             const int* labels, int64_t classes, void* dst, int64_t ldp,
                             cudaStream_t s) {
  const long long blocks = (rows * ldp + 255) / 256;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  if (dtype == kF32)
    head_pack_kernel<float><<<unsigned(blocks), 256, 0, s>>>(
        static_cast<const float*>(src), rows, int(cols), ld, labels, int(classes),
        static_cast<__nv_bfloat16*>(dst), int(ldp));
  else
    head_pack_kernel<__nv_bfloat16><<<unsigned(blocks), 256, 0, s>>>(
        static_cast<const __nv_bfloat16*>(src), rows, int(cols), ld, labels, int(classes),
        static_cast<__nv_bfloat16*>(dst), int(ldp));
  return cudaGetLastError();
}

cudaError_t launch_head_finish(const float2* part, const float* target, const int* labels,
                               int64_t rows, int64_t classes, int64_t parts, float* loss,
                               float* lse, cudaStream_t s) {
  int per = 1;
  while (per < 32 && per < rows) per *= 2;
  const long long blocks = (rows + per - 1) / per;
  head_finish_kernel<<<unsigned(blocks), 256, 0, s>>>(part, target, labels, rows, int(classes),
                                                      int(parts), loss, lse, per);
  return cudaGetLastError();
}

cudaError_t launch_head_reduce(const HeadReduce& a, cudaStream_t s) {
  const long long blocks = (a.M * a.N + 255) / 256;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  head_reduce_kernel<<<unsigned(blocks), 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace mb
