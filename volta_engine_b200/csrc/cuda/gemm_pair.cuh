// Matrix products on pairs of CTAs (tcgen05 cta_group::2) with 32-bit sums that do not lose bits along K.
//
//   D[m, n] = sum over operand pairs (a, b) and over k of A_a[m, k] * B_b[n, k]
//
// Tile: 256 x 256 a pair (or 256 x 64), each CTA holds 128 rows of A, 128 of the 256 rows of B and 128 x 256 of the sums. A step of 64 along K brings
// 32 KB to each CTA for 512 cycles of its tensor core, half of what a 128 x 256 tile of one CTA asks of L2. Either operand is K-major
// ([rows, K]) or MN-major ([K, rows]).
//
// Sums. The tensor core cuts each addition to its accumulator off instead of rounding it: against 64 bits a sum over K = 5120 of random
// products is 5.6e-6 off (4.7e-6 of that too small), over 16384 it is 1.9e-5, where fp32 FMAs are 7e-7 and 1.5e-6 off; over 128 it is 1.2e-7, and
// pieces of 512 added in fp32 are 4.8e-7 off whatever K is. So a sum stays in tensor memory for `chunk` steps only; two buffers alternate, and eight
// warps add each finished piece to registers (128 sums a thread) with ordinary rounding while the next one runs (456 cycles a piece of 256 columns; a
// step of 64 along K is 512).
//
// Operands of more than bf16 precision come as slabs: an fp32 value is the exact sum of three bf16 values (8 + 8 + 8 bits), and the product
// is summed over the pairs of slabs whose orders add up to two at most (what is left out is below 2^-24 of the product).
//
// Roles (384 threads a CTA): warp 0 loads by TMA, warp 1 of the pair's first CTA issues the MMAs, warps 4..11 sum and run the epilogue. The first
// warp group gives registers to the others: 128 x 40 + 256 x 232 = 384 x 168. Every wait is bounded.
#pragma once
#include "common.cuh"

namespace ve {

// A tile is 256 rows x NT columns, 256 or, for logits of few tiles, 64: four times the pairs have work, and a thread finishes 32 columns in place of 128.
template <int NT>
struct PairShape {
  static constexpr int kA = 128 * 128, kB = NT / 2 * 128;                           // bytes of a step and slab in a CTA: 128 rows x 64 of A, NT / 2 of B
  static constexpr int kCols = NT / 2;                                              // of a thread
};
constexpr int kPairRing = 6 * (PairShape<256>::kA + PairShape<256>::kB);
constexpr int kPairStages = kPairRing / (PairShape<64>::kA + PairShape<64>::kB);    // most steps in the ring
constexpr int kPairStaging = 8 * 4096;                     // behind the ring: a box of each summing warp's stores
constexpr int kPairSmem = kPairRing + kPairStaging + 1024;
static_assert(kPairSmem <= 227 * 1024 - 512, "shared memory (beside the barriers)");
constexpr int kPairClusters = 74, kPairThreads = 384;

VE_DEVINL uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
VE_DEVINL uint32_t first_cta_addr(const void* p) {          // the same shared-memory object in the pair's first CTA
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
VE_DEVINL void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// (Without the release at cluster scope, which waits for the thread's stores, 1300 cycles: what has been read from tensor memory is ordered by its fences.)
VE_DEVINL void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A load into this CTA's shared memory that reports to a barrier of the pair's first CTA.
VE_DEVINL void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// A warp's box of 32 rows x ROW = 128 or 64 bytes (`w`: those of the lane's row; the map's swizzle is as wide) to a tensor, through the warp's 4 KB of
// shared memory: a thread's own stores would be 16 bytes of 32 different rows each. ADD: added to what stands there (fp32, in L2). Asynchronous.
template <bool ADD, int ROW = 128>
VE_DEVINL void put_box(const CUtensorMap* map, uint8_t* staging, const uint32_t* w, int x, int y, int z) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");       // the box in front has been read
  __syncwarp();
#pragma unroll
  for (int j = 0; j < ROW / 16; ++j)
    *reinterpret_cast<uint4*>(staging + lane * ROW + ((j ^ (ROW == 128 ? lane & 7 : (lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (ADD)
      asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];"
                   ::"l"(map), "r"(smem_u32(staging)), "r"(x), "r"(y), "r"(z) : "memory");
    else
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                   ::"l"(map), "r"(smem_u32(staging)), "r"(x), "r"(y), "r"(z) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// The warp's boxes are written (before its CTA ends).
VE_DEVINL void put_wait() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
VE_DEVINL void tmem_alloc_pair(uint32_t* smem_holder, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_holder)), "r"(ncols) : "memory");
}
VE_DEVINL void tmem_relinquish_pair() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
VE_DEVINL void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrive on the barrier at this address in both CTAs when the MMAs issued so far are complete.
VE_DEVINL void tc_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
VE_DEVINL void tc_mma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// What one tile covers. Rows and columns count from the operands' own origins; steps of 64 along K.
struct PairTile {
  int m0, n0;                 // first row / column of the tile
  int k0, ksteps;             // first step and number of steps
  int split;
};

// A step brings `na` slabs of A and `nb` of B and multiplies the pairs of them that are listed.
struct PairLoop {
  int na, nb;
  int pairs;
  uint32_t a_slab, b_slab;    // four bits each
  int chunk;                  // steps that a sum stays in tensor memory
};

// The pairs (i, j) of `sa` x `sb` slabs with i + j <= order, the small ones first: what is cut off a sum is cut by its size, so a step that is a piece by
// itself loses as little as one of its first slabs alone. All pairs of a step work on one load of it (6 of 3 x 3 slabs: half of what the pairs one
// after another would bring).
static inline PairLoop pair_loop(int sa, int sb, int order, int chunk) {
  PairLoop l{sa < order + 1 ? sa : order + 1, sb < order + 1 ? sb : order + 1, 0, 0, 0, chunk};
  for (int o = order; o >= 0; --o)
    for (int i = 0; i < l.na; ++i) {
      const int j = o - i;
      if (j < 0 || j >= l.nb) continue;
      l.a_slab |= (uint32_t)i << (4 * l.pairs);
      l.b_slab |= (uint32_t)j << (4 * l.pairs);
      ++l.pairs;
    }
  return l;
}

// Job: gives the tiles (int tiles(), PairTile tile(int i)), what a thread loads in front of its sums (Row begin(tile, row of the tile, first column))
// and takes the sums: finish(tile, row of the tile, first column, Row, sums[NT / 2], omap, 4 KB of shared memory of the warp).
// A_MN / B_MN: the operand is MN-major.
// wait(): the point behind which other kernels' results are read.
// ONE: one slab of either operand, known to the compiler (3 to 4 % of a step's time).
template <int NT, bool A_MN, bool B_MN, bool ONE, class Job, class Wait>
VE_DEVINL void pair_gemm(const Job& job, const PairLoop& loop, const CUtensorMap* amap, const CUtensorMap* bmap, const CUtensorMap* omap, int* status, Wait wait) {
  static_assert(NT == 256 || !B_MN, "64 columns of an MN-major operand are one box of a CTA");
  using S = PairShape<NT>;
  constexpr int kCols = S::kCols;
  const int na = ONE ? 1 : loop.na, nb = ONE ? 1 : loop.nb, stage_bytes = na * S::kA + nb * S::kB, stages = kPairRing / stage_bytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_holder;
  __shared__ int s_fail;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 16); }
    s_fail = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc_pair(&tmem_holder, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // the pair's barriers stand before either CTA signals them
  tc_fence_after();
  const uint32_t tmem_base = tmem_holder;
  wait();
  const int ntiles = job.tiles();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && elect_one()) {
      prefetch_tmap(amap);
      prefetch_tmap(bmap);
      int s = 0, phase = 1;
      bool ok = true;
      for (int t = cluster; t < ntiles && ok; t += clusters) {
        const PairTile tl = job.tile(t);
        const int am = tl.m0 + rank * 128, bn = tl.n0 + rank * kCols;
        for (int k = 0; k < tl.ksteps; ++k) {
          ok = mbar_wait(&empty[s], phase);
          if (!ok) break;
          uint8_t* st = smem + s * stage_bytes;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * stage_bytes);
          const uint32_t bar = first_cta_addr(&full[s]);
          const int kk = (tl.k0 + k) * 64;
          for (int i = 0; i < na; ++i, st += S::kA) {
            if (A_MN) {
              tma_load_3d_pair(st, amap, bar, am, kk, i);
              tma_load_3d_pair(st + S::kA / 2, amap, bar, am + 64, kk, i);
            } else {
              tma_load_3d_pair(st, amap, bar, kk, am, i);
            }
          }
          for (int j = 0; j < nb; ++j, st += S::kB) {
            if (B_MN) {
              tma_load_3d_pair(st, bmap, bar, bn, kk, j);
              tma_load_3d_pair(st + S::kB / 2, bmap, bar, bn + 64, kk, j);
            } else {
              tma_load_3d_pair(st, bmap, bar, kk, bn, j);
            }
          }
          if (++s == stages) { s = 0; phase ^= 1; }
        }
      }
      if (!ok) atomicExch(&s_fail, 1);
    } else if (warp == 1 && rank == 0 && elect_one()) {
      constexpr uint32_t idesc = make_idesc_f16(1, 1, 256, NT) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
      int s = 0, phase = 0, piece = 0;
      bool ok = true;
      for (int t = cluster; t < ntiles && ok; t += clusters) {
        const int total = job.tile(t).ksteps;
        for (int i = 0; i < total && ok; ++piece) {
          const int buf = piece & 1;
          ok = mbar_wait(&acc_empty[buf], ((piece >> 1) & 1) ^ 1);
          if (!ok) break;
          tc_fence_after();
          const int end = min(total, i + loop.chunk);
          for (uint32_t add = 0; i < end; ++i) {
            ok = mbar_wait(&full[s], phase);
            if (!ok) break;
            tc_fence_after();
            const uint32_t st = smem_u32(smem + s * stage_bytes), bs = st + na * S::kA;
            for (int p = 0; p < (ONE ? 1 : loop.pairs); ++p) {
              const uint32_t a = ONE ? st : st + ((loop.a_slab >> (4 * p)) & 15) * S::kA, b = ONE ? bs : bs + ((loop.b_slab >> (4 * p)) & 15) * S::kB;
#pragma unroll
              for (int kb = 0; kb < 4; ++kb) {
                const uint64_t ad = A_MN ? make_desc_sw128_mn(a + kb * 2048, S::kA / 2, 1024) : make_desc_sw128(a) + kb * 2;
                const uint64_t bd = B_MN ? make_desc_sw128_mn(b + kb * 2048, S::kB / 2, 1024) : make_desc_sw128(b) + kb * 2;
                tc_mma_f16_pair(tmem_base + buf * NT, ad, bd, idesc, add);
                add = 1;
              }
            }
            tc_commit_pair(&empty[s]);
            if (++s == stages) { s = 0; phase ^= 1; }
          }
          if (ok) tc_commit_pair(&acc_full[buf]);
        }
      }
      if (!ok) atomicExch(&s_fail, 1);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * kCols;
    int piece = 0;
    bool ok = true;
    const auto begin = [&](int t) { return job.begin(job.tile(t), rank * 128 + quarter * 32 + lane, half * kCols); };
    decltype(begin(0)) row{};
    if (cluster < ntiles) row = begin(cluster);
    for (int t = cluster; t < ntiles; t += clusters) {
      const PairTile tl = job.tile(t);
      const int pieces = (tl.ksteps + loop.chunk - 1) / loop.chunk;
      float acc[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int c = 0; c < pieces; ++c, ++piece) {
        const int buf = piece & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (piece >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < kCols / 32; ++g) {
          uint32_t r[32];
          tmem_ld32(taddr + buf * NT + g * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[g * 32 + j] += __uint_as_float(r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(first_cta_addr(&acc_empty[buf]));
      }
      if (!ok) break;
      const auto now = row;
      if (t + clusters < ntiles) row = begin(t + clusters);  // (what the next tile's rows need is under way while this one's are finished)
      job.finish(tl, rank * 128 + quarter * 32 + lane, half * kCols, now, acc, omap, smem + kPairRing + (warp - 4) * 4096);
    }
    put_wait();
    if (!ok) atomicExch(&s_fail, 1);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // no CTA leaves while its pair may still signal or read it
  if (warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc_pair(tmem_base, 512); }
  if (threadIdx.x == 0 && s_fail && status) atomicExch(status, (int)kErrMbarTimeout);
}

}  // namespace ve
