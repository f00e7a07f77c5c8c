// Block-scaled 8-bit float linear on tcgen05:
//   y[r][o] = sum over 128-column blocks k of
//               (x[r, k] . w[o, k]) * sx[k][r] * sw[o / 128][k]   (+ bias[o])
//
// The tensor core forms the code products of one 128-column block (four
// kind::f8f6f4 MMAs of K = 32, f32 accumulation) from zero in tensor memory;
// the epilogue warps multiply that block sum by its two scales and add it to
// a running f32 total in registers.  No rounding but f32's happens before the
// one at the store.  Two kernels share this scheme:
//
//   many rows  rows of x on the 128 TMEM lanes, 256 outputs per tile: the
//              scale product is one number per thread and block.
//   few rows   outputs on the 128 lanes, NT rows of x in the columns, and the
//              column blocks split over a thread-block cluster: the weights
//              stream through all SMs, and the partial totals meet through
//              distributed shared memory in rank order, so nothing depends on
//              the order of arrival.
//
// What bounds them (B200, device time in a captured graph, weights from HBM).
// Many rows: 8192 x 4096 -> 8192 bf16 takes 259 us (2.12 PFLOP/s), in a stream
// of calls, where the power cap holds the clock, 303 us (1.81 PFLOP/s); a bf16
// library product of that size would take 332 us at its measured 1.65 PFLOP/s.
// The MMAs of a block take 512 cycles; its sums cross to the epilogue and back
// (issue 130, MMAs and their arrival 600, loads and half of the sums 330, two
// wake-ups of about 200) in about 1300 with two accumulators to hide them, and
// the f32 pipe is busy for 330.  TMEM holds no third accumulator of 256
// columns.  A call of quarter units alone takes about 5 us and 0.26 us for
// each column block (100 x 1536 -> 6144 8.3 us, 65 x 4096 -> 4096 13.6);
// halves take longer (512 x 4096 -> 4096 16.3).  Few rows: 1 x 4096 -> 32768
// takes 24 us, 5.5 TB/s; below about 20 MB of weights a call is launch, set-up
// (0.9 us), first bytes (0.8 us) and the cluster's exchange (0.7 us).
//
// Every mbarrier wait is bounded; a timeout records an error word and the
// CTA unwinds.
#include <algorithm>

#include "fp8_rows.cuh"
#include "g4m_kernels.h"
#include "g4m_sm100.cuh"

namespace g4m {

// e4m3 A and B (K-major), f32 D: the format fields are those of fp16 (0).
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) { return idesc_f16_f32(m, n); }

// One 128-column block: D[tmem] = A[smem] * B[smem]^T (kind::f8f6f4, four
// MMAs of K = 32 codes), then an arrival on `bar` when they are done.  Whole
// warp; one elected lane issues.  With the warp converged the descriptors
// stay in uniform registers: 157 cycles for the five instructions, where a
// single-lane branch takes 228.
__device__ __forceinline__ void mma_block(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a1, b1, a2, b2, a3, b3;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\t"
      "add.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
      "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
      "setp.ne.b32 p, 0, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, p;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(smem_u32(bar))
      : "memory");
}

// Whether the phase is complete, without waiting (try_wait may suspend the thread).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait of a whole warp: the same answer in every lane.  A test takes
// 75-140 cycles even when the phase is complete, so loops test the next
// iteration's barrier early (`ready`, from mbar_test) and only read the
// answer here.
__device__ __forceinline__ bool warp_wait(bool ready, uint64_t* bar, uint32_t parity, int* err, int code,
                                          volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, ready)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code, abort_flag));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code, volatile int* abort_flag) {
  return warp_wait(mbar_try_wait(smem_u32(bar), parity), bar, parity, err, code, abort_flag);
}

// 16 columns of this warp's lanes; the values are there after tmem_wait16.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Waits for this thread's TMEM loads.  r passes through, so no use of the
// loaded values can be moved before the wait.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
// The same for four sets.
__device__ __forceinline__ void tmem_wait64(uint32_t (&r)[4][16]) {
  tmem_wait16(r[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[j][i])::"memory");
}

// A tile of this CTA's shared memory to global memory (the map's box and swizzle);
// rows past the tensor's edge are not written, nor columns past the 16 bytes
// that its last column lies in.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// All but this thread's last N stores have read their shared memory; all are complete.
template <int N>
__device__ __forceinline__ void tma_store_read_wait() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 4 bytes from global to shared memory without a register; zero unless `valid`.
__device__ __forceinline__ void cp_async4(float* dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
// Orders nothing but the arrival itself (a release would wait for this thread's global stores).
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// Shared address `addr` of this CTA in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
// Copies `bytes` (a multiple of 16) of this CTA's shared memory into that of a
// CTA of the cluster, where they count towards the phase of a barrier.  One
// copy per CTA: an asynchronous store per thread and row cost 400 cycles each
// on the barrier's account.
__device__ __forceinline__ void cluster_push(uint32_t remote, const void* src, uint32_t bytes, uint32_t remote_bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(remote),
               "r"(smem_u32(src)), "r"(bytes), "r"(remote_bar)
               : "memory");
}

// Waits for what is still on its way after a timeout: copies that nobody has
// consumed, MMAs whose sums nobody takes, totals from the cluster.  A CTA that
// left before would let them write memory that is no longer its own.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t b = smem_u32(bar);
  const long long t0 = clock64();
  while (!mbar_try_wait(b, parity)) {
    if (clock64() - t0 > kWaitCycles) {
      atomicCAS(err, 0, kErrWaitDrain);
      break;
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------
struct ManyCfg {
  static constexpr int BM = 128, BN = 256;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // Four stages, and for every epilogue warp two 32-row x 64-byte blocks on
  // their way to y.  (Three stages and blocks of 128 bytes: 512 x 4096 -> 4096
  // 21.0 -> 22.5 us.)
  static constexpr int STAGES = 4;
  static constexpr int EPI_BLOCK = 2048, EPI_STAGE = 2 * EPI_BLOCK;
  // One warpgroup for the producer, the MMA issuer and the two scale warps,
  // two for the epilogue.  The registers of a launch at 168 a thread are
  // shared out as 56 and 216: 128 * 56 + 256 * 216 <= 384 * 168.  (Sixteen
  // epilogue warps of 64 columns took as long.)
  static constexpr int EPI_WARPS = 8, THREADS = 128 + 32 * EPI_WARPS;
  static constexpr int SCALE_SLOTS = 2;  // blocks whose scale products are in shared memory
  static constexpr int SCALE_BYTES = SCALE_SLOTS * 2 * BM * 4;
  static constexpr int BARS = 2 * STAGES + 2 + SCALE_SLOTS;
  // No static shared memory: the stages start the block's share, which begins
  // on a 1024-byte boundary (the kernel checks), and nothing is spent on
  // rounding up.
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * EPI_STAGE + SCALE_BYTES + 8 * BARS + 16;
  static_assert(SMEM <= 232448, "over 227 KB of shared memory");
  static constexpr int GROUP_M = 16;  // row blocks that share the output blocks in L2 (4 to 32 take the same time)
};

__device__ __forceinline__ void tile_of(int tile, int tiles_m, int tiles_n, int& mb, int& nb) {
  const int group = tile / (ManyCfg::GROUP_M * tiles_n);
  const int m0 = group * ManyCfg::GROUP_M, gm = min(ManyCfg::GROUP_M, tiles_m - m0);
  const int r = tile - m0 * tiles_n;
  nb = r / gm;
  mb = m0 + r - nb * gm;
}

// Tiles [0, full) go round the CTAs whole.  The rest, at most SMs >> LG of
// them, are cut into 2^LG units of 256 >> LG outputs, one for a CTA, its last.
// A kernel for each LG: the narrow epilogues beside the wide one cost it 2 to
// 5 % (8192 x 4096 -> 8192 255 and 261 us).
template <int LG>
__global__ void __launch_bounds__(ManyCfg::THREADS, 1)
    fp8_gemm_many_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap my,
                         const __grid_constant__ Fp8GemmArgs a, const int full) {
  using C = ManyCfg;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  float* scales = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + C::EPI_WARPS * C::EPI_STAGE);
  uint64_t *bar_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(scales) + C::SCALE_BYTES),
           *bar_done = bar_full + C::STAGES, *bar_acce = bar_done + C::STAGES, *bar_scale = bar_acce + 2;
  volatile uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bar_full + C::BARS);
  volatile int& abort_flag = *reinterpret_cast<int*>(bar_full + C::BARS + 1);
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrShape);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kblocks = (a.in + kFp8Block - 1) / kFp8Block, oblocks = (a.out + kFp8Block - 1) / kFp8Block;
  const int tiles_m = (int)((a.rows + C::BM - 1) / C::BM), tiles_n = (oblocks + 1) / 2, tiles = tiles_m * tiles_n;
  // This CTA's share: whole tiles blockIdx.x, + gridDim.x, ..., then maybe a unit.
  const int cta = (int)blockIdx.x, ctas = (int)gridDim.x, last = LG ? full : tiles;
  const int whole = last > cta ? (last - 1 - cta) / ctas + 1 : 0;
  const bool unit = LG > 0 && cta < (tiles - full) << LG;
  const int share = whole + unit;
  constexpr int WIDTH = C::BN >> LG;
  // Row block, and first output, of the i-th of the share.
  auto place_of = [&](int i, int& mb, int& col) {
    const bool cut = LG > 0 && i >= whole;
    int nb;
    tile_of(cut ? full + (cta >> LG) : cta + i * ctas, tiles_m, tiles_n, mb, nb);
    col = nb * C::BN + (cut ? (cta & ((1 << LG) - 1)) * WIDTH : 0);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_done[s], 1);
    }
    for (int b = 0; b < 2; ++b) mbar_init(&bar_acce[b], C::EPI_WARPS);
    for (int s = 0; s < C::SCALE_SLOTS; ++s) mbar_init(&bar_scale[s], 2);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&mx);
  if (warp == 1) tmem_alloc(const_cast<uint32_t*>(&tmem_slot), 2 * C::BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int i = 0; i < share && ok; ++i) {
        int mb, col;
        place_of(i, mb, col);
        const uint8_t* w = a.w + (long)(col / kFp8Block) * kblocks * kFp8TileBytes + col % kFp8Block * 128;
        const bool two = LG == 0 || i < whole;  // both output blocks, or part of one
        const int bytes = two ? kFp8TileBytes : WIDTH * 128;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&bar_done[s], ((it / C::STAGES) & 1) ^ 1, a.err, kErrWaitEmpty, &abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * C::STAGE_BYTES;
          mbar_expect_tx(&bar_full[s], C::A_BYTES + (two ? C::B_BYTES : bytes));
          tma_load_2d(sa, &mx, &bar_full[s], kb * kFp8Block, mb * C::BM);
          bulk_load(sa + C::A_BYTES, w + (long)kb * kFp8TileBytes, bytes, &bar_full[s]);
          if (two) bulk_load(sa + C::A_BYTES + kFp8TileBytes, w + (long)(kblocks + kb) * kFp8TileBytes, kFp8TileBytes, &bar_full[s]);
        }
      }
      for (uint32_t j = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; j < it; ++j)
        drain(&bar_full[j % C::STAGES], (j / C::STAGES) & 1, a.err);
    }
    if (warp == 1) {
      // bar_done of a stage tells both that the stage is free and that the
      // block's sums are complete.
      const uint64_t dbase = desc_k_sw128(smem_u32(smem));
      uint32_t it = 0;
      bool full = false, free = true;  // tested ahead
      auto issue = [&](long until, uint32_t idesc) {
        for (; it < until; ++it) {
          const int s = it % C::STAGES;
          const uint32_t b = it & 1;
          const uint64_t da = desc_add(dbase, s * C::STAGE_BYTES);
          if (!warp_wait(full, &bar_full[s], (it / C::STAGES) & 1, a.err, kErrWaitFull, &abort_flag) ||
              !warp_wait(free, &bar_acce[b], ((it >> 1) & 1) ^ 1, a.err, kErrWaitAccEmpty, &abort_flag))
            return false;
          tc_fence_after();
          mma_block(tmem_base + b * C::BN, da, desc_add(da, C::A_BYTES), idesc, &bar_done[s]);
          full = mbar_test(&bar_full[(it + 1) % C::STAGES], ((it + 1) / C::STAGES) & 1);
          free = mbar_test(&bar_acce[b ^ 1], (((it + 1) >> 1) & 1) ^ 1);
        }
        return true;
      };
      const bool ok = issue((long)whole * kblocks, idesc_e4m3_f32(C::BM, C::BN));
      if (unit && ok) issue((long)share * kblocks, idesc_e4m3_f32(C::BM, WIDTH));
      // Whatever became of the epilogue, the CTA outlives its MMAs.
      if (lane == 0 && it > 0) drain(&bar_done[(it - 1) % C::STAGES], ((it - 1) / C::STAGES) & 1, a.err);
    }
    if (warp >= 2) {
      // Scale products of one output block (half of the tile): slot it % 2
      // takes sx[row] * sw for the 128 rows once the epilogue is done with
      // block it - 2, the slot's last.  Loads run two blocks ahead, into the
      // next tile, too.  In the epilogue's own threads these loads and their
      // bookkeeping took 200 cycles of every block.
      const int half = warp - 2;
      const long total = (long)share * kblocks;
      int i = 0, kb = 0;  // what is fetched next
      const float *sw = nullptr, *sx[4] = {};
      float x[2][4], w[2];
      auto fetch = [&](int to) {
        if (kb == 0) {
          int mb, col;
          place_of(min(i, share - 1), mb, col);
          sw = a.sw + (long)min(col / kFp8Block + (LG == 0 || i < whole ? half : 0), oblocks - 1) * kblocks;
#pragma unroll
          for (int j = 0; j < 4; ++j) sx[j] = a.sx + min((long)mb * C::BM + 32 * j + lane, a.rows - 1);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[to][j] = __ldg(sx[j] + (long)kb * a.lds);
        w[to] = __ldg(sw + kb);
        if (++kb == kblocks) kb = 0, ++i;
      };
      uint32_t it = 0;
      auto put = [&](int from) {
        if (!warp_wait(&bar_acce[it & 1], ((it >> 1) & 1) ^ 1, a.err, kErrWaitAccEmpty, &abort_flag)) return false;
        float* to = scales + (it % C::SCALE_SLOTS) * 2 * C::BM + half * C::BM + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) to[32 * j] = x[from][j] * w[from];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_scale[it % C::SCALE_SLOTS]);
        ++it;
        fetch(from);
        return true;
      };
      fetch(0);
      fetch(1);
      while (it < total) {
        if (!put(0)) break;
        if (it < total && !put(1)) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // Epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31, one row of x per
    // thread, and one half (one output block) of the tile's columns.
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stage = smem + C::STAGES * C::STAGE_BYTES + (warp - 4) * C::EPI_STAGE;
    const uint32_t lanes = tmem_base + ((uint32_t)(32 * q) << 16);
    const float* scale = scales + half * C::BM + 32 * q + lane;
    uint32_t it = 0;
    bool ok = true, done = false, scaled = false;  // the next block's barriers, tested ahead
    // Blocks of y sent by TMA so far, over all tiles: consecutive ones always
    // take turns between the warp's two store blocks, so that all but the last
    // store being read is enough before a block is written again, even after
    // a tile that y's right edge left an odd number of blocks.
    uint32_t sends = 0;
    // One of the share, COLS columns for this warp.
    auto complete = [&](int i, auto cols) {
      constexpr int COLS = decltype(cols)::value;
      int mb, col0;
      place_of(i, mb, col0);
      const long row0 = (long)mb * C::BM + 32 * q;
      col0 += half * COLS;
      const uint32_t tm = lanes + half * COLS;
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
      if (a.bias) {  // padded with zeros to whole tiles
        const float4* bp = reinterpret_cast<const float4*>(a.bias + col0);
#pragma unroll
        for (int i = 0; i < COLS / 4; ++i) {
          const float4 f = __ldg(bp + i);
          acc[4 * i] = f.x, acc[4 * i + 1] = f.y, acc[4 * i + 2] = f.z, acc[4 * i + 3] = f.w;
        }
      }
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const uint32_t b = it & 1, src = tm + b * C::BN;
        ok = warp_wait(scaled, &bar_scale[it % C::SCALE_SLOTS], (it / C::SCALE_SLOTS) & 1, a.err, kErrWaitFull, &abort_flag) &&
             warp_wait(done, &bar_done[it % C::STAGES], (it / C::STAGES) & 1, a.err, kErrWaitAccFull, &abort_flag);
        if (!ok) break;
        const float s = scale[(it % C::SCALE_SLOTS) * 2 * C::BM];
        tc_fence_after();
        // 16 columns at a time through four register blocks: the buffer goes
        // back to the MMA issuer once the last block is loaded, with half of
        // the sums still to be added.  (Single fma: pairs of f32 in one
        // instruction took 14 % longer here.)
        uint32_t r[4][16] = {};
        auto load = [&](int c) { tmem_ld16(src + 16 * c, r[c & 3]); };
        auto add = [&](int c) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[16 * c + i] = fmaf(__uint_as_float(r[c & 3][i]), s, acc[16 * c + i]);
        };
#pragma unroll
        for (int c = 0; c < COLS / 16 && c < 4; ++c) load(c);
        tmem_wait64(r);
        if constexpr (COLS > 64) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            add(c);
            load(c + 4);
          }
          tmem_wait64(r);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_acce[b]);
        done = mbar_test(&bar_done[(it + 1) % C::STAGES], ((it + 1) / C::STAGES) & 1);
        scaled = mbar_test(&bar_scale[(it + 1) % C::SCALE_SLOTS], ((it + 1) / C::SCALE_SLOTS) & 1);
#pragma unroll
        for (int c = COLS > 64 ? 4 : 0; c < COLS / 16; ++c) add(c);
      }
      if (!ok) return;
      const int nrows = (int)min(32l, a.rows - row0);
      if (nrows <= 0 || col0 >= a.out) return;
      // 16 columns (f32) or 32 (16 bits) at a time: 64 bytes of each of the
      // warp's 32 rows go through shared memory, 16-byte chunk c of row r at
      // c ^ (r / 2 & 3), and out by TMA while the next ones are packed.
      // Rows of y that do not start on 16-byte boundaries, and the block that
      // the last column ends inside 16 bytes (a TMA store writes the whole 16),
      // leave by plain stores, a warp's lanes side by side in a row.  (From the
      // lane that holds the row, 8192 x 4096 -> 8192 took three times as long.)
      auto send = [&](const uint4 (&o)[4], int col, int size) {
        const bool tma = a.y_vec && (col + 64 / size <= a.out || a.out % (16 / size) == 0);
        uint8_t* block = stage + (sends & 1) * C::EPI_BLOCK;
        if (lane == 0) tma_store_read_wait<1>();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(block + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = o[i];
        if (tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&my, block, col, (int)row0);
          ++sends;
          return;
        }
        __syncwarp();
        const int per = 64 / size, e = lane % per, at = e * size;  // columns of a row, this lane's
        for (int r = lane / per; r < nrows; r += 32 / per) {
          char* y = static_cast<char*>(a.y) + ((row0 + r) * a.ldy + col) * size;
          const uint8_t* from = block + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 15);
          if (col + e < a.out) {
            if (size == 4) reinterpret_cast<uint32_t*>(y)[e] = *reinterpret_cast<const uint32_t*>(from);
            else reinterpret_cast<uint16_t*>(y)[e] = *reinterpret_cast<const uint16_t*>(from);
          }
        }
        __syncwarp();
      };
      if (a.y_dtype == G4M_F32) {
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          if (col0 + 16 * c >= a.out) break;
          uint4 o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[i] = make_uint4(__float_as_uint(acc[16 * c + 4 * i]), __float_as_uint(acc[16 * c + 4 * i + 1]),
                              __float_as_uint(acc[16 * c + 4 * i + 2]), __float_as_uint(acc[16 * c + 4 * i + 3]));
          send(o, col0 + 16 * c, 4);
        }
      } else {
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
          if (col0 + 32 * c >= a.out) break;
          uint4 o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float f0 = acc[32 * c + 8 * i + 2 * j], f1 = acc[32 * c + 8 * i + 2 * j + 1];
              w[j] = a.y_dtype == G4M_BF16 ? pack2(f0, f1, __nv_bfloat16()) : pack2(f0, f1, __half());
            }
            o[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          send(o, col0 + 32 * c, 2);
        }
      }
    };
    for (int i = 0; i < whole && ok; ++i) complete(i, std::integral_constant<int, 128>());
    if constexpr (LG > 0) {
      if (unit && ok) complete(whole, std::integral_constant<int, WIDTH / 2>());
    }
    if (lane == 0) tma_store_wait();
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * C::BN);
  }
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
template <int NT>
struct FewCfg {
  static constexpr int W_BYTES = kFp8TileBytes, X_BYTES = NT * 128;
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
  // Two CTAs fit an SM.  (Twice the stages for grids of one CTA per SM gained
  // nothing, and cost half a microsecond a launch.)
  static constexpr int STAGES = NT == 16 ? 5 : 4;
  // One accumulator per stage: bar_done of a stage stands for both, and no
  // wait on it can fall a whole turn behind.
  static constexpr int TMEM_COLS = 128;
  static constexpr int SCALE_BLOCKS = NT == 16 ? 8 : 4;  // column blocks whose row scales are fetched together
  static constexpr int SCALE_BYTES = 4 * 2 * SCALE_BLOCKS * NT * 4;     // per epilogue warp, double-buffered
  static constexpr int PART_BYTES = NT * 128 * 4;  // partial totals from the cluster: splits * ceil(rows / splits) <= NT rows, splits a power of 2
  static constexpr int BARS = 3 * STAGES + 1;
  static constexpr int THREADS = 192;
  static constexpr int SMEM = STAGES * STAGE_BYTES + SCALE_BYTES + PART_BYTES + 1024;
  static_assert(STAGES * NT <= TMEM_COLS, "an accumulator per stage");
  static_assert(NT * 512 <= STAGES * STAGE_BYTES, "the outgoing totals reuse the stages");
  static_assert(2 * TMEM_COLS <= 512 && 2 * (SMEM + 1024 + 512) <= 233472, "over the SM's memories");
};

// n rows: the S partial totals, [rank][row][128], added in rank order.
template <int S, class T>
__device__ __forceinline__ void add_parts(const float* part, int n, float bias, T* y, long ldy) {
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    float total = part[j * 128];
#pragma unroll
    for (int p = 1; p < S; ++p) total += part[(p * n + j) * 128];
    from_f32(total + bias, y + j * ldy);
  }
}

template <int NT>
__global__ void __launch_bounds__(FewCfg<NT>::THREADS, 2)
    fp8_gemm_few_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ Fp8GemmArgs a, int lg) {
  using C = FewCfg<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[C::BARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kblocks = (a.in + kFp8Block - 1) / kFp8Block;
  // The cluster's CTAs split the column blocks: 2^lg of them, so that nothing
  // here is a division.
  const int splits = 1 << lg, rank = lg ? (int)cluster_rank() : 0;
  const int ob = blockIdx.x >> lg;
  const long row0 = (long)blockIdx.y * NT;
  const int nrows = (int)min((long)NT, a.rows - row0);
  const int k0 = (int)((long)kblocks * rank >> lg), nk = (int)((long)kblocks * (rank + 1) >> lg) - k0;
  // The rows that this CTA of the cluster completes.
  const int j0 = nrows * rank >> lg, j1 = nrows * (rank + 1) >> lg;
  float* part = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES);

  // bar_done of a stage tells both that the stage is free and that the block's
  // sums are complete.
  uint64_t *bar_full = bars, *bar_done = bars + C::STAGES, *bar_acce = bars + 2 * C::STAGES, *bar_part = bars + C::BARS - 1;
  if (threadIdx.x < C::BARS) {
    mbar_init(bars + threadIdx.x, bars + threadIdx.x >= bar_acce && bars + threadIdx.x < bar_part ? 4 : 1);
    fence_mbar_init();
    if (splits > 1 && bars + threadIdx.x == bar_part) mbar_expect_tx(bar_part, (uint32_t)(splits * (j1 - j0) * 512));
    if (threadIdx.x == 0) abort_flag = 0;
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&mx);
  if (warp == 1) tmem_alloc(&tmem_slot, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (splits > 1) cluster_arrive();  // this CTA's barriers can be reached from the others
  const uint32_t tmem_base = tmem_slot;
  // Epilogue: output ob * 128 + t, all rows of the tile.
  const int q = warp & 3, t = 32 * q + lane;
  uint64_t acc[NT / 2];  // row pairs
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) acc[i] = 0;

  if (warp == 0) {
    if (lane == 0) {
      const uint8_t* w = a.w + ((long)ob * kblocks + k0) * kFp8TileBytes;
      int it = 0;
      for (; it < nk; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&bar_done[s], ((it / C::STAGES) & 1) ^ 1, a.err, kErrWaitEmpty, &abort_flag)) break;
        uint8_t* sw = smem + s * C::STAGE_BYTES;
        mbar_expect_tx(&bar_full[s], C::STAGE_BYTES);
        bulk_load(sw, w + (long)it * kFp8TileBytes, C::W_BYTES, &bar_full[s]);
        tma_load_2d(sw + C::W_BYTES, &mx, &bar_full[s], (k0 + it) * kFp8Block, (int)row0);
      }
      for (int j = max(it - C::STAGES, 0); j < it; ++j) drain(&bar_full[j % C::STAGES], (j / C::STAGES) & 1, a.err);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_e4m3_f32(128, NT);
    const uint64_t dbase = desc_k_sw128(smem_u32(smem));
    int it = 0;
    for (; it < nk; ++it) {
      const int s = it % C::STAGES;
      const uint32_t turn = (it / C::STAGES) & 1;
      const uint64_t dw = desc_add(dbase, s * C::STAGE_BYTES);
      if (!warp_wait(&bar_acce[s], turn ^ 1, a.err, kErrWaitAccEmpty, &abort_flag) ||
          !warp_wait(&bar_full[s], turn, a.err, kErrWaitFull, &abort_flag))
        break;
      tc_fence_after();
      mma_block(tmem_base + s * NT, dw, desc_add(dw, C::W_BYTES), idesc, &bar_done[s]);
    }
    // Whatever became of the epilogue, the CTA outlives its MMAs.
    if (lane == 0 && it > 0) drain(&bar_done[(it - 1) % C::STAGES], ((it - 1) / C::STAGES) & 1, a.err);
  } else {
    const uint32_t tm = tmem_base + ((uint32_t)(32 * q) << 16);
    const float* swp = a.sw + (long)ob * kblocks + k0;
    const float* sxp = a.sx + (long)k0 * a.lds + row0;
    // Row scales come a few column blocks at a time, one fetch ahead; the
    // weight scales of 32 blocks sit in the lanes.
    constexpr int SB = C::SCALE_BLOCKS;
    float* sc = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + C::PART_BYTES) + (warp - 2) * 2 * SB * NT;
    auto fetch = [&](int g) {
#pragma unroll
      for (int p = 0; p < SB * NT / 32; ++p) {
        const int e = lane + 32 * p, i = g * SB + e / NT, j = e % NT;
        const bool valid = i < nk && j < nrows;
        cp_async4(sc + (g & 1) * SB * NT + e, valid ? sxp + (long)i * a.lds + j : sxp, valid);
      }
      cp_async_commit();
    };
    fetch(0);
    float wl = 0.0f, wn = lane < nk ? __ldg(swp + lane) : 0.0f;
    for (int i = 0; i < nk; ++i) {
      if ((i & 31) == 0) {
        wl = wn;
        wn = i + 32 + lane < nk ? __ldg(swp + i + 32 + lane) : 0.0f;
      }
      if (i % SB == 0) {
        __syncwarp();  // every lane is done with the fetch before last
        fetch(i / SB + 1);
        cp_async_wait<1>();
        __syncwarp();
      }
      const float w = __shfl_sync(0xffffffffu, wl, i & 31);
      const uint64_t ww = pack_f32x2(w, w);
      const float* s = sc + (i / SB & 1) * SB * NT + i % SB * NT;
      const int b = i % C::STAGES;
      if (!warp_wait(&bar_done[b], (i / C::STAGES) & 1, a.err, kErrWaitAccFull, &abort_flag)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < NT / 16; ++c) {
        uint32_t r[16];
        tmem_ld16(tm + b * NT + 16 * c, r);
        tmem_wait16(r);
        if (c == NT / 16 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_acce[b]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(s + 16 * c + 4 * j);
          fma_f32x2(acc[8 * c + 2 * j], pack_u32x2(r[4 * j], r[4 * j + 1]), mul_f32x2(f.x, ww));
          fma_f32x2(acc[8 * c + 2 * j + 1], pack_u32x2(r[4 * j + 2], r[4 * j + 3]), mul_f32x2(f.y, ww));
        }
      }
    }
    cp_async_wait<0>();
  }

  const int o = ob * 128 + t;
  const float bias = warp >= 2 && a.bias ? __ldg(a.bias + o) : 0.0f;  // padded with zeros to whole tiles
  if (splits == 1) {
    if (warp >= 2 && o < a.out)
      with_type(a.y_dtype, [&](auto* tp) {
        auto* y = static_cast<decltype(tp)>(a.y) + row0 * a.ldy + o;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float v[2];
          unpack_f32x2(acc[j / 2], v[0], v[1]);
          if (j < nrows) from_f32(v[j & 1] + bias, y + j * a.ldy);
        }
      });
  } else {
    // Each CTA completes a share of the rows: all copy their partial totals of
    // those rows ([row][128 outputs]) into its shared memory, and it adds them
    // in rank order.  The stages hold the outgoing totals: their copies and
    // MMAs are done.
    bool ok = true;
    if (warp >= 2) {
      float* own = reinterpret_cast<float*>(smem) + t;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float v[2];
        unpack_f32x2(acc[j / 2], v[0], v[1]);
        if (j < nrows) own[j * 128] = v[j & 1];
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 128;" ::: "memory");
    }
    cluster_wait();
    if (warp >= 2) {
      if (warp == 2 && lane < splits) {
        const int begin = nrows * lane >> lg, n = (nrows * (lane + 1) >> lg) - begin;
        if (n > 0)
          cluster_push(cluster_map(smem_u32(part + rank * n * 128), lane), smem + begin * 512, n * 512,
                       cluster_map(smem_u32(bar_part), lane));
      }
      __syncwarp();
      ok = warp_wait(bar_part, 0, a.err, kErrWaitAccFull, &abort_flag);
      if (!ok && lane == 0) drain(bar_part, 0, a.err);
      if (ok && o < a.out)
        with_type(a.y_dtype, [&](auto* tp) {
          auto* y = static_cast<decltype(tp)>(a.y) + (row0 + j0) * a.ldy + o;
          if (lg == 1) add_parts<2>(part + t, j1 - j0, bias, y, a.ldy);
          else if (lg == 2) add_parts<4>(part + t, j1 - j0, bias, y, a.ldy);
          else add_parts<8>(part + t, j1 - j0, bias, y, a.ldy);
        });
    }
    // No CTA leaves while another one may still push to it.
    cluster_arrive_relaxed();
    cluster_wait();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Weight tiles
// ---------------------------------------------------------------------------
// Chunk c of row r of a tile lies at chunk c ^ (r & 7) of that row: the
// 128-byte swizzle that the operand descriptors expect.
__global__ void __launch_bounds__(256) fp8_weight_tiles_kernel(const uint8_t* __restrict__ w, int out, int in, int kblocks,
                                                               uint8_t* __restrict__ tiles) {
  const long tile = blockIdx.x;
  const int ob = (int)(tile / kblocks), kb = (int)(tile - (long)ob * kblocks);
  for (int i = threadIdx.x; i < 1024; i += 256) {
    const int r = i >> 3, c = i & 7;
    const int o = ob * 128 + r, k = kb * 128 + c * 16;
    __align__(16) uint8_t b[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) b[j] = o < out && k + j < in ? w[(long)o * in + k + j] : 0;
    *reinterpret_cast<uint4*>(tiles + tile * kFp8TileBytes + r * 128 + ((c ^ (r & 7)) << 4)) = *reinterpret_cast<const uint4*>(b);
  }
}

cudaError_t fp8_weight_tiles(const uint8_t* w, int out, int in, uint8_t* tiles, cudaStream_t st) {
  const long n = fp8_weight_bytes(out, in) / kFp8TileBytes;
  if (n > 0x7fffffffL) return cudaErrorInvalidValue;
  fp8_weight_tiles_kernel<<<(unsigned)n, 256, 0, st>>>(w, out, in, (int)fp8_blocks(in), tiles);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
template <int NT>
static cudaError_t setup_few() {
  using C = FewCfg<NT>;
  return cudaFuncSetAttribute(fp8_gemm_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
}

template <int LG>
static cudaError_t setup_many() {
  return cudaFuncSetAttribute(fp8_gemm_many_kernel<LG>, cudaFuncAttributeMaxDynamicSharedMemorySize, ManyCfg::SMEM);
}

cudaError_t fp8_gemm_setup() {
  cudaError_t e = setup_many<0>();
  if (e == cudaSuccess) e = setup_many<1>();
  if (e == cudaSuccess) e = setup_many<2>();
  if (e == cudaSuccess) e = setup_few<16>();
  if (e == cudaSuccess) e = setup_few<32>();
  return e;
}

template <int NT>
static cudaError_t launch_few(const Fp8GemmArgs& a, int sms, cudaStream_t st) {
  using C = FewCfg<NT>;
  CUtensorMap mx;
  if (!make_tmap_u8_pitch(&mx, a.x, a.rows, a.in, a.ldx, NT)) return cudaErrorInvalidValue;
  const long row_tiles = (a.rows + NT - 1) / NT, units = fp8_blocks(a.out) * row_tiles, kblocks = fp8_blocks(a.in);
  // Split the column blocks while the CTAs stay about as many as the SMs and
  // keep four blocks each, or fewer where they would leave most SMs idle.
  // (1 x 4096 -> 4096: 11.3 us unsplit, 8.2 / 6.8 / 7.5 split by 2 / 4 / 8;
  // 1 x 1536 -> 12288, 96 CTAs unsplit: 7.1, and 8.1 split by 2; 1 x 768 -> 768:
  // 4.5, and 3.9 split by 4.)
  int lg = 0;
  while (lg < 3 && (units << (lg + 1)) <= sms + sms / 8 && (2 << lg) <= kblocks &&
         ((8 << lg) <= kblocks || (units << (lg + 3)) <= sms))
    ++lg;
  const int splits = 1 << lg;
  if (units * splits > 0x7fffffffL || row_tiles > 65535) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(fp8_blocks(a.out) * splits), (unsigned)row_tiles);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_few_kernel<NT>, mx, a, lg);
}

cudaError_t fp8_gemm(const Fp8GemmArgs& a, int dev, cudaStream_t st) {
  const int sms = g_num_sms(dev);
  // Up to 32 rows the weights are read once either way, and the few-rows
  // kernel is the faster one (16 x 4096 -> 9000: 10.4 us, and 22.9 in tiles of
  // 128 rows; 32 x 768 -> 2304: 5.5 and 5.0).  Beyond, only where it can split
  // a long sum over clusters (100 x 4096 -> 1536: 10.0 and 13.7; 64 x 4096 ->
  // 4096: 10.6 and 13.8), not unsplit (65 x 4096 -> 4096: 13.7 and 13.6; 100 x
  // 1536 -> 6144: 8.9 and 8.3) nor for a short one (64 x 768 -> 768: 5.5 and
  // 5.2).
  if (a.rows <= 16) return launch_few<16>(a, sms, st);
  if (a.rows <= 32 || (fp8_blocks(a.in) >= 8 && fp8_blocks(a.out) * ((a.rows + 31) / 32) * 2 <= sms + sms / 8))
    return launch_few<32>(a, sms, st);
  CUtensorMap mx, my;
  if (!make_tmap_u8_pitch(&mx, a.x, a.rows, a.in, a.ldx, ManyCfg::BM)) return cudaErrorInvalidValue;
  if (!a.y_vec) my = mx;  // not used
  else if (!make_tmap_out(&my, a.y, a.rows, a.out, a.ldy, a.y_dtype == G4M_F32 ? 4 : 2, 32)) return cudaErrorInvalidValue;
  const long tiles = (a.rows + ManyCfg::BM - 1) / ManyCfg::BM * ((fp8_blocks(a.out) + 1) / 2);
  if (tiles > 0x3fffffffL) return cudaErrorInvalidValue;
  // What does not fill the SMs once more is cut to use them all: narrower
  // units are done and stored sooner (2304 x 768 -> 2304, 148 + 14 tiles: 15.3
  // us whole, 13.2 in halves, 12.8 in quarters; 512 x 4096 -> 4096, 64 tiles:
  // 19.1 whole, 16.3 in halves).
  const int rest = (int)(tiles % sms);
  const int lg = 4 * rest <= sms ? 2 : 2 * rest <= sms ? 1 : 0;
  const int full = (int)tiles - rest, grid = tiles >= sms ? sms : rest << lg;
  auto go = [&](auto kernel) { kernel<<<grid, ManyCfg::THREADS, ManyCfg::SMEM, st>>>(mx, my, a, full); };
  if (rest == 0 || lg == 0) go(fp8_gemm_many_kernel<0>);
  else if (lg == 1) go(fp8_gemm_many_kernel<1>);
  else go(fp8_gemm_many_kernel<2>);
  return cudaGetLastError();
}

}  // namespace g4m
