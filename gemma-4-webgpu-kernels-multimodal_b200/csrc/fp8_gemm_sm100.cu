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
// Every mbarrier wait is bounded; a timeout records an error word and the
// CTA unwinds.
#include <algorithm>

#include "fp8_rows.cuh"
#include "g4m_kernels.h"
#include "g4m_sm100.cuh"

namespace g4m {

// e4m3 A and B (K-major), f32 D: the format fields are those of fp16 (0).
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) { return idesc_f16_f32(m, n); }

// D[tmem] (+)= A[smem] * B[smem]^T, kind::f8f6f4, K = 32 codes per instruction.
template <bool ACC>
__device__ __forceinline__ void mma_fp8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "n"(ACC ? 1 : 0)
      : "memory");
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The float at this CTA's shared address `addr` in the cluster's CTA `rank`.
__device__ __forceinline__ float cluster_ld(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// The producer's waits for copies that nobody has consumed after a timeout.
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
  static constexpr int STAGES = 4;
  static constexpr int EPI_STAGE = 4096;  // per epilogue warp: a 32-row x 128-byte store block
  static constexpr int THREADS = 64 + 256;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 8 * EPI_STAGE + 1024;
  static_assert(SMEM + 1024 <= 232448, "over 227 KB of shared memory");
  static constexpr int GROUP_M = 16;      // row blocks that share the output blocks in L2
};

__device__ __forceinline__ void tile_of(int tile, int tiles_m, int tiles_n, int& mb, int& nb) {
  const int group = tile / (ManyCfg::GROUP_M * tiles_n);
  const int m0 = group * ManyCfg::GROUP_M, gm = min(ManyCfg::GROUP_M, tiles_m - m0);
  const int r = tile - m0 * tiles_n;
  nb = r / gm;
  mb = m0 + r - nb * gm;
}

__global__ void __launch_bounds__(ManyCfg::THREADS, 1)
    fp8_gemm_many_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ Fp8GemmArgs a) {
  using C = ManyCfg;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::STAGES], bar_empty[C::STAGES], bar_accf[2], bar_acce[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, skip;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kblocks = (a.in + kFp8Block - 1) / kFp8Block, oblocks = (a.out + kFp8Block - 1) / kFp8Block;
  const int tiles_m = (int)((a.rows + C::BM - 1) / C::BM), tiles_n = (oblocks + 1) / 2, tiles = tiles_m * tiles_n;

  if (threadIdx.x == 0) {
    skip = *reinterpret_cast<volatile int*>(a.err) != 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_accf[b], 1);
      mbar_init(&bar_acce[b], 8);
    }
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&mx);
  }
  __syncthreads();
  if (skip) return;  // an earlier kernel on this device already failed
  if (warp == 1) tmem_alloc(&tmem_slot, 2 * C::BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        int mb, nb;
        tile_of(tile, tiles_m, tiles_n, mb, nb);
        const uint8_t* w = a.w + (long)2 * nb * kblocks * kFp8TileBytes;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&bar_empty[s], ((it / C::STAGES) & 1) ^ 1, a.err, kErrWaitEmpty, &abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * C::STAGE_BYTES;
          mbar_expect_tx(&bar_full[s], C::STAGE_BYTES);
          tma_load_2d(sa, &mx, &bar_full[s], kb * kFp8Block, mb * C::BM);
          bulk_load(sa + C::A_BYTES, w + (long)kb * kFp8TileBytes, kFp8TileBytes, &bar_full[s]);
          bulk_load(sa + C::A_BYTES + kFp8TileBytes, w + (long)(kblocks + kb) * kFp8TileBytes, kFp8TileBytes, &bar_full[s]);
        }
      }
      for (uint32_t j = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; j < it; ++j)
        drain(&bar_full[j % C::STAGES], (j / C::STAGES) & 1, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3_f32(C::BM, C::BN);
      const uint64_t dbase = desc_k_sw128(smem_u32(smem));
      uint32_t it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % C::STAGES;
          const uint32_t b = it & 1;
          if (!mbar_wait(&bar_acce[b], ((it >> 1) & 1) ^ 1, a.err, kErrWaitAccEmpty, &abort_flag) ||
              !mbar_wait(&bar_full[s], (it / C::STAGES) & 1, a.err, kErrWaitFull, &abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = desc_add(dbase, s * C::STAGE_BYTES), db = desc_add(da, C::A_BYTES);
          const uint32_t d = tmem_base + b * C::BN;
          mma_fp8_ss<false>(d, da, db, idesc);
#pragma unroll
          for (int k = 1; k < 4; ++k) mma_fp8_ss<true>(d, desc_add(da, k * 32), desc_add(db, k * 32), idesc);
          mma_commit(&bar_empty[s]);
          mma_commit(&bar_accf[b]);
        }
      }
      // The last stage-release commits land before the CTA can exit.
      if (ok && !abort_flag)
        for (uint32_t j = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; j < it; ++j)
          if (!mbar_wait(&bar_empty[j % C::STAGES], (j / C::STAGES) & 1, a.err, kErrWaitDrain, &abort_flag)) break;
    }
  } else {
    // Epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31, one row of x per
    // thread, and one half (one output block) of the tile's columns.
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint4* stage = reinterpret_cast<uint4*>(smem + C::STAGES * C::STAGE_BYTES + (warp - 2) * C::EPI_STAGE);
    const uint32_t tm = tmem_base + ((uint32_t)(32 * q) << 16) + half * 128;
    uint32_t it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      int mb, nb;
      tile_of(tile, tiles_m, tiles_n, mb, nb);
      const long row0 = (long)mb * C::BM + 32 * q;
      const float* sx = a.sx + min(row0 + lane, a.rows - 1);
      const int ob = 2 * nb + half;
      const float* sw = a.sw + (long)min(ob, oblocks - 1) * kblocks;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      float s_next = __ldg(sx) * __ldg(sw);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const float s = s_next;
        if (kb + 1 < kblocks) s_next = __ldg(sx + (long)(kb + 1) * a.lds) * __ldg(sw + kb + 1);
        const uint32_t b = it & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bar_accf[b], (it >> 1) & 1, a.err, kErrWaitAccFull, &abort_flag));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[2][16];
        tmem_ld16(tm + b * C::BN, r[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          tmem_wait16(r[c & 1]);
          if (c < 7) {
            tmem_ld16(tm + b * C::BN + 16 * (c + 1), r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_acce[b]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[16 * c + i] = fmaf(__uint_as_float(r[c & 1][i]), s, acc[16 * c + i]);
        }
      }
      if (!ok) break;
      const int col0 = ob * 128;
      if (col0 >= a.out) continue;
      const int nrows = (int)min(32l, a.rows - row0);
      if (a.bias) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (col0 + i < a.out) acc[i] += __ldg(a.bias + col0 + i);
      }
      if (nrows <= 0) continue;
      if (a.y_vec && col0 + 128 <= a.out) {
        const int size = a.y_dtype == G4M_F32 ? 4 : 2;
        char* y = static_cast<char*>(a.y) + (row0 * a.ldy + col0) * size;
        const size_t stride = (size_t)a.ldy * size;
        if (a.y_dtype == G4M_F32) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              v[i] = make_uint4(__float_as_uint(acc[32 * c + 4 * i]), __float_as_uint(acc[32 * c + 4 * i + 1]),
                                __float_as_uint(acc[32 * c + 4 * i + 2]), __float_as_uint(acc[32 * c + 4 * i + 3]));
            warp_store_block<128>(stage, v, y + c * 128, stride, nrows, lane);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float f0 = acc[64 * c + 8 * i + 2 * j], f1 = acc[64 * c + 8 * i + 2 * j + 1];
                w[j] = a.y_dtype == G4M_BF16 ? pack2(f0, f1, __nv_bfloat16()) : pack2(f0, f1, __half());
              }
              v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            warp_store_block<128>(stage, v, y + c * 128, stride, nrows, lane);
          }
        }
      } else if (lane < nrows) {
        with_type(a.y_dtype, [&](auto* tp) {
          auto* y = static_cast<decltype(tp)>(a.y) + (row0 + lane) * a.ldy + col0;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (col0 + i < a.out) from_f32(acc[i], y + i);
        });
      }
    }
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
  static constexpr int STAGES = NT == 16 ? 6 : NT == 32 ? 5 : NT == 64 ? 4 : 6;
  static constexpr int BUFS = NT == 16 ? 8 : NT == 32 ? 8 : NT == 64 ? 4 : 2;  // accumulators in flight
  static constexpr int TMEM_COLS = BUFS * NT;
  static constexpr int THREADS = 64 + 128;
  static constexpr int CTAS = NT <= 64 ? 2 : 1;  // per SM
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024;
  static_assert(NT * 128 * 4 <= STAGES * STAGE_BYTES, "the partial totals reuse the stages");
  static_assert(CTAS * TMEM_COLS <= 512 && CTAS * (SMEM + 32 * NT + 2048) <= 233472, "over the SM's memories");
};

template <int NT>
__global__ void __launch_bounds__(FewCfg<NT>::THREADS, FewCfg<NT>::CTAS)
    fp8_gemm_few_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ Fp8GemmArgs a, int splits) {
  using C = FewCfg<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::STAGES], bar_empty[C::STAGES], bar_accf[C::BUFS], bar_acce[C::BUFS];
  __shared__ __align__(16) float sc[4][2][NT];  // per epilogue warp: scale products of a block, double-buffered
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kblocks = (a.in + kFp8Block - 1) / kFp8Block;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const int ob = blockIdx.x / splits;
  const long row0 = (long)blockIdx.y * NT;
  const int nrows = (int)min((long)NT, a.rows - row0);
  const int k0 = (int)((long)kblocks * rank / splits), nk = (int)((long)kblocks * (rank + 1) / splits) - k0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < C::BUFS; ++b) {
      mbar_init(&bar_accf[b], 1);
      mbar_init(&bar_acce[b], 4);
    }
    // An earlier kernel on this device failed: nothing is waited for, but the
    // CTA still meets its cluster's barriers.
    abort_flag = *reinterpret_cast<volatile int*>(a.err) != 0;
    fence_mbar_init();
    prefetch_tmap(&mx);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const bool run = abort_flag == 0;
  __syncthreads();  // every thread has read the flag before a wait can raise it
  const int q = warp & 3, t = 32 * q + lane;  // epilogue: output ob * 128 + t
  float acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = 0.0f;

  if (warp == 0) {
    if (lane == 0 && run) {
      int it = 0;
      const uint8_t* w = a.w + ((long)ob * kblocks + k0) * kFp8TileBytes;
      for (; it < nk; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&bar_empty[s], ((it / C::STAGES) & 1) ^ 1, a.err, kErrWaitEmpty, &abort_flag)) break;
        uint8_t* sw = smem + s * C::STAGE_BYTES;
        mbar_expect_tx(&bar_full[s], C::STAGE_BYTES);
        bulk_load(sw, w + (long)it * kFp8TileBytes, C::W_BYTES, &bar_full[s]);
        tma_load_2d(sw + C::W_BYTES, &mx, &bar_full[s], (k0 + it) * kFp8Block, (int)row0);
      }
      for (int j = it > C::STAGES ? it - C::STAGES : 0; j < it; ++j)
        drain(&bar_full[j % C::STAGES], (j / C::STAGES) & 1, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0 && run) {
      constexpr uint32_t idesc = idesc_e4m3_f32(128, NT);
      const uint64_t dbase = desc_k_sw128(smem_u32(smem));
      int it = 0;
      for (; it < nk; ++it) {
        const int s = it % C::STAGES, b = it % C::BUFS;
        if (!mbar_wait(&bar_acce[b], ((it / C::BUFS) & 1) ^ 1, a.err, kErrWaitAccEmpty, &abort_flag) ||
            !mbar_wait(&bar_full[s], (it / C::STAGES) & 1, a.err, kErrWaitFull, &abort_flag))
          break;
        tc_fence_after();
        const uint64_t dw = desc_add(dbase, s * C::STAGE_BYTES), dx = desc_add(dw, C::W_BYTES);
        const uint32_t d = tmem_base + b * NT;
        mma_fp8_ss<false>(d, dw, dx, idesc);
#pragma unroll
        for (int k = 1; k < 4; ++k) mma_fp8_ss<true>(d, desc_add(dw, k * 32), desc_add(dx, k * 32), idesc);
        mma_commit(&bar_empty[s]);
        mma_commit(&bar_accf[b]);
      }
      if (it == nk)  // the last stage-release commits land before the stages are reused or the CTA exits
        for (int j = it > C::STAGES ? it - C::STAGES : 0; j < it; ++j)
          if (!mbar_wait(&bar_empty[j % C::STAGES], (j / C::STAGES) & 1, a.err, kErrWaitDrain, &abort_flag)) break;
    }
  } else if (run) {
    const uint32_t tm = tmem_base + ((uint32_t)(32 * q) << 16);
    const float* swp = a.sw + (long)ob * kblocks + k0;
    const float* sxp = a.sx + (long)k0 * a.lds + row0;
    constexpr int PER = (NT + 31) / 32;
    float nxt[PER];
    auto fetch = [&](int i) {
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int j = lane + 32 * p;
        nxt[p] = i < nk && j < nrows ? __ldg(sxp + (long)i * a.lds + j) * __ldg(swp + i) : 0.0f;
      }
    };
    fetch(0);
    for (int i = 0; i < nk; ++i) {
      float* s = sc[q][i & 1];
#pragma unroll
      for (int p = 0; p < PER; ++p)
        if (lane + 32 * p < NT) s[lane + 32 * p] = nxt[p];
      fetch(i + 1);
      __syncwarp();
      const int b = i % C::BUFS;
      if (!__all_sync(0xffffffffu, mbar_wait(&bar_accf[b], (i / C::BUFS) & 1, a.err, kErrWaitAccFull, &abort_flag))) break;
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
          const float4 f = *reinterpret_cast<const float4*>(s + 16 * c + 4 * j);
          float* o = acc + 16 * c + 4 * j;
          o[0] = fmaf(__uint_as_float(r[4 * j]), f.x, o[0]);
          o[1] = fmaf(__uint_as_float(r[4 * j + 1]), f.y, o[1]);
          o[2] = fmaf(__uint_as_float(r[4 * j + 2]), f.z, o[2]);
          o[3] = fmaf(__uint_as_float(r[4 * j + 3]), f.w, o[3]);
        }
      }
    }
  }

  const int o = ob * 128 + t;
  const float bias = warp >= 2 && o < a.out && a.bias ? __ldg(a.bias + o) : 0.0f;
  if (splits == 1) {
    if (warp >= 2 && o < a.out)
      with_type(a.y_dtype, [&](auto* tp) {
        auto* y = static_cast<decltype(tp)>(a.y) + row0 * a.ldy + o;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (j < nrows) from_f32(acc[j] + bias, y + j * a.ldy);
      });
  } else {
    // Partial totals [row][128 outputs] replace the stages, whose copies and
    // MMAs are done once every warp is here; each CTA of the cluster then
    // adds a share of the rows in rank order.
    __syncthreads();
    float* part = reinterpret_cast<float*>(smem);
    if (warp >= 2) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (j < nrows) part[j * 128 + t] = acc[j];
    }
    cluster_sync();
    const int j0 = nrows * rank / splits, j1 = nrows * (rank + 1) / splits;
    if (warp >= 2 && o < a.out)
      with_type(a.y_dtype, [&](auto* tp) {
        auto* y = static_cast<decltype(tp)>(a.y) + row0 * a.ldy + o;
        for (int j = j0; j < j1; ++j) {
          const uint32_t at = smem_u32(part + j * 128 + t);
          float v[8];
#pragma unroll
          for (int p = 0; p < 8; ++p) v[p] = p < splits ? cluster_ld(at, p) : 0.0f;
          float total = v[0];
#pragma unroll
          for (int p = 1; p < 8; ++p)
            if (p < splits) total += v[p];
          from_f32(total + bias, y + j * a.ldy);
        }
      });
    cluster_sync();  // no CTA leaves while its totals are being read
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
  return cudaFuncSetAttribute(fp8_gemm_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, FewCfg<NT>::SMEM);
}

cudaError_t fp8_gemm_setup() {
  cudaError_t e = cudaFuncSetAttribute(fp8_gemm_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ManyCfg::SMEM);
  if (e == cudaSuccess) e = setup_few<16>();
  if (e == cudaSuccess) e = setup_few<32>();
  if (e == cudaSuccess) e = setup_few<64>();
  if (e == cudaSuccess) e = setup_few<128>();
  return e;
}

template <int NT>
static cudaError_t launch_few(const Fp8GemmArgs& a, int sms, cudaStream_t st) {
  using C = FewCfg<NT>;
  CUtensorMap mx;
  if (!make_tmap_u8_pitch(&mx, a.x, a.rows, a.in, a.ldx, NT)) return cudaErrorInvalidValue;
  const long units = fp8_blocks(a.out) * ((a.rows + NT - 1) / NT), kblocks = fp8_blocks(a.in);
  // Split the column blocks until the CTAs fill the SMs.
  int splits = 1;
  while (splits < 8 && 2 * splits <= kblocks && units * splits < sms) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(fp8_blocks(a.out) * splits), (unsigned)((a.rows + NT - 1) / NT));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_few_kernel<NT>, mx, a, splits);
}

cudaError_t fp8_gemm(const Fp8GemmArgs& a, int dev, cudaStream_t st) {
  const int sms = g_num_sms(dev);
  if (a.rows <= 16) return launch_few<16>(a, sms, st);
  if (a.rows <= 32) return launch_few<32>(a, sms, st);
  if (a.rows <= 64) return launch_few<64>(a, sms, st);
  if (a.rows <= 256) return launch_few<128>(a, sms, st);
  CUtensorMap mx;
  if (!make_tmap_u8_pitch(&mx, a.x, a.rows, a.in, a.ldx, ManyCfg::BM)) return cudaErrorInvalidValue;
  const long tiles = (a.rows + ManyCfg::BM - 1) / ManyCfg::BM * ((fp8_blocks(a.out) + 1) / 2);
  if (tiles > 0x3fffffffL) return cudaErrorInvalidValue;
  fp8_gemm_many_kernel<<<(unsigned)std::min<long>(tiles, sms), ManyCfg::THREADS, ManyCfg::SMEM, st>>>(mx, a);
  return cudaGetLastError();
}

}  // namespace g4m
