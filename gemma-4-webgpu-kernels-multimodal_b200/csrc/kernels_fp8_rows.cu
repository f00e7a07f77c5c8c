// Row operators that emit 8-bit float operands: the quantiser (with an
// optional gated activation) and the residual norm.  Both are one pass over
// HBM; sums, norms and activations are f32, each output is rounded once.
#include <algorithm>

#include "fp8_rows.cuh"
#include "g4m_kernels.h"
#include "g4m_sm100.cuh"

namespace g4m {

// ---------------------------------------------------------------------------
// Quantiser.  16 lanes hold one block (8 columns each): the block's largest
// magnitude is four shuffles, and nothing else crosses lanes.  Half-warps
// walk the blocks of all rows with the next block's loads in flight.  8192 x
// 6144 bf16 with gelu (253 MB) takes 49 us, 5.1 TB/s, 0.78 of the measured
// copy rate (55 us in a stream of calls from Python); silu 47, without
// activation (153 MB) 31.  Issue slots are close behind HBM (the sigmoid, the
// rounded quotient): magnitudes compared as integers cost 2.7 us more, a
// warp-wide reduction in place of the four shuffles 2.0.  Rows off 16-byte
// boundaries, 8191 x 6143: 82 us with gelu, 47 without activation.
// ---------------------------------------------------------------------------
constexpr int kQuantThreads = 256;

// act(x0) * x1.  The gate's sigmoid argument is scaled by -log2(e) in its
// constants: x sigmoid(z) = x / (1 + 2^(-z log2 e)).
template <int ACT>
__device__ __forceinline__ float activate(float x0, float x1) {
  float e;  // -z log2 e: z = x for silu, z = 2 sqrt(2/pi) (x + 0.044715 x^3) for gelu_tanh
  if (ACT == G4M_ACT_SILU) {
    e = x0 * -kLog2eF;
  } else {
    constexpr float k1 = -2.0f * 0.7978845608028654f * kLog2eF, k3 = k1 * 0.044715f;
    e = x0 * fmaf(k3, x0 * x0, k1);
  }
  return x0 * rcp_approx(1.0f + ex2_approx(e)) * x1;
}

template <class T, int ACT, bool FULL>
__global__ void __launch_bounds__(kQuantThreads, 5) fp8_quantize_kernel(const __grid_constant__ QuantArgs a, FastDiv blocks) {
  const int lane16 = threadIdx.x & 15;
  const uint32_t stride = gridDim.x * (kQuantThreads / 16);
  uint32_t u = blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4);
  Raw8<T, FULL> x0, x1;
  uint32_t row = 0, kb = 0;
  auto fetch = [&](uint32_t unit) {
    row = div_by(unit, blocks);
    kb = unit - row * blocks.d;
    const int c = (int)kb * kFp8Block + lane16 * 8;
    const int d = unit < a.units ? a.d : 0;  // past the end: zeros, nothing read
    const T* x = static_cast<const T*>(a.x) + (long)row * a.ldx;
    load_raw8<T, FULL>(x, c, d, x0);
    if (ACT != G4M_ACT_NONE) load_raw8<T, FULL>(x + a.d, c, d, x1);
  };
  fetch(u);
  // The two half-warps of a warp hold neighbouring blocks and stay together:
  // the warp goes on while its first has a block.
  for (; u - ((threadIdx.x >> 4) & 1) < a.units; u += stride) {
    float v[8];
    unpack8<T, FULL>(x0, v);
    if (ACT != G4M_ACT_NONE) {
      float g[8];
      unpack8<T, FULL>(x1, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = activate<ACT>(v[j], g[j]);
    }
    const uint32_t r = row, k = kb;
    fetch(u + stride);
    const float s = fp8_scale(block_amax(amax8(v)));
    if (u < a.units) {
      store_codes8<FULL>(a.codes + (long)r * a.ldc, (int)k * kFp8Block + lane16 * 8, a.d, fp8_encode8(v, s));
      if (lane16 == 0) a.scales[(long)k * a.lds + r] = s;
    }
  }
}

template <class T>
static void launch_quantize(const QuantArgs& a, int sms, cudaStream_t st) {
  const uint32_t per = kQuantThreads / 16, all = (a.units - 1) / per + 1;
  const uint32_t grid = std::min<uint32_t>(all, (uint32_t)sms * 5);
  const FastDiv blocks = fast_div((uint32_t)a.blocks);
  auto go = [&](auto kernel) { kernel<<<grid, kQuantThreads, 0, st>>>(a, blocks); };
  if (a.full) {
    if (a.act == G4M_ACT_SILU) go(fp8_quantize_kernel<T, G4M_ACT_SILU, true>);
    else if (a.act == G4M_ACT_GELU_TANH) go(fp8_quantize_kernel<T, G4M_ACT_GELU_TANH, true>);
    else go(fp8_quantize_kernel<T, G4M_ACT_NONE, true>);
  } else {
    if (a.act == G4M_ACT_SILU) go(fp8_quantize_kernel<T, G4M_ACT_SILU, false>);
    else if (a.act == G4M_ACT_GELU_TANH) go(fp8_quantize_kernel<T, G4M_ACT_GELU_TANH, false>);
    else go(fp8_quantize_kernel<T, G4M_ACT_NONE, false>);
  }
}

cudaError_t fp8_quantize(const QuantArgs& a, int dev, cudaStream_t st) {
  const int sms = g_num_sms(dev);
  if (a.dtype == G4M_F32) launch_quantize<float>(a, sms, st);
  else if (a.dtype == G4M_BF16) launch_quantize<__nv_bfloat16>(a, sms, st);
  else launch_quantize<__half>(a, sms, st);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Residual norm.  A row stays in registers from its loads to its last store:
// thread t of the row's T threads holds columns [8 (k T + t), + 8) for
// k < NCH, so 16 consecutive lanes hold one 128-column block and the e4m3
// scales need no shared memory.  The two means of squares are the only row
// sums.  Blocks walk the rows with the next row's loads in flight: with one
// row per block, loads, sums and stores took turns.  16384 x 4096 (bf16 branch,
// f32 residual, gate, codes out: 739 MB) takes 157 us, 4.7 TB/s, 0.72 of the
// measured copy rate; to bf16 rows without gate (537 MB) 96 us, 5.6 TB/s, 0.85.
// Between them stand the shuffles of the sums and block maxima and the rounded
// quotients.
// ---------------------------------------------------------------------------
struct NormKernelArgs {
  g4m_norm_args a;
  float inv_d;
  FastDiv per_gate;
};
// Sum over the threads of the row; every thread gets it.  The sums that a
// block forms one after another, of one row or of the next, alternate between
// two `part`s, so that one barrier each is enough: a part is written again
// only after the other one's barrier, which every warp reaches with its reads
// of the first behind it.
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x == 32) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = (int)(threadIdx.x & 31) < warps ? part[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);  // at most 16 warps
  return __shfl_sync(0xffffffffu, v, 0);
}

template <int NCH>
__device__ __forceinline__ float square_sum(const float (&v)[NCH][8]) {
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[k][i], v[k][i], ss);
  return ss;
}

// v = v * inv * w for the chunk at column c (w null: all ones).
template <bool FULL>
__device__ __forceinline__ void scale8(float (&v)[8], float inv, const float* w, int c, int d) {
  if (w) {
    float f[8];
    load8<FULL>(w, c, d, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (v[i] * inv) * f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv;
  }
}

// The most threads of a row, blocks an SM shall hold.  Shifting chunks into
// place (rows off 16-byte boundaries) takes registers: those rows get more
// threads with fewer chunks each, no loads ahead, and as many blocks as hide
// each other's waits (2947 x 5193 bf16: 124 us with one block of 512 threads
// an SM, 95 us with three of 384; 76 since row edges are stored by a mask).
// Three such blocks leave a thread 56 registers: with two chunks 232 to 472
// bytes of it spill, with one 16 to 104, by the types.
template <int NCH, bool FULL>
struct NormCfg {
  static constexpr int T = NCH == 4 ? 512 : FULL ? 256 : 384;
  static constexpr int BLOCKS = NCH == 4 ? 1 : FULL && NCH == 1 ? 4 : 3;
};

template <class TY, class TH, int NCH, bool FULL>
__global__ void __launch_bounds__(NormCfg<NCH, FULL>::T, NormCfg<NCH, FULL>::BLOCKS)
    norm_residual_kernel(const __grid_constant__ NormKernelArgs p) {
  __shared__ float part[2][16];
  int turn = 0;
  const g4m_norm_args& a = p.a;
  const int T = blockDim.x, t = threadIdx.x, d = a.d;
  Raw8<TY, FULL> ry[NCH];
  Raw8<TH, FULL> rh[NCH];
  auto fetch_y = [&](long row) {
    const int dd = row < a.rows && a.y ? d : 0;  // past the end: zeros, nothing read
    const TY* y = static_cast<const TY*>(a.y) + row * a.ldy;
#pragma unroll
    for (int k = 0; k < NCH; ++k) load_raw8<TY, FULL>(y, 8 * (k * T + t), dd, ry[k]);
  };
  auto fetch_h = [&](long row) {
    const int dd = row < a.rows && a.h ? d : 0;
    const TH* x = static_cast<const TH*>(a.h) + row * a.ldh;
#pragma unroll
    for (int k = 0; k < NCH; ++k) load_raw8<TH, FULL>(x, 8 * (k * T + t), dd, rh[k]);
  };
  // Rows of one warp share a block four at a time and meet no block barrier.
  const long stride = (long)gridDim.x * blockDim.y;
  long row = (long)blockIdx.x * blockDim.y + threadIdx.y;
  if (FULL) {
    fetch_y(row);
    fetch_h(row);
  }
  for (; row < a.rows; row += stride) {
    if (!FULL) {
      fetch_y(row);
      fetch_h(row);
    }
    float b[NCH][8], h[NCH][8];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      unpack8<TY, FULL>(ry[k], b[k]);
      unpack8<TH, FULL>(rh[k], h[k]);
    }
    if (FULL) fetch_y(row + stride);
    if (a.y) {
      if (a.norm_post) {
        const float inv = rsqrtf(fmaf(row_sum(square_sum<NCH>(b), part[turn ^= 1]), p.inv_d, a.eps));
#pragma unroll
        for (int k = 0; k < NCH; ++k) scale8<FULL>(b[k], inv, a.w_post, 8 * (k * T + t), d);
      }
      if (a.gate) {
        const TY* g = static_cast<const TY*>(a.gate) + (long)div_by((uint32_t)row, p.per_gate) * a.ldg;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          float f[8];
          load8<FULL>(g, 8 * (k * T + t), d, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) b[k][i] *= f[i];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) h[k][i] = a.res_scale * fmaf(a.branch_scale, b[k][i], h[k][i]);
    if (a.h_out) {
      TH* o = static_cast<TH*>(a.h_out) + row * a.ldh_out;
#pragma unroll
      for (int k = 0; k < NCH; ++k) store8<FULL>(o, 8 * (k * T + t), d, h[k]);
    }
    if (FULL) fetch_h(row + stride);  // here, where the branch's registers are free again
    if (!a.n_out && !a.out.codes) continue;
    if (a.norm_pre) {
      const float inv = rsqrtf(fmaf(row_sum(square_sum<NCH>(h), part[turn ^= 1]), p.inv_d, a.eps));
#pragma unroll
      for (int k = 0; k < NCH; ++k) scale8<FULL>(h[k], inv, a.w_pre, 8 * (k * T + t), d);
    }
    if (a.n_out) {
      TY* o = static_cast<TY*>(a.n_out) + row * a.ldn;
#pragma unroll
      for (int k = 0; k < NCH; ++k) store8<FULL>(o, 8 * (k * T + t), d, h[k]);
    }
    if (a.out.codes) {
      uint8_t* codes = a.out.codes + row * a.out.ldc;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int c = 8 * (k * T + t);
        const float s = fp8_scale(block_amax(amax8(h[k])));
        if (c < d) {
          store_codes8<FULL>(codes, c, d, fp8_encode8(h[k], s));
          if ((t & 15) == 0) a.out.scales[(long)(c / kFp8Block) * a.out.lds + row] = s;
        }
      }
    }
  }
}

// Rows that start on 16-byte boundaries, or are absent.
static bool rows16(const void* p, int64_t ld, int dtype) {
  const int64_t size = dtype == G4M_F32 ? 4 : 2;
  return !p || (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size)) % 16 == 0;
}

template <class TY, class TH, int NCH, bool FULL>
static void launch_norm(const NormKernelArgs& p, int sms, cudaStream_t st) {
  using C = NormCfg<NCH, FULL>;
  const int chunks = (p.a.d + 7) / 8, T = ((chunks + NCH - 1) / NCH + 31) / 32 * 32;
  const dim3 block(T, T == 32 ? 4 : 1);
  const long blocks = (p.a.rows + block.y - 1) / block.y;
  const long resident = (long)sms * std::max(1, C::T * C::BLOCKS / (T * (int)block.y));
  norm_residual_kernel<TY, TH, NCH, FULL><<<(unsigned)(FULL ? std::min(blocks, resident) : blocks), block, 0, st>>>(p);
}
template <class TY, class TH>
static void launch_norm_h(const NormKernelArgs& p, int sms, cudaStream_t st) {
  const g4m_norm_args& a = p.a;
  const int chunks = (a.d + 7) / 8;
  const bool full = a.d % 8 == 0 && rows16(a.y, a.ldy, a.dtype) && rows16(a.gate, a.ldg, a.dtype) && rows16(a.h, a.ldh, a.h_dtype) &&
                    rows16(a.h_out, a.ldh_out, a.h_dtype) && rows16(a.n_out, a.ldn, a.dtype) && rows16(a.w_post, 0, G4M_F32) &&
                    rows16(a.w_pre, 0, G4M_F32);
  if (full) {
    if (chunks <= 256) launch_norm<TY, TH, 1, true>(p, sms, st);
    else if (chunks <= 512) launch_norm<TY, TH, 2, true>(p, sms, st);
    else launch_norm<TY, TH, 4, true>(p, sms, st);
  } else {
    if (chunks <= 384) launch_norm<TY, TH, 1, false>(p, sms, st);
    else if (chunks <= 768) launch_norm<TY, TH, 2, false>(p, sms, st);
    else launch_norm<TY, TH, 4, false>(p, sms, st);
  }
}
template <class TY>
static void launch_norm_y(const NormKernelArgs& p, int sms, cudaStream_t st) {
  if (p.a.h_dtype == G4M_F32) launch_norm_h<TY, float>(p, sms, st);
  else if (p.a.h_dtype == G4M_BF16) launch_norm_h<TY, __nv_bfloat16>(p, sms, st);
  else launch_norm_h<TY, __half>(p, sms, st);
}

cudaError_t norm_residual(const g4m_norm_args& a, int dev, cudaStream_t st) {
  NormKernelArgs p;
  p.a = a;
  p.inv_d = 1.0f / (float)a.d;
  p.per_gate = fast_div((uint32_t)std::min<int64_t>(std::max<int64_t>(a.rows_per_gate, 1), 0x7fffffff));
  const int sms = g_num_sms(dev);
  if (a.dtype == G4M_F32) launch_norm_y<float>(p, sms, st);
  else if (a.dtype == G4M_BF16) launch_norm_y<__nv_bfloat16>(p, sms, st);
  else launch_norm_y<__half>(p, sms, st);
  return cudaGetLastError();
}

}  // namespace g4m
