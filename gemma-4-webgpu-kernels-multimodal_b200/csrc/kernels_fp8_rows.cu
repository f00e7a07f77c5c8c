// Row operators that emit 8-bit float operands: the quantiser (with an
// optional gated activation) and the residual norm.  Both are one pass over
// HBM; sums, norms and activations are f32, each output is rounded once.
#include <algorithm>

#include "fp8_rows.cuh"
#include "g4m_sm100.cuh"

namespace g4m {

// ---------------------------------------------------------------------------
// Quantiser.  16 lanes hold one block (8 columns each): the block's largest
// magnitude is four shuffles, and nothing else crosses lanes.  Each half-warp
// takes kQuantUnroll blocks, all of whose loads are issued before the first
// is used.
// ---------------------------------------------------------------------------
constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 2;

template <int ACT>
__device__ __forceinline__ float activate(float x0, float x1) {
  if (ACT == G4M_ACT_SILU) return x0 * sigmoid_f(x0) * x1;
  // gelu_tanh(x) = x sigmoid(2 u), u = sqrt(2/pi) (x + 0.044715 x^3)
  const float u = 0.7978845608028654f * (x0 + 0.044715f * x0 * x0 * x0);
  return x0 * sigmoid_f(2.0f * u) * x1;
}

template <class T, int ACT>
__global__ void __launch_bounds__(kQuantThreads) fp8_quantize_kernel(QuantArgs a) {
  constexpr int PER = kQuantThreads / 16;
  const int lane16 = threadIdx.x & 15;
  const uint32_t u0 = blockIdx.x * (PER * kQuantUnroll) + (threadIdx.x >> 4);
  float v[kQuantUnroll][8], g[kQuantUnroll][8];
  uint32_t row[kQuantUnroll], kb[kQuantUnroll];
#pragma unroll
  for (int i = 0; i < kQuantUnroll; ++i) {
    const uint32_t u = u0 + i * PER;
    row[i] = u / (uint32_t)a.blocks;
    kb[i] = u - row[i] * (uint32_t)a.blocks;
    const int c = (int)kb[i] * kFp8Block + lane16 * 8;
    const int d = u < a.units ? a.d : 0;  // past the end: zeros, nothing read
    const T* x = static_cast<const T*>(a.x) + (long)row[i] * a.ldx;
    load8(x, c, d, a.vec & 1, v[i]);
    if (ACT != G4M_ACT_NONE) load8(x + a.d, c, d, a.vec & 2, g[i]);
  }
#pragma unroll
  for (int i = 0; i < kQuantUnroll; ++i) {
    if (ACT != G4M_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = activate<ACT>(v[i][j], g[i][j]);
    }
    const float s = fp8_scale(block_amax_bits(amax_bits8(v[i])));
    if (u0 + i * PER < a.units) {
      store_codes8(a.codes + (long)row[i] * a.ldc, (int)kb[i] * kFp8Block + lane16 * 8, a.d, fp8_encode8(v[i], s));
      if (lane16 == 0) a.scales[(long)kb[i] * a.lds + row[i]] = s;
    }
  }
}

template <class T>
static void launch_quantize(const QuantArgs& a, cudaStream_t st) {
  constexpr uint32_t per = kQuantThreads / 16 * kQuantUnroll;
  const uint32_t grid = (a.units - 1) / per + 1;
  if (a.act == G4M_ACT_SILU) fp8_quantize_kernel<T, G4M_ACT_SILU><<<grid, kQuantThreads, 0, st>>>(a);
  else if (a.act == G4M_ACT_GELU_TANH) fp8_quantize_kernel<T, G4M_ACT_GELU_TANH><<<grid, kQuantThreads, 0, st>>>(a);
  else fp8_quantize_kernel<T, G4M_ACT_NONE><<<grid, kQuantThreads, 0, st>>>(a);
}

cudaError_t fp8_quantize(const QuantArgs& a, cudaStream_t st) {
  if (a.dtype == G4M_F32) launch_quantize<float>(a, st);
  else if (a.dtype == G4M_BF16) launch_quantize<__nv_bfloat16>(a, st);
  else launch_quantize<__half>(a, st);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Residual norm.  A row stays in registers from its loads to its last store:
// thread t of the row's T threads holds columns [8 (k T + t), + 8) for
// k < NCH, so 16 consecutive lanes hold one 128-column block and the e4m3
// scales need no shared memory.  The two means of squares are the only row
// sums.
// ---------------------------------------------------------------------------
struct NormKernelArgs {
  g4m_norm_args a;
  uint32_t vec;  // which row sets start on 16-byte boundaries (bits below)
};
enum : uint32_t { kVecY = 1, kVecGate = 2, kVecH = 4, kVecHOut = 8, kVecN = 16, kVecPost = 32, kVecPre = 64 };

// Sum over the threads of the row; every thread gets it.
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
__device__ __forceinline__ void scale8(float (&v)[8], float inv, const float* w, int c, int d, bool vec) {
  if (w) {
    float f[8];
    load8(w, c, d, vec, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (v[i] * inv) * f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv;
  }
}

template <int NCH>
__global__ void __launch_bounds__(512) norm_residual_kernel(const __grid_constant__ NormKernelArgs p) {
  __shared__ float part[2][16];
  const g4m_norm_args& a = p.a;
  const int T = blockDim.x, t = threadIdx.x, d = a.d;
  const long row = blockIdx.x;
  float b[NCH][8], h[NCH][8];
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) b[k][i] = h[k][i] = 0.0f;
  if (a.y)
    with_type(a.dtype, [&](auto* tp) {
      auto* y = static_cast<decltype(tp)>(const_cast<void*>(a.y)) + row * a.ldy;
#pragma unroll
      for (int k = 0; k < NCH; ++k) load8(y, 8 * (k * T + t), d, p.vec & kVecY, b[k]);
    });
  if (a.h)
    with_type(a.h_dtype, [&](auto* tp) {
      auto* x = static_cast<decltype(tp)>(const_cast<void*>(a.h)) + row * a.ldh;
#pragma unroll
      for (int k = 0; k < NCH; ++k) load8(x, 8 * (k * T + t), d, p.vec & kVecH, h[k]);
    });
  if (a.y) {
    if (a.norm_post) {
      const float inv = 1.0f / sqrtf(row_sum(square_sum<NCH>(b), part[0]) / (float)d + a.eps);
#pragma unroll
      for (int k = 0; k < NCH; ++k) scale8(b[k], inv, a.w_post, 8 * (k * T + t), d, p.vec & kVecPost);
    }
    if (a.gate)
      with_type(a.dtype, [&](auto* tp) {
        auto* g = static_cast<decltype(tp)>(const_cast<void*>(a.gate)) + row / a.rows_per_gate * a.ldg;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          float f[8];
          load8(g, 8 * (k * T + t), d, p.vec & kVecGate, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) b[k][i] *= f[i];
        }
      });
  }
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) h[k][i] = a.res_scale * fmaf(a.branch_scale, b[k][i], h[k][i]);
  if (a.h_out)
    with_type(a.h_dtype, [&](auto* tp) {
      auto* o = static_cast<decltype(tp)>(a.h_out) + row * a.ldh_out;
#pragma unroll
      for (int k = 0; k < NCH; ++k) store8(o, 8 * (k * T + t), d, p.vec & kVecHOut, h[k]);
    });
  if (!a.n_out && !a.out.codes) return;
  if (a.norm_pre) {
    const float inv = 1.0f / sqrtf(row_sum(square_sum<NCH>(h), part[1]) / (float)d + a.eps);
#pragma unroll
    for (int k = 0; k < NCH; ++k) scale8(h[k], inv, a.w_pre, 8 * (k * T + t), d, p.vec & kVecPre);
  }
  if (a.n_out)
    with_type(a.dtype, [&](auto* tp) {
      auto* o = static_cast<decltype(tp)>(a.n_out) + row * a.ldn;
#pragma unroll
      for (int k = 0; k < NCH; ++k) store8(o, 8 * (k * T + t), d, p.vec & kVecN, h[k]);
    });
  if (a.out.codes) {
    uint8_t* codes = a.out.codes + row * a.out.ldc;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = 8 * (k * T + t);
      const float s = fp8_scale(block_amax_bits(amax_bits8(h[k])));
      if (c < d) {
        store_codes8(codes, c, d, fp8_encode8(h[k], s));
        if ((t & 15) == 0) a.out.scales[(long)(c / kFp8Block) * a.out.lds + row] = s;
      }
    }
  }
}

static bool rows16(const void* p, int64_t ld, int dtype) {
  const int64_t size = dtype == G4M_F32 ? 4 : 2;
  return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size)) % 16 == 0;
}

cudaError_t norm_residual(const g4m_norm_args& a, cudaStream_t st) {
  NormKernelArgs p;
  p.a = a;
  p.vec = (rows16(a.y, a.ldy, a.dtype) ? kVecY : 0) | (rows16(a.gate, a.ldg, a.dtype) ? kVecGate : 0) |
          (rows16(a.h, a.ldh, a.h_dtype) ? kVecH : 0) | (rows16(a.h_out, a.ldh_out, a.h_dtype) ? kVecHOut : 0) |
          (rows16(a.n_out, a.ldn, a.dtype) ? kVecN : 0) | (rows16(a.w_post, 0, G4M_F32) ? kVecPost : 0) |
          (rows16(a.w_pre, 0, G4M_F32) ? kVecPre : 0);
  const int chunks = (a.d + 7) / 8;
  const unsigned grid = (unsigned)a.rows;
  auto threads = [&](int nch) { return std::max(32, ((chunks + nch - 1) / nch + 31) / 32 * 32); };
  if (chunks <= 512) norm_residual_kernel<1><<<grid, threads(1), 0, st>>>(p);
  else if (chunks <= 1024) norm_residual_kernel<2><<<grid, threads(2), 0, st>>>(p);
  else norm_residual_kernel<4><<<grid, threads(4), 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace g4m
