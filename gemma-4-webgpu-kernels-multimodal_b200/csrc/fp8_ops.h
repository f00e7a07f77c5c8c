// Kernel launch interface of the 8-bit float operators (C ABI in fp8_ops.cu).
// All launchers are asynchronous on `st`.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/g4m.h"

namespace g4m {

constexpr int kFp8Block = 128;  // columns of a row (and rows of a weight block) that share one scale

struct QuantArgs {
  const void* x;
  long ldx;
  uint32_t units;  // rows * blocks
  int d, blocks, act, dtype, vec;
  uint8_t* codes;
  long ldc;
  float* scales;
  long lds;
};
cudaError_t fp8_quantize(const QuantArgs& a, cudaStream_t st);

constexpr int kNormMaxD = 16384;
cudaError_t norm_residual(const g4m_norm_args& a, cudaStream_t st);

struct RopeArgs {
  const uint64_t* turns;  // [rotary / 2] turns per position, 0.64 fixed point
  float scale;
  int head_dim, half;     // half = rotary / 2
  int interleaved, dtype, vec, pos64;
  g4m_rope_view v[2];     // v[1].heads == 0: one view
  int copy[2];            // elements from `rotary` on have to be copied
  long tokens;
  const void* positions;
  int token_block, head_slices;  // filled in by the launcher
};
cudaError_t rope_run(RopeArgs a, cudaStream_t st);

struct Fp8GemmArgs {
  long rows;
  int in, out;
  const uint8_t* x;
  long ldx;
  const float* sx;
  long lds;
  const uint8_t* w;
  const float* sw;
  const float* bias;
  void* y;
  int y_dtype;
  long ldy;
  int* err;
};
cudaError_t fp8_gemm(const Fp8GemmArgs& a, cudaStream_t st);

}  // namespace g4m
