// Kernel launch interface of the 8-bit float operators (C ABI in fp8_ops.cu).
// All launchers are asynchronous on `st`.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/g4m.h"

namespace g4m {

constexpr int kFp8MaxCols = 1 << 24;  // keeps column arithmetic far inside 32 bits
constexpr int kFp8Block = 128;  // columns of a row (and rows of a weight block) that share one scale

struct QuantArgs {
  const void* x;
  long ldx;
  uint32_t units;  // rows * blocks
  int d, blocks, act, dtype;
  int full;               // rows (both halves) start on 16-byte boundaries and hold whole chunks of 8
  uint8_t* codes;
  long ldc;
  float* scales;
  long lds;
};
cudaError_t fp8_quantize(const QuantArgs& a, int dev, cudaStream_t st);

constexpr int kNormMaxD = 16384;
cudaError_t norm_residual(const g4m_norm_args& a, int dev, cudaStream_t st);

struct RopeArgs {
  const uint64_t* turns;  // [rotary / 2] turns per position, 0.64 fixed point
  float scale;
  int head_dim, half;     // half = rotary / 2
  int interleaved, dtype, vec, pos64;
  g4m_rope_view v[2];     // v[1].heads == 0: one view
  int copy[2];            // elements from `rotary` on have to be copied
  long tokens;
  const void* positions;
};
cudaError_t rope_run(const RopeArgs& a, int dev, cudaStream_t st);

// Weights live in HBM as the tiles the tensor core reads: 128 outputs x 128
// columns of codes, 16 KB each, in the 128-byte-swizzled order of shared
// memory, [output block][column block], zeros past the edges.  A tile is one
// contiguous copy.  The output blocks are padded to an even number.
constexpr int kFp8TileBytes = kFp8Block * kFp8Block;
inline long fp8_blocks(long n) { return (n + kFp8Block - 1) / kFp8Block; }
inline long fp8_weight_bytes(long out, long in) { return (fp8_blocks(out) + 1) / 2 * 2 * fp8_blocks(in) * kFp8TileBytes; }
// w: codes [out][in] on the device.
cudaError_t fp8_weight_tiles(const uint8_t* w, int out, int in, uint8_t* tiles, cudaStream_t st);

struct Fp8GemmArgs {
  long rows;
  int in, out;
  const uint8_t* x;  // codes [rows][ldx], fetched through a tensor map
  long ldx;
  const float* sx;   // [blocks of in][lds]
  long lds;
  const uint8_t* w;  // tiles
  const float* sw;   // [blocks of out][blocks of in]
  const float* bias; // [blocks of out, padded to an even number, x 128], zeros past out; or null
  void* y;
  int y_dtype, y_vec;  // y_vec: rows of y start on 16-byte boundaries
  long ldy;
  int* err;
};
// Once per device before the first fp8_gemm: shared-memory limits (loads the kernels, too).
cudaError_t fp8_gemm_setup();
cudaError_t fp8_gemm(const Fp8GemmArgs& a, int dev, cudaStream_t st);

}  // namespace g4m
