// Device helpers of the 8-bit float row operators: typed loads and stores of
// eight consecutive elements, and the e4m3 encoding of a 128-column block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "fp8_ops.h"

namespace g4m {

__device__ __forceinline__ void unpack2(uint32_t w, __nv_bfloat16, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, __half, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* p) { *p = __float2half_rn(v); }

// Elements [c, c + 8) of a row of d, zeros from d on.  vec: the row starts on
// a 16-byte boundary (c is a multiple of 8).
__device__ __forceinline__ void load8(const float* row, int c, int d, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= d) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < d ? row[c + i] : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void load8(const T* row, int c, int d, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= d) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + c);
    unpack2(a.x, T(), v[0], v[1]);
    unpack2(a.y, T(), v[2], v[3]);
    unpack2(a.z, T(), v[4], v[5]);
    unpack2(a.w, T(), v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < d ? to_f32(row[c + i]) : 0.0f;
  }
}
__device__ __forceinline__ void store8(float* row, int c, int d, bool vec, const float (&v)[8]) {
  if (vec && c + 8 <= d) {
    *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) row[c + i] = v[i];
  }
}
template <class T>
__device__ __forceinline__ void store8(T* row, int c, int d, bool vec, const float (&v)[8]) {
  if (vec && c + 8 <= d) {
    *reinterpret_cast<uint4*>(row + c) =
        make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) from_f32(v[i], row + c + i);
  }
}

// Runs f(T*) for the element type `dtype` names.  The branch is uniform over
// the grid and stands outside the unrolled loads, so they stay in flight
// together.
template <class F>
__device__ __forceinline__ void with_type(int dtype, F f) {
  if (dtype == G4M_F32) f(static_cast<float*>(nullptr));
  else if (dtype == G4M_BF16) f(static_cast<__nv_bfloat16*>(nullptr));
  else f(static_cast<__half*>(nullptr));
}

// Bits of the largest magnitude of v.  Magnitudes compare as integers, and
// there infinities and NaN come above every finite value, so a block that
// holds one keeps it.
__device__ __forceinline__ uint32_t amax_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
// Over the 16 lanes that hold one block of 128 columns (all 32 lanes call).
__device__ __forceinline__ uint32_t block_amax_bits(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// scale = max(amax, 2^-96) / 448; the floor keeps the scale of an all-zero
// block (and its reciprocal) a normal number.  NaN for a block that is not
// finite.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  return __fdiv_rn(fmaxf(__uint_as_float(amax_bits), 0x1p-96f), 448.0f);
}

// Eight codes e4m3(v / s), to nearest even.  The quotient is v * (1/s)
// corrected by its fma residual (Markstein, IBM J. Res. Develop. 34(1),
// 1990), which gives the rounded quotient in three operations: the codes are
// those of a true division.
__device__ __forceinline__ uint2 fp8_encode8(const float (&v)[8], float s) {
  const float inv = __frcp_rn(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float x = v[2 * i + j], q0 = x * inv;
      q[j] = fmaf(fmaf(-q0, s, x), inv, q0);
    }
    uint16_t p;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(q[1]), "f"(q[0]));
    w[i] = p;
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Codes [c, c + 8) of a row of d codes that starts on a 16-byte boundary.
__device__ __forceinline__ void store_codes8(uint8_t* row, int c, int d, uint2 w) {
  if (c + 8 <= d) {
    *reinterpret_cast<uint2*>(row + c) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) row[c + i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

}  // namespace g4m
