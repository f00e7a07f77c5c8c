// Device helpers of the 8-bit float row operators: typed loads and stores of
// eight consecutive elements, and the e4m3 encoding of a 128-column block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "fp8_ops.h"

namespace g4m {

// Pairs of f32 in one register pair: one instruction for two fma or products.
// The f32 pipe takes two cycles for it, so the gain is in issue slots.
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ uint64_t pack_u32x2(uint32_t a, uint32_t b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
// acc += x * s, elementwise, each rounded to nearest.
__device__ __forceinline__ void fma_f32x2(uint64_t& acc, uint64_t x, uint64_t s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(s));
}
// a * b + c
__device__ __forceinline__ uint64_t fma3_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

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

// Eight consecutive elements as they lie in memory, for loads whose values
// are wanted later: converting at once would wait for the load at once.
template <class T>
struct Raw8 {
  static constexpr int WORDS = sizeof(T) / 2;
  uint4 w[WORDS];
};
// Elements [c, c + 8) of a row of d, zeros from d on (c a multiple of 8).
// vec: the row starts on a 16-byte boundary.  FULL: d is a multiple of 8, too,
// and a chunk is either inside the row or outside it.
template <bool FULL = false, class T>
__device__ __forceinline__ void load_raw8(const T* row, int c, int d, bool vec, Raw8<T>& r) {
  if (FULL) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::WORDS; ++i)
      r.w[i] = c < d ? reinterpret_cast<const uint4*>(row + c)[i] : make_uint4(0, 0, 0, 0);
  } else if (vec && c + 8 <= d) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::WORDS; ++i) r.w[i] = reinterpret_cast<const uint4*>(row + c)[i];
  } else {
    union {
      Raw8<T> raw;
      T e[8];
    } u = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) u.e[i] = row[c + i];
    r = u.raw;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(r.w[i].x);
    v[4 * i + 1] = __uint_as_float(r.w[i].y);
    v[4 * i + 2] = __uint_as_float(r.w[i].z);
    v[4 * i + 3] = __uint_as_float(r.w[i].w);
  }
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  unpack2(r.w[0].x, T(), v[0], v[1]);
  unpack2(r.w[0].y, T(), v[2], v[3]);
  unpack2(r.w[0].z, T(), v[4], v[5]);
  unpack2(r.w[0].w, T(), v[6], v[7]);
}

// Elements [c, c + 8) of a row of d as floats, zeros from d on.
template <bool FULL = false, class T>
__device__ __forceinline__ void load8(const T* row, int c, int d, bool vec, float (&v)[8]) {
  Raw8<T> r;
  load_raw8<FULL>(row, c, d, vec, r);
  unpack8(r, v);
}
// Elements [c, c + 8) of a row of d, each rounded once; nothing from d on.
template <bool FULL = false>
__device__ __forceinline__ void store8(float* row, int c, int d, bool vec, const float (&v)[8]) {
  if (FULL ? c < d : vec && c + 8 <= d) {
    *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else if (!FULL) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) row[c + i] = v[i];
  }
}
template <bool FULL = false, class T>
__device__ __forceinline__ void store8(T* row, int c, int d, bool vec, const float (&v)[8]) {
  if (FULL ? c < d : vec && c + 8 <= d) {
    *reinterpret_cast<uint4*>(row + c) =
        make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
  } else if (!FULL) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) from_f32(v[i], row + c + i);
  }
}

// Quotient by a divisor fixed for the launch: n / d = (n * m) >> (32 + s) for
// every n < 2^31 (Granlund and Montgomery, PLDI 1994), m and s from the host.
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;  // 2^s >= d
  if (s == 0) return {d, 0, 0};
  --s;                          // d > 1: m in (2^31, 2^32)
  return {d, (uint32_t)(((1ull << (32 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return f.m ? __umulhi(n, f.m) >> f.s : n;
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

// Correctly rounded n / d from a reciprocal r of d that is within a unit of
// 1 / d: the product, corrected by its fma residual (Markstein, IBM J. Res.
// Develop. 34(1), 1990).  Three operations, no branch.
__device__ __forceinline__ float div_by_rcp(float n, float d, float r) {
  const float q = n * r;
  return fmaf(fmaf(-q, d, n), r, q);
}

// scale = max(amax, 2^-96) / 448; the floor keeps the scale of an all-zero
// block (and its reciprocal) a normal number.  NaN for a block that is not
// finite.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
  const float s = div_by_rcp(fmaxf(__uint_as_float(amax_bits), 0x1p-96f), 448.0f, 1.0f / 448.0f);
  return amax_bits < 0x7f800000u ? s : __uint_as_float(0x7fffffffu);
}

// Eight codes e4m3(v / s), to nearest even, of the rounded quotient: the
// codes are those of a true division.
__device__ __forceinline__ uint2 fp8_encode8(const float (&v)[8], float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = fmaf(fmaf(-s, inv, 1.0f), inv, inv);  // one Newton step
  const uint64_t inv2 = pack_f32x2(inv, inv), neg2 = pack_f32x2(-s, -s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // div_by_rcp of two
    const uint64_t x = pack_f32x2(v[2 * i], v[2 * i + 1]), q = mul_f32x2(x, inv2);
    float q0, q1;
    unpack_f32x2(fma3_f32x2(fma3_f32x2(q, neg2, x), inv2, q), q0, q1);
    uint16_t p;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(q1), "f"(q0));
    w[i] = p;
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Codes [c, c + 8) of a row of d codes that starts on a 16-byte boundary.
template <bool FULL = false>
__device__ __forceinline__ void store_codes8(uint8_t* row, int c, int d, uint2 w) {
  if (FULL ? c < d : c + 8 <= d) {
    *reinterpret_cast<uint2*>(row + c) = w;
  } else if (!FULL) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) row[c + i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

}  // namespace g4m
