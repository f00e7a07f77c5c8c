// Device helpers of the 8-bit float row operators: typed loads and stores of
// eight consecutive elements, and the e4m3 encoding of a 128-column block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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
// FULL: rows start on 16-byte boundaries and hold whole chunks of eight.
// Otherwise a row may start m bytes past a boundary: the chunk then comes as
// the aligned 16-byte words around it and is shifted into place when it is
// unpacked.  (Element by element, 2947 x 5193 bf16 through the residual norm
// took 146 us, now 76.)
template <class T, bool FULL>
struct Raw8 {
  static constexpr int WORDS = sizeof(T) / 2;  // 16-byte words of a chunk
  uint4 w[WORDS + (FULL ? 0 : 1)];
  uint32_t m;
};
// Elements [c, c + 8) of a row of d, zeros from d on (c a multiple of 8).
// Nothing outside the row is read: the row's first and last whole chunks and
// its rest come element by element where the row is not aligned.
template <class T, bool FULL>
__device__ __forceinline__ void load_raw8(const T* row, int c, int d, Raw8<T, FULL>& r) {
  constexpr int W = Raw8<T, FULL>::WORDS;
  if (FULL) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = c < d ? reinterpret_cast<const uint4*>(row + c)[i] : make_uint4(0, 0, 0, 0);
    return;
  }
  const uint32_t m = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);
  if (c + 8 <= d && (m == 0 || (c >= 8 && c + 16 <= d))) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row + c) - m);
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = p[i];
    r.w[FULL ? 0 : W] = m ? p[W] : make_uint4(0, 0, 0, 0);
    r.m = m;
  } else {
    union {
      uint4 w[W];
      T e[8];
    } u = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) u.e[i] = row[c + i];
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = u.w[i];
    r.m = 0;
  }
}

// out[i] = 32-bit word at byte 4 i + m of in, m < 16.
template <int N>
__device__ __forceinline__ void shift_words(const uint32_t (&in)[N + 4], uint32_t m, uint32_t (&out)[N]) {
  const uint32_t bits = 8 * (m & 3);
  auto by = [&](auto first) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(in[i + first.value], in[i + first.value + 1], bits);
  };
  if ((m >> 2) == 0) by(std::integral_constant<int, 0>());
  else if ((m >> 2) == 1) by(std::integral_constant<int, 1>());
  else if ((m >> 2) == 2) by(std::integral_constant<int, 2>());
  else by(std::integral_constant<int, 3>());
}

__device__ __forceinline__ void words_to_f32(const uint32_t (&w)[8], float (&v)[8], float) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
template <class T>
__device__ __forceinline__ void words_to_f32(const uint32_t (&w)[4], float (&v)[8], T) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(w[i], T(), v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void f32_to_words(const float (&v)[8], uint32_t (&w)[8], float) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
}
template <class T>
__device__ __forceinline__ void f32_to_words(const float (&v)[8], uint32_t (&w)[4], T) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], T());
}

template <class T, bool FULL>
__device__ __forceinline__ void unpack8(const Raw8<T, FULL>& r, float (&v)[8]) {
  constexpr int N = 4 * Raw8<T, FULL>::WORDS;
  uint32_t w[N];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) w[4 * i] = r.w[i].x, w[4 * i + 1] = r.w[i].y, w[4 * i + 2] = r.w[i].z, w[4 * i + 3] = r.w[i].w;
  if (!FULL && r.m != 0) {
    uint32_t in[N + 4];
#pragma unroll
    for (int i = 0; i < N; ++i) in[i] = w[i];
    const uint4 last = r.w[FULL ? 0 : N / 4];
    in[N] = last.x, in[N + 1] = last.y, in[N + 2] = last.z, in[N + 3] = last.w;
    shift_words<N>(in, r.m, w);
  }
  words_to_f32(w, v, T());
}

// Elements [c, c + 8) of a row of d as floats, zeros from d on.
template <bool FULL, class T>
__device__ __forceinline__ void load8(const T* row, int c, int d, float (&v)[8]) {
  Raw8<T, FULL> r;
  load_raw8<T, FULL>(row, c, d, r);
  unpack8<T, FULL>(r, v);
}

// Those of the eight elements in w whose bit of mask is set.
__device__ __forceinline__ void store_elements(float* p, const uint32_t (&w)[8], uint32_t mask) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (mask & (1u << i)) p[i] = __uint_as_float(w[i]);
}
template <class T>
__device__ __forceinline__ void store_elements(T* p, const uint32_t (&w)[4], uint32_t mask) {
  uint16_t* u = reinterpret_cast<uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (mask & (1u << i)) u[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
}

// Elements [c, c + 8) of a row of d, each rounded once; nothing from d on.
// Without FULL the whole warp calls, its lanes at neighbouring chunks: where
// the row starts m bytes past a 16-byte boundary, a lane writes the aligned
// words that begin in its chunk, the last of them with the head of the next
// lane's, and only the warp's and the row's edges go element by element.
template <bool FULL, class T>
__device__ __forceinline__ void store8(T* row, int c, int d, const float (&v)[8]) {
  constexpr int N = 4 * Raw8<T, FULL>::WORDS;
  uint32_t w[N];
  f32_to_words(v, w, T());
  const uint32_t m = FULL ? 0 : (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);
  if (m == 0) {
    if (c + 8 <= d) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        reinterpret_cast<uint4*>(row + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if (!FULL && c < d) {
      store_elements(row + c, w, (1u << (d - c)) - 1);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  uint32_t in[N + 4], out[N];
#pragma unroll
  for (int i = 0; i < N; ++i) in[i] = w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) in[N + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
  shift_words<N>(in, 16 - m, out);
  const bool own = c + 8 <= d, next = lane < 31 && c + 16 <= d;  // whole chunks here, and in the next lane
  uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<char*>(row + c) + 16 - m);
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    if (own && (i < N / 4 - 1 || next)) p[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
  // What no aligned word of a lane covers: this chunk's head, unless the lane
  // before wrote it, and its tail, unless this lane did with the next's head.
  const int head = (16 - m) / sizeof(T), tail = 8 - m / sizeof(T);
  if (own) {
    const uint32_t mask = (lane == 0 ? (1u << head) - 1 : 0u) | (next ? 0u : 0x100u - (1u << tail));
    if (mask) store_elements(row + c, w, mask);
  } else if (c < d) {
    store_elements(row + c, w, (1u << (d - c)) - 1);
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

// Largest magnitude of v; a NaN among them makes it NaN.
__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 7; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[7])));
  return m;
}
// Over the 16 lanes that hold one block of 128 columns (all 32 lanes call).
__device__ __forceinline__ float block_amax(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__shfl_xor_sync(0xffffffffu, m, o)));
  return m;
}

// Correctly rounded n / d from r, the correctly rounded reciprocal of d: the
// product, corrected by its fma residual (Markstein, IBM J. Res. Develop.
// 34(1), 1990).  Three operations, no branch.  (A reciprocal that is merely
// within a unit of 1 / d is not enough.)
__device__ __forceinline__ float div_by_rcp(float n, float d, float r) {
  const float q = n * r;
  return fmaf(fmaf(-q, d, n), r, q);
}

// scale = max(amax, 2^-96) / 448; the floor keeps the scale of an all-zero
// block (and its reciprocal) a normal number.  NaN for a block that is not
// finite.
__device__ __forceinline__ float fp8_scale(float amax) {
  const float s = div_by_rcp(fmaxf(amax, 0x1p-96f), 448.0f, 1.0f / 448.0f);
  return amax < __int_as_float(0x7f800000) ? s : __uint_as_float(0x7fffffffu);
}

// Eight codes e4m3(v / s), to nearest even, of the rounded quotient, where
// no residual falls among the subnormals.  The Newton step on this GPU's
// approximate reciprocal, never more than a unit off, gives the correctly
// rounded one for each of the 1.9e9 f32 from 2^-106 to 2^120 (tried one by
// one; as mathematics alone some estimates a unit off would stay there), and
// scales lie between 2^-105 and 2^120.
__device__ __forceinline__ uint2 fp8_encode8_normal(const float (&v)[8], float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = fmaf(fmaf(-s, inv, 1.0f), inv, inv);  // one Newton step
  const uint64_t s2 = pack_f32x2(s, s), neg2 = pack_f32x2(-inv, -inv);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // div_by_rcp of two, with the sign turned until the code: so a zero keeps
    // its own (a residual of +0 added to a quotient of -0 would make it +0).
    const uint64_t x = pack_f32x2(v[2 * i], v[2 * i + 1]), q = mul_f32x2(x, neg2);
    float q0, q1;
    unpack_f32x2(fma3_f32x2(fma3_f32x2(q, s2, x), neg2, q), q0, q1);
    uint16_t p;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(q1), "f"(q0));
    w[i] = p;
  }
  return make_uint2((w[0] | (w[1] << 16)) ^ 0x80808080u, (w[2] | (w[3] << 16)) ^ 0x80808080u);
}
// The same for any block: the codes are those of a true division.  In blocks
// with maxima below 2^-71 both sides of the division go up by 2^64 first.
// Two copies of the code, so that other blocks pay for the test alone (8192 x
// 6144 with gelu: 49.3 us, 50.4 with one copy that both ways join, 48.4
// without the test; with a division there rows of zeros took 127 us, now 53).
__device__ __forceinline__ uint2 fp8_encode8(const float (&v)[8], float s) {
  if (s < 0x1p-80f) {
    float up[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) up[i] = v[i] * 0x1p64f;
    return fp8_encode8_normal(up, s * 0x1p64f);
  }
  return fp8_encode8_normal(v, s);
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
