// Rotary positions on the heads of one or two projections.  HBM bound: every
// element is read and written once.
//
// The angle of (token, pair) is position * frequency modulo one turn.  The
// frequency is kept as a 64-bit fixed-point fraction of a turn, so the
// integer product wraps modulo one turn by itself and the phase is exact to
// position * 2^-65 turns at any position, without a 64-bit float operation.
// A block computes the cosines and sines of its tokens once into shared
// memory and turns all (or a slice) of the heads with them.
#include <algorithm>

#include "fp8_rows.cuh"

namespace g4m {

constexpr int kRopeThreads = 256;
constexpr int kRopeTable = 4096;  // (cos, sin) pairs a block holds: 32 KB, eight tokens of 512 pairs

template <class T, bool INTERLEAVED>
__device__ __forceinline__ void rope_chunk(const T* x, T* o, const float2* cs, int c, int half) {
  float u[8], v[8];
  if (INTERLEAVED) {  // columns [2 c, 2 c + 16): pairs [c, c + 8)
    float p[8], q[8];
    load8(x, 2 * c, 2 * c + 8, true, p);
    load8(x, 2 * c + 8, 2 * c + 16, true, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = p[2 * i], v[i] = p[2 * i + 1], u[4 + i] = q[2 * i], v[4 + i] = q[2 * i + 1];
  } else {
    load8(x, c, c + 8, true, u);
    load8(x, half + c, half + c + 8, true, v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 r = cs[c + i];
    const float a = u[i] * r.x - v[i] * r.y, b = v[i] * r.x + u[i] * r.y;
    u[i] = a;
    v[i] = b;
  }
  if (INTERLEAVED) {
    float p[8], q[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[2 * i] = u[i], p[2 * i + 1] = v[i], q[2 * i] = u[4 + i], q[2 * i + 1] = v[4 + i];
    store8(o, 2 * c, 2 * c + 8, true, p);
    store8(o, 2 * c + 8, 2 * c + 16, true, q);
  } else {
    store8(o, c, c + 8, true, u);
    store8(o, half + c, half + c + 8, true, v);
  }
}

// VEC: every head starts on a 16-byte boundary and the pairs come in whole
// chunks of 8; a thread then turns 8 pairs.  Otherwise it turns one.
template <class T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[kRopeTable];
  const long t0 = (long)blockIdx.x * a.token_block;
  const int nt = (int)min((long)a.token_block, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * a.half; i += kRopeThreads) {
    const int t = i / a.half, j = i - t * a.half;
    const long pos = a.pos64 ? static_cast<const long*>(a.positions)[t0 + t] : static_cast<const int*>(a.positions)[t0 + t];
    const uint64_t phase = (uint64_t)pos * a.turns[j];
    float s, c;
    sincospif(__ll2float_rn((long long)phase) * 0x1p-63f, &s, &c);  // half turns in [-1, 1]
    cs[i] = make_float2(c * a.scale, s * a.scale);
  }
  __syncthreads();
  const int heads = a.v[0].heads + a.v[1].heads;
  const int h0 = (int)((long)heads * blockIdx.y / gridDim.y), nh = (int)((long)heads * (blockIdx.y + 1) / gridDim.y) - h0;
  const int pass = a.head_dim - 2 * a.half;  // elements that pass through
  const int turn_items = VEC ? a.half / 8 : a.half;
  const int pass_items = (a.copy[0] | a.copy[1]) ? (VEC ? (pass + 7) / 8 : pass) : 0;
  const int items = turn_items + pass_items;
  const int total = nt * nh * items;
  for (int i = threadIdx.x; i < total; i += kRopeThreads) {
    const int th = i / items, c = i - th * items;
    const int t = th / nh, hh = h0 + th - t * nh;
    const int w = hh >= a.v[0].heads;
    const g4m_rope_view& v = a.v[w];
    const int head = hh - (w ? a.v[0].heads : 0);
    const T* x = static_cast<const T*>(v.x) + (t0 + t) * v.token_stride + head * v.head_stride;
    T* o = static_cast<T*>(v.out) + (t0 + t) * v.out_token_stride + head * v.out_head_stride;
    if (c < turn_items) {
      const float2* r = cs + t * a.half;
      if (VEC) {
        rope_chunk<T, INTERLEAVED>(x, o, r, 8 * c, a.half);
      } else {
        const int iu = INTERLEAVED ? 2 * c : c, iv = INTERLEAVED ? 2 * c + 1 : a.half + c;
        const float u = to_f32(x[iu]), z = to_f32(x[iv]);
        from_f32(u * r[c].x - z * r[c].y, o + iu);
        from_f32(z * r[c].x + u * r[c].y, o + iv);
      }
    } else if (a.copy[w]) {
      const int e = 2 * a.half + (VEC ? 8 : 1) * (c - turn_items);
      if (VEC && e + 8 <= a.head_dim) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k)
          reinterpret_cast<uint4*>(o + e)[k] = reinterpret_cast<const uint4*>(x + e)[k];
      } else {
        for (int k = e; k < min(e + (VEC ? 8 : 1), a.head_dim); ++k) o[k] = x[k];
      }
    }
  }
}

template <class T>
static void launch_rope(const RopeArgs& a, dim3 grid, cudaStream_t st) {
  if (a.vec) {
    if (a.interleaved) rope_kernel<T, true, true><<<grid, kRopeThreads, 0, st>>>(a);
    else rope_kernel<T, true, false><<<grid, kRopeThreads, 0, st>>>(a);
  } else {
    if (a.interleaved) rope_kernel<T, false, true><<<grid, kRopeThreads, 0, st>>>(a);
    else rope_kernel<T, false, false><<<grid, kRopeThreads, 0, st>>>(a);
  }
}

cudaError_t rope_run(RopeArgs a, cudaStream_t st) {
  const int heads = a.v[0].heads + a.v[1].heads;
  // About eight waves' worth of tokens per block at most, so that short
  // inputs still spread over the SMs; the table bounds it from above.
  long tb = std::max<long>(1, std::min<long>(8, a.tokens / (148 * 4)));
  tb = std::min<long>(tb, kRopeTable / a.half);
  a.token_block = (int)tb;
  const long groups = (a.tokens + tb - 1) / tb;
  a.head_slices = (int)std::min<long>(heads, std::max<long>(1, 148 * 2 / groups));
  const dim3 grid((unsigned)groups, (unsigned)a.head_slices);
  if (a.dtype == G4M_F32) launch_rope<float>(a, grid, st);
  else if (a.dtype == G4M_BF16) launch_rope<__nv_bfloat16>(a, grid, st);
  else launch_rope<__half>(a, grid, st);
  return cudaGetLastError();
}

}  // namespace g4m
