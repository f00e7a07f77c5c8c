// Rotary positions on the heads of one or two projections.  HBM bound: every
// element is read and written once.
//
// The angle of (token, pair) is position * frequency modulo one turn.  The
// frequency is kept as a 64-bit fixed-point fraction of a turn, so the
// integer product wraps modulo one turn by itself and the phase is exact to
// position * 2^-65 turns at any position, without a 64-bit float operation.
// A block computes the cosines and sines of its tokens once into shared
// memory; a thread then keeps those of its pairs in registers and walks the
// heads, the next one's loads in flight.  A warp covers one token's
// neighbouring heads, so that it reads and writes contiguous memory.  For
// 16384 tokens x 40 heads x 128 bf16 (335 MB): 73 us with one head per thread
// and step but four tokens per warp, 71 us with the angles read from shared
// memory for every head, 58 us as it is.
#include <algorithm>

#include "fp8_rows.cuh"
#include "g4m_kernels.h"

namespace g4m {

constexpr int kRopeThreads = 256;
constexpr int kRopeTable = 4096;  // most (cos, sin) pairs a block holds: 32 KB, eight tokens of 512 pairs

struct RopeLaunch {
  RopeArgs a;
  int token_block;  // tokens of a block
  int items;        // threads of one (token, head): chunks or single pairs, then what passes through
  int lanes;        // heads of a token that threads of the block walk side by side
};

// The chunk of 8 pairs that a thread turns, as raw words.  Two halves: pairs
// [c, c + 8) at columns c and half + c.  Interleaved: columns [2 c, 2 c + 16).
template <class T, bool INTERLEAVED>
struct RopeChunk {
  Raw8<T> p, q;
  __device__ __forceinline__ void load(const T* x, int c, int half) {
    const int cp = INTERLEAVED ? 2 * c : c, cq = INTERLEAVED ? 2 * c + 8 : half + c;
    load_raw8(x, cp, cp + 8, true, p);
    load_raw8(x, cq, cq + 8, true, q);
  }
  __device__ __forceinline__ void turn(T* o, int c, int half, const float2 (&r)[8]) const {
    float a[8], b[8];
    unpack8(p, a);
    unpack8(q, b);
    if (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn1(a[2 * i], a[2 * i + 1], r[i]);
        turn1(b[2 * i], b[2 * i + 1], r[4 + i]);
      }
      store8(o, 2 * c, 2 * c + 8, true, a);
      store8(o, 2 * c + 8, 2 * c + 16, true, b);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn1(a[i], b[i], r[i]);
      store8(o, c, c + 8, true, a);
      store8(o, half + c, half + c + 8, true, b);
    }
  }
  static __device__ __forceinline__ void turn1(float& u, float& v, const float2& r) {
    const float a = u * r.x - v * r.y, b = v * r.x + u * r.y;
    u = a;
    v = b;
  }
};

// VEC: every head starts on a 16-byte boundary and the pairs come in whole
// chunks of 8; a thread then turns 8 pairs of a head.  Otherwise it turns one.
template <class T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeLaunch l) {
  extern __shared__ float4 cs4[];
  float2* cs = reinterpret_cast<float2*>(cs4);
  const RopeArgs& a = l.a;
  const long t0 = (long)blockIdx.x * l.token_block;
  const int nt = (int)min((long)l.token_block, a.tokens - t0);
  const int heads = a.v[0].heads + a.v[1].heads;
  const int turn_items = VEC ? a.half / 8 : a.half;
  // Work of a thread: (token, lane, item), heads h0, h0 + step, ...
  const int step = l.lanes * gridDim.y, total = nt * l.lanes * l.items;
  int w = threadIdx.x, t, c, h0;
  auto work_of = [&] {
    const int tl = w / l.items;
    c = w - tl * l.items;
    t = tl / l.lanes;
    h0 = tl - t * l.lanes + l.lanes * blockIdx.y;
  };
  auto head_of = [&](int h, const T*& x, T*& o) {
    const int k = h >= a.v[0].heads;
    const g4m_rope_view& v = a.v[k];
    const int head = h - (k ? a.v[0].heads : 0);
    x = static_cast<const T*>(v.x) + (t0 + t) * v.token_stride + head * v.head_stride;
    o = static_cast<T*>(v.out) + (t0 + t) * v.out_token_stride + head * v.out_head_stride;
    return k;
  };
  // What a thread has in flight: one head's chunk, or four heads' elements.
  constexpr int B = VEC ? 1 : 4;
  RopeChunk<T, INTERLEAVED> ka, kb;
  T e0[B], e1[B];
  const T* x;
  T* o;
  auto load_chunk = [&](int h, RopeChunk<T, INTERLEAVED>& k) {
    if (h < heads) {
      head_of(h, x, o);
      k.load(x, 8 * c, a.half);
    }
  };
  auto load_elements = [&](int h) {
    const bool turns = c < turn_items;
    const int iu = !turns ? a.half + c : INTERLEAVED ? 2 * c : c, iv = !turns ? iu : INTERLEAVED ? 2 * c + 1 : a.half + c;
#pragma unroll
    for (int i = 0; i < B; ++i)
      if (h + i * step < heads) {
        head_of(h + i * step, x, o);
        e0[i] = x[iu];
        e1[i] = x[iv];
      }
  };
  // The first loads go out before the angles are computed.
  if (w < total) {
    work_of();
    if (VEC && c < turn_items) load_chunk(h0, ka);
    if (!VEC) load_elements(h0);
  }
  for (int i = threadIdx.x; i < nt * a.half; i += kRopeThreads) {
    const int ti = i / a.half, j = i - ti * a.half;
    const long pos = a.pos64 ? static_cast<const long*>(a.positions)[t0 + ti] : static_cast<const int*>(a.positions)[t0 + ti];
    const uint64_t phase = (uint64_t)pos * a.turns[j];
    float sn, cn;
    sincospif(__ll2float_rn((long long)phase) * 0x1p-63f, &sn, &cn);  // half turns in [-1, 1]
    cs[i] = make_float2(cn * a.scale, sn * a.scale);
  }
  __syncthreads();
  for (bool first = true; w < total; w += kRopeThreads, first = false) {
    if (!first) {
      work_of();
      if (VEC && c < turn_items) load_chunk(h0, ka);
      if (!VEC) load_elements(h0);
    }
    if (VEC && c < turn_items) {
      float2 r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = cs[t * a.half + 8 * c + i];
      for (int h = h0; h < heads; h += 2 * step) {
        load_chunk(h + step, kb);
        head_of(h, x, o);
        ka.turn(o, 8 * c, a.half, r);
        if (h + step >= heads) break;
        load_chunk(h + 2 * step, ka);
        head_of(h + step, x, o);
        kb.turn(o, 8 * c, a.half, r);
      }
    } else if (VEC) {  // columns that pass through
      const int e = 2 * a.half + 8 * (c - turn_items);
      for (int h = h0; h < heads; h += step) {
        if (!a.copy[head_of(h, x, o)]) continue;
        if (e + 8 <= a.head_dim) {
          Raw8<T> r;
          load_raw8(x, e, e + 8, true, r);
#pragma unroll
          for (int i = 0; i < Raw8<T>::WORDS; ++i) reinterpret_cast<uint4*>(o + e)[i] = r.w[i];
        } else {
          for (int i = e; i < a.head_dim; ++i) o[i] = x[i];
        }
      }
    } else {
      const bool turns = c < turn_items;
      const float2 r = turns ? cs[t * a.half + c] : make_float2(0.0f, 0.0f);
      const int iu = !turns ? a.half + c : INTERLEAVED ? 2 * c : c, iv = INTERLEAVED ? 2 * c + 1 : a.half + c;
      for (int h = h0;;) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (h + i * step < heads) {
            const int k = head_of(h + i * step, x, o);
            if (turns) {
              const float u = to_f32(e0[i]), v = to_f32(e1[i]);
              from_f32(u * r.x - v * r.y, o + iu);
              from_f32(v * r.x + u * r.y, o + iv);
            } else if (a.copy[k]) {
              o[iu] = e0[i];
            }
          }
        h += B * step;
        if (h >= heads) break;
        load_elements(h);
      }
    }
  }
}

template <class T>
static void launch_rope(const RopeLaunch& l, dim3 grid, cudaStream_t st) {
  const size_t table = sizeof(float2) * l.token_block * l.a.half;
  if (l.a.vec) {
    if (l.a.interleaved) rope_kernel<T, true, true><<<grid, kRopeThreads, table, st>>>(l);
    else rope_kernel<T, true, false><<<grid, kRopeThreads, table, st>>>(l);
  } else {
    if (l.a.interleaved) rope_kernel<T, false, true><<<grid, kRopeThreads, table, st>>>(l);
    else rope_kernel<T, false, false><<<grid, kRopeThreads, table, st>>>(l);
  }
}

cudaError_t rope_run(const RopeArgs& a, int dev, cudaStream_t st) {
  RopeLaunch l;
  l.a = a;
  const int heads = a.v[0].heads + a.v[1].heads, sms = g_num_sms(dev);
  const int pass = a.copy[0] | a.copy[1] ? a.head_dim - 2 * a.half : 0;
  l.items = a.vec ? a.half / 8 + (pass + 7) / 8 : a.half + pass;
  // Lanes enough that a warp covers one token's neighbouring heads, then as
  // many tokens as fill the block; short inputs take fewer tokens per block
  // and spread their heads over more lanes, then over more blocks.
  const long want = (long)sms * 4;  // blocks
  const long lanes = std::max<long>(1, std::min<long>(heads, 32 / l.items));
  long tb = std::max<long>(1, std::min<long>(a.tokens / want, kRopeThreads / (lanes * l.items)));
  tb = std::min<long>(tb, kRopeTable / a.half);
  l.token_block = (int)tb;
  const long groups = (a.tokens + tb - 1) / tb;
  const bool few = tb * lanes * l.items < kRopeThreads;
  l.lanes = (int)(few ? std::max<long>(1, std::min<long>(heads, kRopeThreads / (tb * l.items))) : lanes);
  const long slices = std::max<long>(1, std::min<long>((heads + l.lanes - 1) / l.lanes, want / groups));
  const dim3 grid((unsigned)groups, (unsigned)slices);
  if (a.dtype == G4M_F32) launch_rope<float>(l, grid, st);
  else if (a.dtype == G4M_BF16) launch_rope<__nv_bfloat16>(l, grid, st);
  else launch_rope<__half>(l, grid, st);
  return cudaGetLastError();
}

}  // namespace g4m
