// Rotary positions on the heads of one or two projections.  HBM bound: every
// element is read and written once.
//
// The angle of (token, pair) is position * frequency modulo one turn.  The
// frequency is kept as a 64-bit fixed-point fraction of a turn, so the
// integer product wraps modulo one turn by itself and the phase is off by at
// most |position| * 2^-65 turns, without a 64-bit float operation.
// A block computes the cosines and sines of its tokens once into shared
// memory; a thread then keeps those of its pairs in registers and walks the
// heads, the next one's loads in flight.  A warp covers one token's
// neighbouring heads, so that it reads and writes contiguous memory.  For
// 16384 tokens x 40 heads x 128 bf16 (335 MB): 73 us with one head per thread
// and step but four tokens per warp, 71 us with the angles read from shared
// memory for every head, 60 us as it is.
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
  Raw8<T, true> p, q;
  __device__ __forceinline__ void load(const T* x, int c, int half) {
    const int cp = INTERLEAVED ? 2 * c : c, cq = INTERLEAVED ? 2 * c + 8 : half + c;
    load_raw8<T, true>(x, cp, cp + 8, p);
    load_raw8<T, true>(x, cq, cq + 8, q);
  }
  __device__ __forceinline__ void turn(T* o, int c, int half, const float2 (&r)[8]) const {
    float a[8], b[8];
    unpack8<T, true>(p, a);
    unpack8<T, true>(q, b);
    if (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn1(a[2 * i], a[2 * i + 1], r[i]);
        turn1(b[2 * i], b[2 * i + 1], r[4 + i]);
      }
      store8<true>(o, 2 * c, 2 * c + 8, a);
      store8<true>(o, 2 * c + 8, 2 * c + 16, b);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn1(a[i], b[i], r[i]);
      store8<true>(o, c, c + 8, a);
      store8<true>(o, half + c, half + c + 8, b);
    }
  }
  static __device__ __forceinline__ void turn1(float& u, float& v, const float2& r) {
    const float a = u * r.x - v * r.y, b = v * r.x + u * r.y;
    u = a;
    v = b;
  }
};

// Cosines and sines of the block's tokens.
__device__ __forceinline__ void rope_table(const RopeArgs& a, float2* cs, long t0, int nt) {
  for (int i = threadIdx.x; i < nt * a.half; i += blockDim.x) {
    const int t = i / a.half, j = i - t * a.half;
    const long pos = a.pos64 ? static_cast<const long*>(a.positions)[t0 + t] : static_cast<const int*>(a.positions)[t0 + t];
    const uint64_t phase = (uint64_t)pos * a.turns[j];
    // The nearest quarter turn comes off in integers, so that the rounding to
    // f32 is relative to what is left, at most an eighth of a turn.
    const uint64_t quarter = (phase + (1ull << 61)) >> 62;
    const long long rest = (long long)(phase - (quarter << 62));
    float sn, cn;
    sincospif(__ll2float_rn(rest) * 0x1p-63f, &sn, &cn);  // half turns in [-1/4, 1/4]
    const float c = quarter & 1 ? sn : cn, s = quarter & 1 ? cn : sn;
    cs[i] = make_float2((quarter + 1) & 2 ? -c * a.scale : c * a.scale, quarter & 2 ? -s * a.scale : s * a.scale);
  }
}

// Every head starts on a 16-byte boundary and the pairs come in whole chunks
// of 8: a thread turns 8 pairs of a head.
template <class T, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeLaunch l) {
  extern __shared__ float4 cs4[];
  float2* cs = reinterpret_cast<float2*>(cs4);
  const RopeArgs& a = l.a;
  const long t0 = (long)blockIdx.x * l.token_block;
  const int nt = (int)min((long)l.token_block, a.tokens - t0);
  const int heads = a.v[0].heads + a.v[1].heads;
  const int turn_items = a.half / 8;
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
  RopeChunk<T, INTERLEAVED> ka, kb;
  const T* x;
  T* o;
  auto load = [&](int h, RopeChunk<T, INTERLEAVED>& k) {
    if (h < heads) {
      head_of(h, x, o);
      k.load(x, 8 * c, a.half);
    }
  };
  // The first loads go out before the angles are computed.
  if (w < total) {
    work_of();
    if (c < turn_items) load(h0, ka);
  }
  rope_table(a, cs, t0, nt);
  __syncthreads();
  for (bool first = true; w < total; w += kRopeThreads, first = false) {
    if (!first) {
      work_of();
      if (c < turn_items) load(h0, ka);
    }
    if (c < turn_items) {
      float2 r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = cs[t * a.half + 8 * c + i];
      for (int h = h0; h < heads; h += 2 * step) {
        load(h + step, kb);
        head_of(h, x, o);
        ka.turn(o, 8 * c, a.half, r);
        if (h + step >= heads) break;
        load(h + 2 * step, ka);
        head_of(h + step, x, o);
        kb.turn(o, 8 * c, a.half, r);
      }
    } else {  // columns that pass through
      const int e = 2 * a.half + 8 * (c - turn_items);
      for (int h = h0; h < heads; h += step) {
        if (!a.copy[head_of(h, x, o)]) continue;
        if (e + 8 <= a.head_dim) {
          Raw8<T, true> r;
          load_raw8<T, true>(x, e, e + 8, r);
#pragma unroll
          for (int i = 0; i < Raw8<T, true>::WORDS; ++i) reinterpret_cast<uint4*>(o + e)[i] = r.w[i];
        } else {
          for (int i = e; i < a.head_dim; ++i) o[i] = x[i];
        }
      }
    }
  }
}

// Any other head: a warp brings a few whole heads into shared memory in the
// widest words that all of them allow, turns their pairs there, and writes
// them back in such words, the next heads on their way.  (Pair by pair from
// global memory 3143 tokens x 24 heads x 172 f16, of which 34 turn, took 43 us
// where this takes 11; 15568 x 24 x 110 bf16 70 and 53.)
struct RopeStaged {
  RopeArgs a;
  int token_block, word, per;  // bytes of a word; heads of a batch
  int flat;                    // the heads of a batch lie side by side: one run of words
  int bytes[2], pitch, stage;  // of a head that move (all, or in place what turns); of a head, a batch in shared memory
  int batches[2];              // of a token, per view
  FastDiv by_half, by_batches, by_words[2];
};

template <int W>
__device__ __forceinline__ void copy_word_async(void* dst, const void* src) {
  if (W >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "n"(W >= 4 ? W : 4)
                 : "memory");
  } else {
    *static_cast<uint16_t*>(dst) = *static_cast<const uint16_t*>(src);
  }
}
template <int W>
__device__ __forceinline__ void copy_word(void* dst, const void* src) {
  if (W == 16) *static_cast<uint4*>(dst) = *static_cast<const uint4*>(src);
  else if (W == 8) *static_cast<uint2*>(dst) = *static_cast<const uint2*>(src);
  else if (W == 4) *static_cast<uint32_t*>(dst) = *static_cast<const uint32_t*>(src);
  else *static_cast<uint16_t*>(dst) = *static_cast<const uint16_t*>(src);
}

template <class T, bool INTERLEAVED, int W>
__global__ void __launch_bounds__(kRopeThreads) rope_staged_kernel(const __grid_constant__ RopeStaged l) {
  extern __shared__ float4 cs4[];
  const RopeArgs& a = l.a;
  float2* cs = reinterpret_cast<float2*>(cs4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int table = (l.token_block * a.half + 1) / 2 * 16;  // bytes, in whole 16
  char* stage = reinterpret_cast<char*>(cs4) + table + warp * 2 * l.stage;
  const long t0 = (long)blockIdx.x * l.token_block;
  const int nt = (int)min((long)l.token_block, a.tokens - t0);
  const int batches = l.batches[0] + l.batches[1], units = nt * batches, step = warps * gridDim.y;
  struct Unit {
    int t, k, h0, n;
  };
  auto unit_of = [&](int u) {
    Unit r;
    r.t = (int)div_by((uint32_t)u, l.by_batches);
    const int b = u - r.t * batches;
    r.k = b >= l.batches[0];
    r.h0 = (b - (r.k ? l.batches[0] : 0)) * l.per;
    r.n = min(l.per, a.v[r.k].heads - r.h0);
    return r;
  };
  auto bring = [&](int u, char* to) {
    if (u < units) {
      const Unit r = unit_of(u);
      const g4m_rope_view& v = a.v[r.k];
      const char* x = reinterpret_cast<const char*>(static_cast<const T*>(v.x) + (t0 + r.t) * v.token_stride + r.h0 * v.head_stride);
      if (l.flat) {
        for (int i = lane * W; i < r.n * l.pitch; i += 32 * W) copy_word_async<W>(to + i, x + i);
      } else {
        const int words = l.bytes[r.k] / W;
        for (int i = lane; i < r.n * words; i += 32) {
          const int b = (int)div_by((uint32_t)i, l.by_words[r.k]), w = i - b * words;
          copy_word_async<W>(to + b * l.pitch + w * W, x + b * v.head_stride * (long)sizeof(T) + w * W);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int u = blockIdx.y * warps + warp;
  bring(u, stage);
  rope_table(a, cs, t0, nt);
  __syncthreads();
  for (int buf = 0; u < units; u += step, buf ^= 1) {
    char* s = stage + buf * l.stage;
    bring(u + step, stage + (buf ^ 1) * l.stage);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const Unit r = unit_of(u);
    for (int i = lane; i < r.n * a.half; i += 32) {
      const int b = (int)div_by((uint32_t)i, l.by_half), j = i - b * a.half;
      T* p = reinterpret_cast<T*>(s + b * l.pitch);
      T &pu = p[INTERLEAVED ? 2 * j : j], &pv = p[INTERLEAVED ? 2 * j + 1 : a.half + j];
      const float2 f = cs[r.t * a.half + j];
      const float x = to_f32(pu), y = to_f32(pv);
      from_f32(x * f.x - y * f.y, &pu);
      from_f32(y * f.x + x * f.y, &pv);
    }
    __syncwarp();
    const g4m_rope_view& v = a.v[r.k];
    char* o = reinterpret_cast<char*>(static_cast<T*>(v.out) + (t0 + r.t) * v.out_token_stride + r.h0 * v.out_head_stride);
    if (l.flat) {
      for (int i = lane * W; i < r.n * l.pitch; i += 32 * W) copy_word<W>(o + i, s + i);
    } else {
      const int words = l.bytes[r.k] / W;
      for (int i = lane; i < r.n * words; i += 32) {
        const int b = (int)div_by((uint32_t)i, l.by_words[r.k]), w = i - b * words;
        copy_word<W>(o + b * v.out_head_stride * (long)sizeof(T) + w * W, s + b * l.pitch + w * W);
      }
    }
    __syncwarp();  // the buffer is free for the next but one
  }
}

template <class T>
static void launch_chunks(const RopeArgs& a, int sms, cudaStream_t st) {
  RopeLaunch l;
  l.a = a;
  const int heads = a.v[0].heads + a.v[1].heads;
  const int pass = a.copy[0] | a.copy[1] ? a.head_dim - 2 * a.half : 0;
  l.items = a.half / 8 + (pass + 7) / 8;
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
  const size_t table = sizeof(float2) * l.token_block * a.half;
  if (a.interleaved) rope_kernel<T, true><<<grid, kRopeThreads, table, st>>>(l);
  else rope_kernel<T, false><<<grid, kRopeThreads, table, st>>>(l);
}

template <class T, int W>
static void launch_staged_w(const RopeStaged& l, dim3 grid, int threads, size_t smem, cudaStream_t st) {
  if (l.a.interleaved) rope_staged_kernel<T, true, W><<<grid, threads, smem, st>>>(l);
  else rope_staged_kernel<T, false, W><<<grid, threads, smem, st>>>(l);
}

template <class T>
static void launch_staged(const RopeArgs& a, int sms, cudaStream_t st) {
  RopeStaged l;
  l.a = a;
  const int size = sizeof(T);
  l.pitch = (a.head_dim * size + 15) / 16 * 16;
  l.per = std::max(1, std::min(4, 2048 / l.pitch));
  l.flat = 1;
  for (int k = 0; k < 2; ++k) {
    const g4m_rope_view& v = a.v[k];
    l.bytes[k] = (a.copy[k] ? a.head_dim : 2 * a.half) * size;
    if (v.heads > 0 && (l.bytes[k] != a.head_dim * size || v.head_stride != a.head_dim || v.out_head_stride != a.head_dim)) l.flat = 0;
  }
  if (l.flat) l.pitch = a.head_dim * size;
  l.stage = (l.per * l.pitch + 15) / 16 * 16;
  // The widest word that every address and length is a multiple of.
  uintptr_t all = 0;
  int batches = 0;
  for (int k = 0; k < 2; ++k) {
    const g4m_rope_view& v = a.v[k];
    l.batches[k] = (v.heads + l.per - 1) / l.per;
    batches += l.batches[k];
    if (v.heads == 0) continue;
    all |= (uintptr_t)v.x | (uintptr_t)v.out | (uintptr_t)(v.token_stride * size) | (uintptr_t)(v.out_token_stride * size);
    if (l.flat) all |= (uintptr_t)(v.heads >= l.per ? l.per * l.pitch : 0) | (uintptr_t)(v.heads % l.per * l.pitch);
    else all |= (uintptr_t)l.bytes[k] | (uintptr_t)(v.head_stride * size) | (uintptr_t)(v.out_head_stride * size);
  }
  l.word = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  for (int k = 0; k < 2; ++k) l.by_words[k] = fast_div((uint32_t)(l.bytes[k] / l.word));
  l.by_half = fast_div((uint32_t)a.half);
  l.by_batches = fast_div((uint32_t)batches);
  const int threads = l.pitch > 2048 ? 128 : 256, warps = threads / 32;  // at most 32 KB of stages
  const long want = (long)sms * 6;
  long tb = std::max<long>(1, std::min<long>(a.tokens / want, 8));
  tb = std::min<long>(tb, std::max<long>(1, 1024 / a.half));  // and 8 KB of table
  l.token_block = (int)tb;
  const long groups = (a.tokens + tb - 1) / tb;
  const long slices = std::max<long>(1, std::min<long>((tb * batches + warps - 1) / warps, want / groups));
  const dim3 grid((unsigned)groups, (unsigned)slices);
  const size_t smem = (size_t)(tb * a.half + 1) / 2 * 16 + (size_t)warps * 2 * l.stage;
  if (l.word == 16) launch_staged_w<T, 16>(l, grid, threads, smem, st);
  else if (l.word == 8) launch_staged_w<T, 8>(l, grid, threads, smem, st);
  else if (l.word == 4) launch_staged_w<T, 4>(l, grid, threads, smem, st);
  else if (size == 2) launch_staged_w<T, size == 2 ? 2 : 4>(l, grid, threads, smem, st);
}

template <class T>
static void launch_rope(const RopeArgs& a, int sms, cudaStream_t st) {
  if (a.vec) launch_chunks<T>(a, sms, st);
  else launch_staged<T>(a, sms, st);
}

cudaError_t rope_run(const RopeArgs& a, int dev, cudaStream_t st) {
  const int sms = g_num_sms(dev);
  if (a.dtype == G4M_F32) launch_rope<float>(a, sms, st);
  else if (a.dtype == G4M_BF16) launch_rope<__nv_bfloat16>(a, sms, st);
  else launch_rope<__half>(a, sms, st);
  return cudaGetLastError();
}

}  // namespace g4m
