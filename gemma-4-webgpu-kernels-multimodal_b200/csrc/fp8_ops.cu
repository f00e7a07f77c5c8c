// C ABI of the 8-bit float operators: argument checks, resident handles and
// launches.  Calls allocate nothing, share no workspace and leave the calling
// thread's current device as it was, so calls on different streams may
// overlap and every call can be captured into a graph.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <string>
#include <vector>

#include "fp8_ops.h"
#include "g4m_kernels.h"
#include "runtime_internal.h"

using namespace g4m;

struct g4m_fp8_linear {
  Device* d = nullptr;
  int dev = 0, in = 0, out = 0;
  uint8_t* w = nullptr;
  float* sw = nullptr;
  float* bias = nullptr;
};

struct g4m_rope {
  Device* d = nullptr;
  int dev = 0, head_dim = 0, half = 0, interleaved = 0;
  float scale = 1.0f;
  uint64_t* turns = nullptr;
};

namespace {

// The calling thread's current device is changed for the length of a call only.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int id) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev == id) prev = -1;
    else cudaSetDevice(id);
    (void)cudaGetLastError();
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// No C++ exception (an allocation that fails) leaves a C entry.
template <class F>
int no_throw(F f) {
  try {
    return f();
  } catch (...) {
    try {
      return fail(G4M_E_CUDA, "host allocation failed");
    } catch (...) {
      return G4M_E_CUDA;
    }
  }
}

bool dtype_ok(int t) { return t == G4M_F32 || t == G4M_BF16 || t == G4M_F16; }
int64_t dtype_size(int t) { return t == G4M_F32 ? 4 : 2; }
bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)to == 0; }
bool rows16(const void* p, int64_t ld, int64_t size) { return aligned(p, 16) && (ld * size) % 16 == 0; }
cudaStream_t stream_of(void* s) { return s ? (cudaStream_t)s : cudaStreamLegacy; }
bool device_ok(const g4m_ctx* ctx, int di) { return ctx && di >= 0 && di < (int)ctx->devs.size(); }

// A row set: pointer aligned to its elements, stride no less than its width.
int check_rows(const char* what, const void* p, int64_t ld, int64_t width, int dtype) {
  if (!aligned(p, dtype_size(dtype))) return fail(G4M_E_ARG, std::string(what) + ": pointer is not aligned to its elements");
  if (ld < width) return fail(G4M_E_SHAPE, std::string(what) + ": row stride " + std::to_string(ld) + " is less than " + std::to_string(width));
  return G4M_OK;
}

int check_fp8(const char* what, const g4m_fp8_rows& x, int64_t rows, int64_t width) {
  if (!x.codes || !x.scales) return fail(G4M_E_ARG, std::string(what) + ": null codes or scales");
  if (!aligned(x.codes, 16) || x.ldc % 16 != 0)
    return fail(G4M_E_ARG, std::string(what) + ": codes need a 16-byte aligned pointer and row stride");
  if (!aligned(x.scales, 4)) return fail(G4M_E_ARG, std::string(what) + ": scales are not aligned");
  if (x.ldc < width) return fail(G4M_E_SHAPE, std::string(what) + ": codes row stride " + std::to_string(x.ldc) + " is less than " + std::to_string(width));
  if (x.lds < rows) return fail(G4M_E_SHAPE, std::string(what) + ": scales stride " + std::to_string(x.lds) + " is less than " + std::to_string(rows) + " rows");
  return G4M_OK;
}

int check_norm(const g4m_norm_args& a) {
  if (!a.y && !a.h) return fail(G4M_E_ARG, "neither y nor h is given");
  if (!a.y && a.gate) return fail(G4M_E_ARG, "a gate needs y");
  if (!a.h_out && !a.n_out && !a.out.codes) return fail(G4M_E_ARG, "no output is given");
  if (a.gate && a.rows_per_gate <= 0) return fail(G4M_E_ARG, "rows_per_gate must be positive");
  if (!aligned(a.w_post, 4) || !aligned(a.w_pre, 4)) return fail(G4M_E_ARG, "a norm weight is not aligned");
  if ((a.h && a.h_out == a.h && a.ldh_out != a.ldh) || (a.y && a.n_out == a.y && a.ldn != a.ldy))
    return fail(G4M_E_ARG, "an output in place of its input needs the input's row stride");
  if (a.h_out && a.h_out == a.n_out) return fail(G4M_E_ARG, "h_out and n_out are the same buffer");
  int rc = G4M_OK;
  if (a.y) rc = check_rows("y", a.y, a.ldy, a.d, a.dtype);
  if (!rc && a.h) rc = check_rows("h", a.h, a.ldh, a.d, a.h_dtype);
  if (!rc && a.gate) rc = check_rows("gate", a.gate, a.ldg, a.d, a.dtype);
  if (!rc && a.h_out) rc = check_rows("h_out", a.h_out, a.ldh_out, a.d, a.h_dtype);
  if (!rc && a.n_out) rc = check_rows("n_out", a.n_out, a.ldn, a.d, a.dtype);
  if (!rc && a.out.codes) rc = check_fp8("out", a.out, a.rows, a.d);
  return rc;
}

// Device copy of n elements.  A copy from pageable memory may still be on its
// way when cudaMemcpy returns, and no non-blocking stream waits for the legacy
// stream that it runs on: it has landed before this returns.
template <class T>
bool to_device(T** dst, const T* src, size_t n) {
  return cudaMalloc(dst, n * sizeof(T)) == cudaSuccess &&
         cudaMemcpy(*dst, src, n * sizeof(T), cudaMemcpyHostToDevice) == cudaSuccess &&
         cudaStreamSynchronize(cudaStreamLegacy) == cudaSuccess;
}

}  // namespace

extern "C" {

int g4m_synchronize(g4m_ctx* ctx, int di, void* stream) {
  return no_throw([&]() -> int {
    if (!device_ok(ctx, di)) return fail(G4M_E_ARG, "bad context or device index");
    Device& d = *ctx->devs[di];
    DeviceGuard guard(d.id);
    return finish(d, stream_of(stream));
  });
}

int g4m_fp8_quantize(g4m_ctx* ctx, int di, int act, const void* x, int dtype, int64_t ldx, int64_t rows, int cols,
                     const g4m_fp8_rows* out, void* stream) {
  return no_throw([&]() -> int {
    if (act < G4M_ACT_NONE || act > G4M_ACT_GELU_TANH) return fail(G4M_E_ARG, "unknown activation " + std::to_string(act));
    if (!dtype_ok(dtype)) return fail(G4M_E_ARG, "unknown dtype " + std::to_string(dtype));
    if (rows < 0 || cols <= 0) return fail(G4M_E_ARG, "rows must not be negative and d must be positive");
    if (cols > kFp8MaxCols) return fail(G4M_E_UNSUPPORTED, "d = " + std::to_string(cols) + " is above " + std::to_string(kFp8MaxCols));
    QuantArgs a;
    a.blocks = (cols - 1) / kFp8Block + 1;
    if (rows > INT_MAX / a.blocks) return fail(G4M_E_UNSUPPORTED, "more than 2^31 - 1 blocks of 128 columns in one call");
    if (rows > 0) {
      if (!x || !out) return fail(G4M_E_ARG, "null x or out");
      const int64_t width = act == G4M_ACT_NONE ? (int64_t)cols : 2 * (int64_t)cols;
      int rc = check_rows("x", x, ldx, width, dtype);
      if (!rc) rc = check_fp8("out", *out, rows, cols);
      if (rc) return rc;
    }
    if (!device_ok(ctx, di)) return fail(G4M_E_ARG, "bad context or device index");
    if (rows == 0) return G4M_OK;
    a.x = x;
    a.ldx = ldx;
    a.units = (uint32_t)(rows * a.blocks);
    a.d = cols;
    a.act = act;
    a.dtype = dtype;
    const int64_t size = dtype_size(dtype);
    a.full = cols % 8 == 0 && rows16(x, ldx, size) && (act == G4M_ACT_NONE || rows16((const char*)x + cols * size, ldx, size));
    a.codes = out->codes;
    a.ldc = out->ldc;
    a.scales = out->scales;
    a.lds = out->lds;
    Device& d = *ctx->devs[di];
    DeviceGuard guard(d.id);
    cudaStream_t st = stream_of(stream);
    G4M_RUN("fp8_quantize", fp8_quantize(a, d.id, st));
    return G4M_OK;
  });
}

int g4m_norm_residual(g4m_ctx* ctx, int di, const g4m_norm_args* args, void* stream) {
  return no_throw([&]() -> int {
    if (!args) return fail(G4M_E_ARG, "null args");
    const g4m_norm_args& a = *args;
    if (!dtype_ok(a.dtype) || !dtype_ok(a.h_dtype)) return fail(G4M_E_ARG, "unknown dtype");
    if (a.rows < 0 || a.d <= 0) return fail(G4M_E_ARG, "rows must not be negative and d must be positive");
    if (a.d > kNormMaxD) return fail(G4M_E_UNSUPPORTED, "d = " + std::to_string(a.d) + " is above " + std::to_string(kNormMaxD));
    if (a.rows > INT_MAX) return fail(G4M_E_UNSUPPORTED, "more than 2^31 - 1 rows in one call");
    if (!(a.eps >= 0.0f) || isinf(a.eps)) return fail(G4M_E_ARG, "eps must be finite and not negative");
    int rc = a.rows > 0 ? check_norm(a) : G4M_OK;
    if (rc) return rc;
    if (!device_ok(ctx, di)) return fail(G4M_E_ARG, "bad context or device index");
    if (a.rows == 0) return G4M_OK;
    Device& d = *ctx->devs[di];
    DeviceGuard guard(d.id);
    cudaStream_t st = stream_of(stream);
    G4M_RUN("norm_residual", norm_residual(a, d.id, st));
    return G4M_OK;
  });
}

int g4m_fp8_linear_prepare(g4m_ctx* ctx, int di, const uint8_t* w, const float* w_scales, int out, int in,
                           const float* bias, g4m_fp8_linear** out_linear) {
  return no_throw([&]() -> int {
    if (!device_ok(ctx, di) || !w || !w_scales || !out_linear || in <= 0 || out <= 0) return fail(G4M_E_ARG, "bad argument");
    if (in > kFp8MaxCols || out > kFp8MaxCols)
      return fail(G4M_E_UNSUPPORTED, "in or out is above " + std::to_string(kFp8MaxCols));
    Device& d = *ctx->devs[di];
    DeviceGuard guard(d.id);
    g4m_fp8_linear* L = new g4m_fp8_linear();
    L->d = &d;
    L->dev = d.id;
    L->in = in;
    L->out = out;
    uint8_t* raw = nullptr;
    std::vector<float> padded;
    if (bias) {
      padded.assign((size_t)(fp8_blocks(out) + 1) / 2 * 2 * kFp8Block, 0.0f);
      memcpy(padded.data(), bias, (size_t)out * sizeof(float));
    }
    const bool ok = fp8_gemm_setup() == cudaSuccess && to_device(&raw, w, (size_t)out * in) &&
                    cudaMalloc(&L->w, fp8_weight_bytes(out, in)) == cudaSuccess &&
                    fp8_weight_tiles(raw, out, in, L->w, cudaStreamLegacy) == cudaSuccess &&
                    to_device(&L->sw, w_scales, (size_t)(fp8_blocks(out) * fp8_blocks(in))) &&
                    (!bias || to_device(&L->bias, padded.data(), padded.size())) &&
                    cudaStreamSynchronize(cudaStreamLegacy) == cudaSuccess;
    if (raw) cudaFree(raw);
    if (!ok) {
      (void)cudaGetLastError();
      g4m_fp8_linear_free(L);
      return fail(G4M_E_CUDA, "8-bit float linear: weight upload failed");
    }
    *out_linear = L;
    return G4M_OK;
  });
}

int g4m_fp8_linear_run(g4m_fp8_linear* L, const g4m_fp8_rows* x, int64_t rows, void* y, int y_dtype, int64_t ldy,
                       void* stream) {
  return no_throw([&]() -> int {
    if (!L || rows < 0) return fail(G4M_E_ARG, "null linear or negative rows");
    if (!dtype_ok(y_dtype)) return fail(G4M_E_ARG, "unknown dtype " + std::to_string(y_dtype));
    if (rows == 0) return G4M_OK;
    if (!x || !y) return fail(G4M_E_ARG, "null x or y");
    if (rows > INT_MAX - 1024) return fail(G4M_E_UNSUPPORTED, "too many rows in one call");
    int rc = check_fp8("x", *x, rows, L->in);
    if (!rc) rc = check_rows("y", y, ldy, L->out, y_dtype);
    if (rc) return rc;
    Device& d = *L->d;
    DeviceGuard guard(L->dev);
    cudaStream_t st = stream_of(stream);
    Fp8GemmArgs a;
    a.rows = rows;
    a.in = L->in;
    a.out = L->out;
    a.x = x->codes;
    a.ldx = x->ldc;
    a.sx = x->scales;
    a.lds = x->lds;
    a.w = L->w;
    a.sw = L->sw;
    a.bias = L->bias;
    a.y = y;
    a.y_dtype = y_dtype;
    a.y_vec = rows16(y, ldy, dtype_size(y_dtype));
    a.ldy = ldy;
    a.err = d.err;
    G4M_RUN("fp8_gemm", fp8_gemm(a, L->dev, st));
    return G4M_OK;
  });
}

void g4m_fp8_linear_free(g4m_fp8_linear* L) {
  if (!L) return;
  DeviceGuard guard(L->dev);
  if (L->w) cudaFree(L->w);
  if (L->sw) cudaFree(L->sw);
  if (L->bias) cudaFree(L->bias);
  delete L;
}

int g4m_rope_frequencies(int rotary, double theta, int scaling, double factor, double low, double high, double trained,
                         double* inv_freq, double* attention_scale) {
  return no_throw([&]() -> int {
    if (rotary < 2 || rotary % 2 != 0) return fail(G4M_E_SHAPE, "rotary must be even and at least 2");
    if (!inv_freq || !attention_scale) return fail(G4M_E_ARG, "null output");
    if (scaling < G4M_ROPE_NONE || scaling > G4M_ROPE_YARN) return fail(G4M_E_ARG, "unknown scaling " + std::to_string(scaling));
    if (!(theta > 0) || isinf(theta)) return fail(G4M_E_ARG, "theta must be positive");
    if (scaling != G4M_ROPE_NONE && (!(factor > 0) || isinf(factor))) return fail(G4M_E_ARG, "factor must be positive");
    const bool bands = scaling == G4M_ROPE_BANDED || scaling == G4M_ROPE_YARN;
    if (bands && (!(low > 0) || !(high > low) || isinf(high) || !(trained > 0) || isinf(trained)))
      return fail(G4M_E_ARG, "0 < low < high and trained > 0 are needed");
    if (scaling == G4M_ROPE_YARN && !(theta > 1)) return fail(G4M_E_ARG, "theta must be above 1 for this scaling");
    const double two_pi = 6.283185307179586476925287;
    // the pair index at which `turns` whole turns fall within the trained positions
    auto index_of = [&](double turns) { return rotary * log(trained / (turns * two_pi)) / (2.0 * log(theta)); };
    double first = 0, last = 1;
    if (scaling == G4M_ROPE_YARN) {
      first = fmax(floor(index_of(high)), 0.0);
      last = fmin(ceil(index_of(low)), rotary - 1.0);
    }
    for (int j = 0; j < rotary / 2; ++j) {
      const double f = pow(theta, -2.0 * j / rotary);
      double keep = 1.0;  // share of the unstretched frequency
      if (scaling == G4M_ROPE_LINEAR) keep = 0.0;
      if (scaling == G4M_ROPE_BANDED) keep = fmin(fmax((trained * f / two_pi - low) / (high - low), 0.0), 1.0);
      if (scaling == G4M_ROPE_YARN) keep = 1.0 - fmin(fmax((j - first) / fmax(last - first, 0.001), 0.0), 1.0);
      inv_freq[j] = scaling == G4M_ROPE_NONE ? f : keep * f + (1.0 - keep) * f / factor;
    }
    // only a stretch raises the attention's temperature
    *attention_scale = scaling == G4M_ROPE_YARN && factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0;
    return G4M_OK;
  });
}

int g4m_rope_prepare(g4m_ctx* ctx, int di, int head_dim, int rotary, const double* inv_freq, double scale, int interleaved,
                     g4m_rope** out_rope) {
  return no_throw([&]() -> int {
    if (!device_ok(ctx, di) || !inv_freq || !out_rope) return fail(G4M_E_ARG, "bad argument");
    if (rotary < 2 || rotary % 2 != 0 || rotary > head_dim)
      return fail(G4M_E_SHAPE, "rotary must be even, at least 2 and at most head_dim");
    if (head_dim > 1024) return fail(G4M_E_UNSUPPORTED, "head_dim above 1024");
    if (!isfinite((float)scale)) return fail(G4M_E_ARG, "scale is not finite");
    std::vector<uint64_t> turns(rotary / 2);
    for (int j = 0; j < rotary / 2; ++j) {
      if (!isfinite(inv_freq[j])) return fail(G4M_E_ARG, "a frequency is not finite");
      // whole turns per position drop out at integer positions
      const long double t = (long double)inv_freq[j] / 6.283185307179586476925286766559L;
      const long double frac = t - floorl(t);  // [0, 1]
      const long double fixed = floorl(frac * 18446744073709551616.0L + 0.5L);
      turns[j] = fixed >= 18446744073709551616.0L ? 0 : (uint64_t)fixed;
    }
    Device& d = *ctx->devs[di];
    DeviceGuard guard(d.id);
    g4m_rope* R = new g4m_rope();
    R->d = &d;
    R->dev = d.id;
    R->head_dim = head_dim;
    R->half = rotary / 2;
    R->interleaved = interleaved != 0;
    R->scale = (float)scale;
    if (!to_device(&R->turns, turns.data(), turns.size())) {
      (void)cudaGetLastError();
      g4m_rope_free(R);
      return fail(G4M_E_CUDA, "rotary table upload failed");
    }
    *out_rope = R;
    return G4M_OK;
  });
}

int g4m_rope_run(g4m_rope* R, const g4m_rope_view* q, const g4m_rope_view* k, int dtype, int64_t tokens,
                 const void* positions, int pos_bits, void* stream) {
  return no_throw([&]() -> int {
    if (!R || !q) return fail(G4M_E_ARG, "null rope or q");
    if (!dtype_ok(dtype)) return fail(G4M_E_ARG, "unknown dtype " + std::to_string(dtype));
    if (pos_bits != 32 && pos_bits != 64) return fail(G4M_E_ARG, "pos_bits must be 32 or 64");
    if (tokens < 0) return fail(G4M_E_ARG, "negative tokens");
    if (tokens > INT_MAX) return fail(G4M_E_UNSUPPORTED, "more than 2^31 - 1 tokens in one call");
    RopeArgs a;
    memset(&a, 0, sizeof(a));
    const int64_t size = dtype_size(dtype);
    bool vec = R->half % 8 == 0;
    int64_t heads = 0;
    const g4m_rope_view* views[2] = {q, k};
    for (int i = 0; i < 2; ++i) {
      if (!views[i]) continue;
      const g4m_rope_view& v = *views[i];
      if (v.heads < 0) return fail(G4M_E_ARG, "negative heads");
      heads += v.heads;
      if (v.heads == 0 || tokens == 0) continue;
      if (!v.x || !v.out) return fail(G4M_E_ARG, "null heads pointer");
      if (!aligned(v.x, size) || !aligned(v.out, size)) return fail(G4M_E_ARG, "a heads pointer is not aligned to its elements");
      const bool in_place = v.out == v.x;
      if (in_place && ((tokens > 1 && v.out_token_stride != v.token_stride) || (v.heads > 1 && v.out_head_stride != v.head_stride)))
        return fail(G4M_E_ARG, "in place, out needs the strides of x");
      // no two (token, head) pairs may share an output element
      const int64_t hs = v.heads > 1 ? v.out_head_stride : 0, ts = tokens > 1 ? v.out_token_stride : 0, hd = R->head_dim;
      if (hs < 0 || ts < 0 || (v.heads > 1 && hs < hd) || (tokens > 1 && ts < hd) ||
          (v.heads > 1 && tokens > 1 && (ts - hd) / (v.heads - 1) < hs && (hs - hd) / (tokens - 1) < ts))
        return fail(G4M_E_SHAPE, "out strides make heads overlap");
      a.v[i] = v;
      a.copy[i] = !in_place && R->head_dim > 2 * R->half;
      vec = vec && aligned(v.x, 16) && aligned(v.out, 16) && (v.token_stride * size) % 16 == 0 &&
            (v.head_stride * size) % 16 == 0 && (v.out_token_stride * size) % 16 == 0 && (v.out_head_stride * size) % 16 == 0;
    }
    if (heads == 0 || tokens == 0) return G4M_OK;
    if (heads > 65535) return fail(G4M_E_UNSUPPORTED, "more than 65535 heads");
    if (!positions || !aligned(positions, pos_bits / 8)) return fail(G4M_E_ARG, "positions are null or not aligned");
    a.turns = R->turns;
    a.scale = R->scale;
    a.head_dim = R->head_dim;
    a.half = R->half;
    a.interleaved = R->interleaved;
    a.dtype = dtype;
    a.vec = vec;
    a.pos64 = pos_bits == 64;
    a.tokens = tokens;
    a.positions = positions;
    Device& d = *R->d;
    DeviceGuard guard(R->dev);
    cudaStream_t st = stream_of(stream);
    G4M_RUN("rope", rope_run(a, R->dev, st));
    return G4M_OK;
  });
}

void g4m_rope_free(g4m_rope* R) {
  if (!R) return;
  DeviceGuard guard(R->dev);
  if (R->turns) cudaFree(R->turns);
  delete R;
}

}  // extern "C"
