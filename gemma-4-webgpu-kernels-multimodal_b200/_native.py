"""ctypes bindings to libg4m.so, the CUDA (sm_100a) library behind the API.

There is no CPU fallback: if the library is missing or cannot load, every
entry point raises.
"""
from __future__ import annotations

import ctypes
import os
import weakref

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libg4m.so")

G4M_OK = 0
STATUS_NAMES = {0: "OK", 1: "E_ARG", 2: "E_SHAPE", 3: "E_DTYPE", 4: "E_CUDA", 5: "E_TIMEOUT", 6: "E_CANCELLED",
                7: "E_IO", 8: "E_NOT_LOADED", 9: "E_UNSUPPORTED", 10: "E_LAYOUT"}

# (name, restype, argtypes) for every function declared in include/g4m.h
_VP = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_D = ctypes.c_double
_I64 = ctypes.c_int64
_SIGS = [
    ("g4m_create", _VP, [_VP, _I]),
    ("g4m_destroy", None, [_VP]),
    ("g4m_device_count", _I, [_VP]),
    ("g4m_last_error", ctypes.c_char_p, []),
    ("g4m_load_weights", _I, [_VP, ctypes.c_char_p]),
    ("g4m_loaded_towers", _I, [_VP]),
    ("g4m_cancel", None, [_VP]),
    ("g4m_clear_cancel", None, [_VP]),
    ("g4m_set_debug", _I, [_VP, _I]),
    ("g4m_qat_linear", _I, [_VP, _I, _VP, _I, _I, _I, _VP, _I, _VP, _F, _F, _VP, _VP]),
    ("g4m_linear_prepare", _I, [_VP, _I, _VP, _I, _I, _I, _VP, _F, _F, _VP, ctypes.POINTER(_VP)]),
    ("g4m_linear_run", _I, [_VP, _VP, _I, _VP, _VP]),
    ("g4m_linear_free", None, [_VP]),
    ("g4m_linear_run_noalloc", _I, [_VP, _VP, _I, _VP, _VP]),
    ("g4m_vision_embed_images", _I, [_VP, _I, _VP, _VP, _VP, _I, _I, _I, _VP, _VP, _VP]),
    ("g4m_resize_rgb", _I, [_VP, _I, _VP, _I, _I, _I, _I, _I, _VP]),
    ("g4m_selftest_wait_timeout", _I, [_VP, _I, ctypes.c_longlong]),
    ("g4m_synchronize", _I, [_VP, _I, _VP]),
    ("g4m_fp8_quantize", _I, [_VP, _I, _I, _VP, _I, _I64, _I64, _I, _VP, _VP]),
    ("g4m_fp8_linear_prepare", _I, [_VP, _I, _VP, _VP, _I, _I, _VP, ctypes.POINTER(_VP)]),
    ("g4m_fp8_linear_run", _I, [_VP, _VP, _I64, _VP, _I, _I64, _VP]),
    ("g4m_fp8_linear_free", None, [_VP]),
    ("g4m_norm_residual", _I, [_VP, _I, _VP, _VP]),
    ("g4m_rope_frequencies", _I, [_I, _D, _I, _D, _D, _D, _D, ctypes.POINTER(_D), ctypes.POINTER(_D)]),
    ("g4m_rope_prepare", _I, [_VP, _I, _I, _I, _VP, _D, _I, ctypes.POINTER(_VP)]),
    ("g4m_rope_run", _I, [_VP, _VP, _VP, _I, _I64, _VP, _I, _VP]),
    ("g4m_rope_free", None, [_VP]),
    ("g4m_vision_embed_batch", _I, [_VP, _I, _VP, _I, _I, _I, _I, _VP, _VP, _VP]),
    ("g4m_vision_embed_device", _I, [_VP, _I, _I, _VP, _I, _I, _I, _I, _VP, _VP]),
    ("g4m_vision_debug_hidden", _I, [_VP, _I, _I, _VP, ctypes.c_size_t]),
    ("g4m_vision_layers", _I, [_VP, _I, _I, _I, _I, _I, _I, _VP]),
    ("g4m_audio_embed_batch", _I, [_VP, _I, _VP, _VP, _I, _I, _I64, _VP, _VP, _VP]),
    ("g4m_audio_embed_device", _I, [_VP, _I, _I, _VP, _VP, _VP, _I, _I, _I64, _VP, _VP, _VP]),
    ("g4m_audio_debug_hidden", _I, [_VP, _I, _I, _VP, ctypes.c_size_t]),
    ("g4m_audio_layers", _I, [_VP, _I, _I, _VP, _I, _I, _VP]),
    ("g4m_image_token_layout", _I, [_I, _I, _I, _I, _I, ctypes.POINTER(_I64)]),
    ("g4m_audio_soft_token_count", _I64, [_I64, _I, _I, _I]),
    ("g4m_checksum_floats", ctypes.c_double, [_VP, _I64]),
    ("g4m_profile_begin", _I, [_VP, _I]),
    ("g4m_profile_end", _I, [_VP, _I, ctypes.c_char_p, ctypes.c_size_t]),
    ("g4m_kernel_launches", ctypes.c_longlong, []),
    ("g4m_version", ctypes.c_char_p, []),
]

# element types, gated activations and frequency scalings (enums of include/g4m.h)
F32, BF16, F16 = 0, 1, 2
ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2}
ROPE_SCALINGS = {"none": 0, "linear": 1, "banded": 2, "yarn": 3}


class Fp8Rows(ctypes.Structure):
    """g4m_fp8_rows: device pointers of e4m3 codes and their block scales."""
    _fields_ = [("codes", _VP), ("ldc", _I64), ("scales", _VP), ("lds", _I64)]


class NormArgs(ctypes.Structure):
    """g4m_norm_args."""
    _fields_ = [("rows", _I64), ("d", ctypes.c_int32), ("dtype", ctypes.c_int32), ("h_dtype", ctypes.c_int32), ("eps", _F),
                ("y", _VP), ("ldy", _I64), ("w_post", _VP), ("norm_post", ctypes.c_int32), ("norm_pre", ctypes.c_int32),
                ("gate", _VP), ("ldg", _I64), ("rows_per_gate", _I64), ("branch_scale", _F), ("res_scale", _F),
                ("h", _VP), ("ldh", _I64), ("h_out", _VP), ("ldh_out", _I64), ("w_pre", _VP), ("n_out", _VP),
                ("ldn", _I64), ("out", Fp8Rows)]


class RopeView(ctypes.Structure):
    """g4m_rope_view."""
    _fields_ = [("x", _VP), ("token_stride", _I64), ("head_stride", _I64), ("out", _VP), ("out_token_stride", _I64),
                ("out_head_stride", _I64), ("heads", ctypes.c_int32)]


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"libg4m.so is not built ({LIB_PATH}); run build() first -- there is no CPU fallback")
        L = ctypes.CDLL(LIB_PATH)
        for name, res, args in _SIGS:
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def exported_names():
    return [s[0] for s in _SIGS]


class G4MError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"{STATUS_NAMES.get(status, status)}: {message}")
        self.status = status
        self.message = message


def last_error() -> str:
    m = lib().g4m_last_error()
    return m.decode() if m else ""


def check(rc: int) -> None:
    if rc != G4M_OK:
        raise G4MError(rc, last_error())


def ptr(a: np.ndarray):
    return ctypes.c_void_p(a.ctypes.data)


class Context:
    """Owns a g4m_ctx (resident weights on one or more CUDA devices)."""

    def __init__(self, devices=None):
        L = lib()
        if devices:
            arr = (ctypes.c_int * len(devices))(*devices)
            self.h = L.g4m_create(ctypes.cast(arr, ctypes.c_void_p), len(devices))
        else:
            self.h = L.g4m_create(None, 0)
        if not self.h:
            raise G4MError(4, last_error())
        self._handles = weakref.WeakSet()  # linears and rotary tables, freed before the context

    def close(self):
        if getattr(self, "h", None):
            for handle in list(getattr(self, "_handles", ())):
                handle.close()
            lib().g4m_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def device_count(self) -> int:
        return lib().g4m_device_count(self.h)

    def load_weights(self, path: str) -> None:
        check(lib().g4m_load_weights(self.h, path.encode()))

    @property
    def loaded_towers(self) -> int:
        return lib().g4m_loaded_towers(self.h)

    def cancel(self):
        lib().g4m_cancel(self.h)

    def clear_cancel(self):
        lib().g4m_clear_cancel(self.h)

    def profile_begin(self, device=0):
        check(lib().g4m_profile_begin(self.h, device))

    def profile_end(self, device=0) -> dict:
        import json
        buf = ctypes.create_string_buffer(1 << 16)
        check(lib().g4m_profile_end(self.h, device, buf, len(buf)))
        return {k: (int(v[0]), float(v[1])) for k, v in json.loads(buf.value.decode()).items()}

    def set_debug(self, on: bool):
        check(lib().g4m_set_debug(self.h, 1 if on else 0))

    def qat_linear(self, x, w, w_scale, s_in=0.0, s_out=0.0, bias=None, bits=0, in_dim=None, device=0) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        rows, inp = x.shape
        if bits == 0:
            w = np.ascontiguousarray(w, dtype=np.int8)
            out = w.shape[0]
        else:
            w = np.ascontiguousarray(w, dtype=np.uint8)
            out = w.shape[0]
        s = np.ascontiguousarray(w_scale, dtype=np.float32).reshape(-1)
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32).reshape(-1)
        y = np.empty((rows, out), np.float32)
        check(lib().g4m_qat_linear(self.h, device, ptr(x), rows, inp, out, ptr(w), bits, ptr(s), float(s_in), float(s_out),
                                   None if b is None else ptr(b), ptr(y)))
        return y

    def vision_embed(self, pixels_list, max_soft_tokens=280, layer_count=16, outs=None):
        """pixels_list: list of float32 [h, w, 3] arrays of one size; `outs`
        optionally supplies the [tokens, 1536] float32 output arrays."""
        n = len(pixels_list)
        if n == 0:
            return [], []
        h, w = pixels_list[0].shape[:2]
        pix = [np.ascontiguousarray(p, dtype=np.float32) for p in pixels_list]
        lay = (ctypes.c_int64 * 6)()
        check(lib().g4m_image_token_layout(h, w, 16, max_soft_tokens, 3, lay))
        tokens = lay[5]
        if outs is None:
            outs = [np.empty((tokens, 1536), np.float32) for _ in range(n)]
        elif any(o.shape != (tokens, 1536) or o.dtype != np.float32 or not o.flags.c_contiguous for o in outs):
            raise ValueError("outs must be C-contiguous float32 [tokens, 1536] arrays")
        pin = (ctypes.c_void_p * n)(*[p.ctypes.data for p in pix])
        pout = (ctypes.c_void_p * n)(*[o.ctypes.data for o in outs])
        rows = np.zeros(n, np.int32)
        status = np.zeros(n, np.int32)
        rc = lib().g4m_vision_embed_batch(self.h, n, ctypes.cast(pin, ctypes.c_void_p), h, w, max_soft_tokens, layer_count,
                                          ctypes.cast(pout, ctypes.c_void_p), ptr(rows), ptr(status))
        check(rc)
        return outs, rows

    def vision_embed_images(self, images, max_soft_tokens=280, layer_count=16):
        """images: list of uint8 [h, w, 3 | 4] arrays of any sizes (one channel
        count).  Returns ([tokens_i, 1536] float32 arrays, rows, statuses);
        per-image failures are reported in the statuses, not raised."""
        n = len(images)
        if n == 0:
            return [], np.zeros(0, np.int32), np.zeros(0, np.int32)
        imgs = [np.ascontiguousarray(im, dtype=np.uint8) for im in images]
        ch = imgs[0].shape[2]
        if any(im.ndim != 3 or im.shape[2] != ch for im in imgs):
            raise ValueError("images must be [h, w, c] uint8 with one channel count")
        hs = np.array([im.shape[0] for im in imgs], np.int32)
        ws = np.array([im.shape[1] for im in imgs], np.int32)
        outs = []
        for im in imgs:
            lay = (ctypes.c_int64 * 6)()
            rc = lib().g4m_image_token_layout(im.shape[0], im.shape[1], 16, max_soft_tokens, 3, lay)
            outs.append(np.empty((max(int(lay[5]), 1) if rc == 0 else 1, 1536), np.float32))
        pin = (ctypes.c_void_p * n)(*[im.ctypes.data for im in imgs])
        pout = (ctypes.c_void_p * n)(*[o.ctypes.data for o in outs])
        rows = np.zeros(n, np.int32)
        status = np.zeros(n, np.int32)
        rc = lib().g4m_vision_embed_images(self.h, n, ctypes.cast(pin, ctypes.c_void_p), ptr(hs), ptr(ws), ch,
                                           max_soft_tokens, layer_count, ctypes.cast(pout, ctypes.c_void_p),
                                           ptr(rows), ptr(status))
        if rc and not (status != 0).any():
            check(rc)
        return [o[: int(r)] for o, r in zip(outs, rows)], rows, status

    def resize_rgb(self, image, target_height: int, target_width: int, device=0) -> np.ndarray:
        im = np.ascontiguousarray(image, dtype=np.uint8)
        out = np.empty((target_height, target_width, 3), np.float32)
        check(lib().g4m_resize_rgb(self.h, device, ptr(im), im.shape[0], im.shape[1], im.shape[2], target_height,
                                   target_width, ptr(out)))
        return out

    def vision_embed_device(self, pixels_ptr: int, n: int, height: int, width: int, out_ptr: int, max_soft_tokens=280,
                            layer_count=16, stream: int = 0, device=0) -> None:
        check(lib().g4m_vision_embed_device(self.h, device, n, ctypes.c_void_p(pixels_ptr), height, width, max_soft_tokens,
                                            layer_count, ctypes.c_void_p(out_ptr), ctypes.c_void_p(stream) if stream else None))

    def vision_debug_hidden(self, which: int, rows: int, device=0) -> np.ndarray:
        out = np.empty((rows, 768), np.float32)
        check(lib().g4m_vision_debug_hidden(self.h, device, which, ptr(out), out.size))
        return out

    def vision_layers(self, h: np.ndarray, n: int, height: int, width: int, first: int, count: int, device=0) -> np.ndarray:
        h = np.ascontiguousarray(h, dtype=np.float32).copy()
        check(lib().g4m_vision_layers(self.h, device, n, height, width, first, count, ptr(h)))
        return h

    def audio_embed(self, clips, sampling_rate=16000, layer_count=12, max_samples=0, outs=None):
        """clips: list of float32 sample arrays; `outs` optionally supplies
        C-contiguous float32 output arrays of at least [rows_i, 1536] each."""
        n = len(clips)
        xs = [np.ascontiguousarray(c, dtype=np.float32).reshape(-1) for c in clips]
        lens = np.array([x.size for x in xs], np.int64)
        cap = max_samples if max_samples else 480000
        need = [int(lib().g4m_audio_soft_token_count(min(x.size, cap), 320, 160, 750)) for x in xs]
        if outs is None:
            outs = [np.empty((max(r, 1), 1536), np.float32) for r in need]
        elif any(o.dtype != np.float32 or not o.flags.c_contiguous or o.ndim != 2 or o.shape[1] != 1536
                 or o.shape[0] < r for o, r in zip(outs, need)):
            raise ValueError("outs must be C-contiguous float32 [>= rows, 1536] arrays")
        pin = (ctypes.c_void_p * n)(*[x.ctypes.data for x in xs])
        pout = (ctypes.c_void_p * n)(*[o.ctypes.data for o in outs])
        rows = np.zeros(n, np.int32)
        status = np.zeros(n, np.int32)
        check(lib().g4m_audio_embed_batch(self.h, n, ctypes.cast(pin, ctypes.c_void_p), ptr(lens), sampling_rate, layer_count,
                                          int(max_samples), ctypes.cast(pout, ctypes.c_void_p), ptr(rows), ptr(status)))
        return [o[: int(r)] for o, r in zip(outs, rows)], rows

    def audio_debug_hidden(self, rows: int, which: int = 1, device=0) -> np.ndarray:
        out = np.empty((rows, 3072 if which == 2 else 1024), np.float32)
        check(lib().g4m_audio_debug_hidden(self.h, device, which, ptr(out), out.size))
        return out

    def audio_layers(self, h: np.ndarray, rows_per_clip, first: int, count: int, device=0) -> np.ndarray:
        h = np.ascontiguousarray(h, dtype=np.float32).copy()
        rows = np.ascontiguousarray(rows_per_clip, dtype=np.int32)
        check(lib().g4m_audio_layers(self.h, device, rows.size, ptr(rows), first, count, ptr(h)))
        return h

    def audio_embed_device(self, samples_ptr: int, offsets: np.ndarray, lengths: np.ndarray, out_ptr: int,
                           sampling_rate=16000, layer_count=12, max_samples=0, stream: int = 0, device=0) -> np.ndarray:
        offsets = np.ascontiguousarray(offsets, dtype=np.int64)
        lengths = np.ascontiguousarray(lengths, dtype=np.int64)
        rows = np.zeros(offsets.size, np.int32)
        check(lib().g4m_audio_embed_device(self.h, device, offsets.size, ctypes.c_void_p(samples_ptr), ptr(offsets),
                                           ptr(lengths), sampling_rate, layer_count, int(max_samples),
                                           ctypes.c_void_p(out_ptr), ptr(rows), ctypes.c_void_p(stream) if stream else None))
        return rows

    def synchronize(self, stream: int = 0, device=0) -> None:
        """Wait for the stream; raises E_TIMEOUT when a device-side wait expired
        in a call since the last report."""
        check(lib().g4m_synchronize(self.h, device, stream or None))

    def fp8_quantize(self, x: int, dtype: int, ldx: int, rows: int, d: int, codes: int, ldc: int, scales: int, lds: int,
                     act="none", stream: int = 0, device=0) -> None:
        """g4m_fp8_quantize on device pointers; act: "none", "silu" or "gelu"."""
        check(lib().g4m_fp8_quantize(self.h, device, ACTIVATIONS[act], x, dtype, ldx, rows, d,
                                     ctypes.byref(Fp8Rows(codes, ldc, scales, lds)), stream or None))

    def norm_residual(self, args: NormArgs, stream: int = 0, device=0) -> None:
        """g4m_norm_residual; args as norm_args() builds them."""
        check(lib().g4m_norm_residual(self.h, device, ctypes.byref(args), stream or None))

    def fp8_linear(self, w, w_scales, bias=None, device=0) -> "Fp8Linear":
        """Resident 8-bit float linear: w uint8 e4m3 codes [out, in], w_scales
        float32 [ceil(out / 128), ceil(in / 128)], bias float32 [out]."""
        return Fp8Linear(self, w, w_scales, bias, device)

    def rope(self, head_dim: int, inv_freq, interleaved=False, attention_scale=1.0, device=0) -> "Rope":
        """Rotary positions on the first 2 * len(inv_freq) elements of each head."""
        return Rope(self, head_dim, inv_freq, interleaved, attention_scale, device)


class _Handle:
    """A resident object of a context; close() frees it, at the latest when the context closes."""
    _free = ""

    def __init__(self, ctx):
        if not ctx.h:
            raise G4MError(1, "the context is closed")
        self._h = ctypes.c_void_p()
        ctx._handles.add(self)
        self._ctx = ctx

    def close(self):
        if getattr(self, "_h", None):
            getattr(lib(), self._free)(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Fp8Linear(_Handle):
    _free = "g4m_fp8_linear_free"

    def __init__(self, ctx, w, w_scales, bias=None, device=0):
        super().__init__(ctx)
        w = np.ascontiguousarray(w)
        if w.dtype != np.uint8 or w.ndim != 2:
            raise ValueError("w must be uint8 e4m3 codes [out, in]")
        self.out_features, self.in_features = w.shape
        s = np.ascontiguousarray(w_scales, dtype=np.float32)
        want = (-(-self.out_features // 128), -(-self.in_features // 128))
        if s.shape != want:
            raise ValueError(f"w_scales must be float32 {list(want)}, one for each 128 x 128 block")
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        if b is not None and b.shape != (self.out_features,):
            raise ValueError("bias must be float32 [out]")
        check(lib().g4m_fp8_linear_prepare(ctx.h, device, ptr(w), ptr(s), self.out_features, self.in_features,
                                           None if b is None else ptr(b), ctypes.byref(self._h)))

    def run(self, codes: int, ldc: int, scales: int, lds: int, rows: int, y: int, y_dtype: int, ldy: int,
            stream: int = 0) -> None:
        """g4m_fp8_linear_run on device pointers."""
        check(lib().g4m_fp8_linear_run(self._h, ctypes.byref(Fp8Rows(codes, ldc, scales, lds)), rows, y, y_dtype, ldy,
                                       stream or None))


class Rope(_Handle):
    _free = "g4m_rope_free"

    def __init__(self, ctx, head_dim, inv_freq, interleaved=False, attention_scale=1.0, device=0):
        super().__init__(ctx)
        f = np.ascontiguousarray(inv_freq, dtype=np.float64).reshape(-1)
        check(lib().g4m_rope_prepare(ctx.h, device, head_dim, 2 * f.size, ptr(f), float(attention_scale), int(interleaved),
                                     ctypes.byref(self._h)))

    def run(self, q: RopeView, k, dtype: int, tokens: int, positions: int, pos_bits=64, stream: int = 0) -> None:
        """g4m_rope_run: q and (or None) k as rope_view() builds them, positions a device pointer."""
        check(lib().g4m_rope_run(self._h, ctypes.byref(q), None if k is None else ctypes.byref(k), dtype, tokens, positions,
                                 pos_bits, stream or None))


def norm_args(**fields) -> NormArgs:
    """g4m_norm_args; fields left out are 0 / NULL, the scales 1, rows_per_gate
    1, and codes, ldc, scales, lds name the 8-bit output."""
    out = Fp8Rows(*(fields.pop(k, 0) for k in ("codes", "ldc", "scales", "lds")))
    return NormArgs(**{"branch_scale": 1.0, "res_scale": 1.0, "rows_per_gate": 1, **fields, "out": out})


def rope_view(x: int, token_stride: int, head_stride: int, out: int, out_token_stride: int, out_head_stride: int,
              heads: int) -> RopeView:
    return RopeView(x, token_stride, head_stride, out, out_token_stride, out_head_stride, heads)


def rope_frequencies(rotary: int, theta: float, scaling="none", factor=1.0, low=1.0, high=32.0, trained=1.0):
    """(float64 [rotary / 2] radians per position, attention scale) of g4m_rope_frequencies."""
    f, m = (ctypes.c_double * max(rotary // 2, 1))(), ctypes.c_double()
    check(lib().g4m_rope_frequencies(rotary, theta, ROPE_SCALINGS[scaling], factor, low, high, trained, f, ctypes.byref(m)))
    return np.array(f), m.value


def image_token_layout(height: int, width: int, patch_size: int, max_soft_tokens: int, pooling_kernel_size: int):
    out = (ctypes.c_int64 * 6)()
    check(lib().g4m_image_token_layout(int(height), int(width), int(patch_size), int(max_soft_tokens),
                                       int(pooling_kernel_size), out))
    return list(out)


def audio_soft_token_count(samples: int, frame_length: int, hop_length: int, audio_seq_length: int) -> int:
    return int(lib().g4m_audio_soft_token_count(int(samples), int(frame_length), int(hop_length), int(audio_seq_length)))


def checksum_floats(values: np.ndarray) -> int:
    v = np.ascontiguousarray(values, dtype=np.float32).reshape(-1)
    return int(lib().g4m_checksum_floats(ptr(v), v.size))


def kernel_launches() -> int:
    return int(lib().g4m_kernel_launches())


def version() -> str:
    return lib().g4m_version().decode()
