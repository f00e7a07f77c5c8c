"""CPU tests of the 8-bit float operators' host side: argument checks (they
come before the context, so no device is needed) and rotary frequencies."""
import ctypes

import numpy as np
import pytest

ARG, SHAPE, UNSUPPORTED = 1, 2, 9
P = 1 << 20  # a 16-byte aligned address that is never read


def quantize(native, act=0, x=P, dtype=1, ldx=256, rows=4, d=200, codes=P, ldc=208, scales=P, lds=4, out=True):
    o = native.Fp8Rows(codes, ldc, scales, lds)
    return native.lib().g4m_fp8_quantize(None, 0, act, x, dtype, ldx, rows, d, ctypes.byref(o) if out else None, None)


@pytest.mark.parametrize("bad,status,says", [
    (dict(act=3), ARG, "activation"), (dict(act=-1), ARG, "activation"), (dict(dtype=3), ARG, "dtype"),
    (dict(rows=-1), ARG, "negative"), (dict(d=0), ARG, "positive"), (dict(x=None), ARG, "null"), (dict(out=False), ARG, "null"),
    (dict(x=P + 1), ARG, "aligned"), (dict(dtype=0, x=P + 2), ARG, "aligned"), (dict(ldx=199), SHAPE, "stride"),
    (dict(act=1), SHAPE, "stride"), (dict(codes=P + 8), ARG, "16-byte"), (dict(ldc=204), ARG, "16-byte"),
    (dict(ldc=192), SHAPE, "stride"), (dict(scales=P + 2), ARG, "scales"), (dict(codes=None), ARG, "null"),
    (dict(scales=None), ARG, "null"), (dict(lds=3), SHAPE, "scales stride"),
    (dict(rows=1 << 30, lds=1 << 30), UNSUPPORTED, "blocks"), (dict(d=(1 << 24) + 1, ldx=1 << 25, ldc=1 << 25), UNSUPPORTED, "above"), (dict(), ARG, "context"), (dict(rows=0, x=None), ARG, "context"),
])
def test_quantize_refuses(native, bad, status, says):
    assert quantize(native, **bad) == status
    assert says in native.last_error(), native.last_error()


def norm(native, **kw):
    f = dict(rows=4, d=200, dtype=1, h_dtype=1, eps=1e-6, y=P, ldy=200, h=2 * P, ldh=200, h_out=3 * P, ldh_out=200,
             n_out=4 * P, ldn=200, codes=5 * P, ldc=208, scales=6 * P, lds=4, norm_post=1, norm_pre=1)
    f.update(kw)
    return native.lib().g4m_norm_residual(None, 0, ctypes.byref(native.norm_args(**f)), None)


@pytest.mark.parametrize("bad,status,says", [
    (dict(dtype=4), ARG, "dtype"), (dict(h_dtype=-1), ARG, "dtype"), (dict(rows=-2), ARG, "negative"), (dict(d=0), ARG, "positive"),
    (dict(d=16385, ldy=20000), UNSUPPORTED, "16384"), (dict(rows=1 << 31), UNSUPPORTED, "rows"),
    (dict(eps=-1.0), ARG, "eps"), (dict(eps=float("nan")), ARG, "eps"), (dict(eps=float("inf")), ARG, "eps"),
    (dict(y=0, h=0), ARG, "neither"), (dict(y=0, gate=P, ldg=200), ARG, "gate needs"),
    (dict(h_out=0, n_out=0, codes=0), ARG, "no output"), (dict(gate=P, ldg=200, rows_per_gate=0), ARG, "rows_per_gate"),
    (dict(gate=P, ldg=100), SHAPE, "gate"), (dict(w_post=P + 1), ARG, "weight"), (dict(w_pre=P + 2), ARG, "weight"),
    (dict(h_out=2 * P, ldh_out=208), ARG, "in place"), (dict(n_out=P, ldn=208), ARG, "in place"),
    (dict(n_out=3 * P), ARG, "same buffer"), (dict(ldy=199), SHAPE, "y:"), (dict(ldh=199), SHAPE, "h:"),
    (dict(ldh_out=199), SHAPE, "h_out"), (dict(ldn=199), SHAPE, "n_out"), (dict(y=P + 1), ARG, "y:"),
    (dict(h_dtype=0, h=2 * P + 2), ARG, "h:"), (dict(ldc=200), ARG, "16-byte"), (dict(scales=0), ARG, "null"),
    (dict(lds=3), SHAPE, "scales"), (dict(), ARG, "context"), (dict(rows=0, y=0, h=0), ARG, "context"),
])
def test_norm_refuses(native, bad, status, says):
    assert norm(native, **bad) == status
    assert says in native.last_error(), native.last_error()


def test_handles_refuse(native):
    L = native.lib()
    h = ctypes.c_void_p()
    assert L.g4m_fp8_linear_prepare(None, 0, P, P, 8, 8, None, ctypes.byref(h)) == ARG and not h.value
    v = native.rope_view(P, 8, 8, P, 8, 8, 1)
    assert L.g4m_rope_prepare(None, 0, 8, 8, P, 1.0, 0, ctypes.byref(h)) == ARG and not h.value
    assert L.g4m_fp8_linear_run(None, ctypes.byref(native.Fp8Rows(P, 16, P, 4)), 1, P, 0, 8, None) == ARG
    assert L.g4m_rope_run(None, ctypes.byref(v), None, 0, 1, P, 64, None) == ARG
    L.g4m_fp8_linear_free(None)
    L.g4m_rope_free(None)


def test_synchronize_refuses(native):
    assert native.lib().g4m_synchronize(None, 0, None) == ARG and "context" in native.last_error()
    assert native.lib().g4m_selftest_wait_timeout(None, 0, -5) == ARG


@pytest.mark.parametrize("bad,status", [
    (dict(rotary=7), SHAPE), (dict(rotary=0), SHAPE), (dict(theta=0.0), ARG), (dict(theta=float("nan")), ARG),
    (dict(scaling="linear", factor=0.0), ARG), (dict(scaling="banded", factor=2.0, low=4.0, high=4.0, trained=64), ARG),
    (dict(scaling="yarn", factor=2.0, low=0.0, high=4.0, trained=64), ARG),
    (dict(scaling="yarn", factor=2.0, low=1.0, high=4.0, trained=0), ARG),
    (dict(scaling="yarn", theta=1.0, factor=2.0, low=1.0, high=4.0, trained=64), ARG),
])
def test_rope_frequencies_refuse(native, bad, status):
    with pytest.raises(native.G4MError) as e:
        native.rope_frequencies(**{"rotary": 64, "theta": 10000.0, **bad})
    assert e.value.status == status


@pytest.mark.parametrize("rotary,theta", [(2, 10000.0), (64, 10000.0), (36, 500000.0), (256, 1e6)])
def test_rope_frequencies(native, rotary, theta):
    """Each frequency within a few roundings (relative 2^-50) of the formula."""
    j = np.arange(rotary // 2)
    f = theta ** (-2.0 * j / rotary)
    got, m = native.rope_frequencies(rotary, theta)
    np.testing.assert_allclose(got, f, rtol=2.0 ** -50)
    assert m == 1.0
    got, m = native.rope_frequencies(rotary, theta, "linear", factor=8.0)
    np.testing.assert_allclose(got, f / 8, rtol=2.0 ** -50)
    assert m == 1.0
    got, m = native.rope_frequencies(rotary, theta, "banded", factor=8.0, low=1.0, high=4.0, trained=8192)
    turns = 8192 * f / (2 * np.pi)
    blend = (turns - 1) / 3
    exp = np.where(turns < 1, f / 8, np.where(turns > 4, f, (1 - blend) * f / 8 + blend * f))
    np.testing.assert_allclose(got, exp, rtol=2.0 ** -48)
    assert m == 1.0
    got, m = native.rope_frequencies(rotary, theta, "yarn", factor=16.0, low=1.0, high=32.0, trained=4096)
    at = lambda n: rotary * np.log(4096 / (n * 2 * np.pi)) / (2 * np.log(theta))  # noqa: E731
    lo, hi = max(np.floor(at(32.0)), 0), min(np.ceil(at(1.0)), rotary - 1)
    ramp = np.clip((j - lo) / max(hi - lo, 0.001), 0, 1)
    np.testing.assert_allclose(got, f * (1 - ramp) + f / 16 * ramp, rtol=2.0 ** -48)
    assert abs(m - (0.1 * np.log(16) + 1)) < 1e-15


@pytest.mark.parametrize("factor,scale", [(0.25, 1.0), (0.999, 1.0), (1.0, 1.0), (1.5, 0.1 * np.log(1.5) + 1), (40.0, 0.1 * np.log(40.0) + 1)])
def test_rope_yarn_scale_never_shrinks(native, factor, scale):
    """Factors up to 1 leave the attention scale at 1; the frequencies follow the factor either way."""
    f, m = native.rope_frequencies(64, 10000.0, "yarn", factor=factor, low=1.0, high=32.0, trained=4096)
    assert abs(m - scale) < 1e-15
    np.testing.assert_allclose(f[-1], 10000.0 ** (-62 / 64) / factor, rtol=2.0 ** -48)


def test_python_side_refuses(native):
    """Shapes that the bindings know are refused before anything reaches the library."""
    class Ctx:
        h = None
    with pytest.raises(native.G4MError):
        native.Fp8Linear(Ctx(), np.zeros((8, 8), np.uint8), np.ones((1, 1), np.float32))
    Ctx.h, Ctx._handles = 1, set()
    with pytest.raises(ValueError):
        native.Fp8Linear(Ctx(), np.zeros((8, 8), np.int8), np.ones((1, 1), np.float32))
    with pytest.raises(ValueError):
        native.Fp8Linear(Ctx(), np.zeros((130, 8), np.uint8), np.ones((1, 1), np.float32))
    with pytest.raises(ValueError):
        native.Fp8Linear(Ctx(), np.zeros((8, 8), np.uint8), np.ones((1, 1), np.float32), bias=np.zeros(7, np.float32))
