"""GPU tests of the 8-bit float operators against plain evaluations in 64 bits.

Rounding to type t moves a value by at most eps(t)/2 of itself (H below); f32
work inside the kernels adds terms that each test derives beside its bound.
"""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}
H = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}            # half a step among the f16 subnormals
U = 2.0 ** -24
FLOOR = 2.0 ** -96


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows_like(rows, d, pad, off, dtype, g, scale=1.0):
    """[rows, d] view with row stride d + pad that starts `off` elements into its buffer."""
    buf = (scale * torch.randn(rows * (d + pad) + off, device="cuda", generator=g)).to(dtype)
    return buf, buf[off:off + rows * (d + pad)].view(rows, d + pad)[:, :d]


class Codes:
    """An 8-bit operand's buffers, filled with marks; `padded` leaves spare rows, columns and scale places."""

    def __init__(self, rows, d, padded=False):
        self.rows, self.d = rows, d
        ld = (d + 15) // 16 * 16 + (32 if padded else 0)
        self.lds = rows + (5 if padded else 0)
        self.buf = torch.full((rows + 2, ld), 0xAB, dtype=torch.uint8, device="cuda")
        self.sbuf = torch.full(((d + 127) // 128 + 1, self.lds), -7.0, device="cuda")

    @property
    def fields(self):
        return dict(codes=self.buf.data_ptr(), ldc=self.buf.shape[1], scales=self.sbuf.data_ptr(), lds=self.lds)

    @property
    def args(self):
        return self.buf.data_ptr(), self.buf.shape[1], self.sbuf.data_ptr(), self.lds

    def codes(self):
        return self.buf[:self.rows, :self.d].view(torch.float8_e4m3fn)

    def scales(self):
        return self.sbuf[:(self.d + 127) // 128, :self.rows]

    def values(self):
        s = self.scales().double().t().repeat_interleave(128, 1)[:, :self.d]
        return self.codes().double() * s

    def assert_rest_untouched(self):
        assert (self.buf[:self.rows, self.d:] == 0xAB).all() and (self.buf[self.rows:] == 0xAB).all()
        assert (self.sbuf[:, self.rows:] == -7.0).all() and (self.sbuf[-1] == -7.0).all()


def block_amax(v):
    b = torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 128)).view(v.shape[0], -1, 128)
    return b.amax(2)


def assert_codes(c, v, err):
    """c holds v, known to `err` (absolute, elementwise).  The scale is the
    block's largest magnitude / 448, known to that element's error and two
    roundings; a code is off by half an e4m3 step of the quotient, 2^-4 of it
    or 2^-10 among the subnormals, and by the quotient's own error."""
    s = (block_amax(v).clamp_min(FLOOR) / 448).t()
    serr = block_amax(err).t() / 448 + 3 * U * s
    assert ((c.scales().double() - s).abs() <= serr).all()
    per = c.scales().double().t().repeat_interleave(128, 1)[:, :v.shape[1]]
    rel = (serr / s).t().repeat_interleave(128, 1)[:, :v.shape[1]] + 4 * U
    q = v.abs() / per
    # a quotient above 448 by its error saturates: within the same bound
    bound = per * (torch.maximum(q * 2.0 ** -4, torch.full_like(q, 2.0 ** -10)) + q * rel) * (1 + 2.0 ** -4) + err * (1 + 2.0 ** -4)
    bad = (c.values() - v).abs() > bound
    assert not bad.any(), (bad.sum().item(), (c.values() - v)[bad][:4], bound[bad][:4])
    c.assert_rest_untouched()


# ------------------------------------------------------------------- quantise

def act64(x, d, act):
    """Value and its f32 evaluation error (absolute).  sigmoid(z) through
    exp2 and a reciprocal: relative |dz| + 2^-22 + 2^-23 + a rounding, with z
    known to 6 roundings; then two products."""
    if act == "none":
        return x, torch.zeros_like(x)
    g, u = x[:, :d], x[:, d:]
    z = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    v = g / (1 + torch.exp(-z)) * u
    return v, v.abs() * U * (6 * z.abs() + 12) + 2.0 ** -120


@pytest.mark.parametrize("rows,d,pad,off", [(1, 1, 0, 0), (1, 128, 0, 0), (3, 129, 0, 0), (5, 127, 1, 1), (17, 1000, 24, 0),
                                            (33, 1536, 0, 8), (2, 4097, 7, 3), (257, 768, 0, 0), (1, 12288, 0, 0), (100, 40, 3, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_quantize(ctx, rows, d, pad, off, dtype, act):
    w = d if act == "none" else 2 * d
    buf, x = rows_like(rows, w, pad, off, DT[dtype][1], gen(rows * 7 + d), 3.0)
    c = Codes(rows, d, padded=rows % 2 == 1)
    ctx.fp8_quantize(x.data_ptr(), DT[dtype][0], w + pad, rows, d, *c.args, act=act, stream=stream())
    v, err = act64(x.double(), d, act)
    assert_codes(c, v, err)
    if act == "none":  # exact inputs: the codes of a true division, bit for bit
        # (torch divides a GPU tensor by a number through its reciprocal: numpy divides)
        s = torch.from_numpy(block_amax(x.float()).clamp_min(FLOOR).cpu().numpy() / np.float32(448)).cuda()
        assert torch.equal(c.scales(), s.t())
        q = (x.float() / s.repeat_interleave(128, 1)[:, :d]).to(torch.float8_e4m3fn)
        assert torch.equal(c.codes().view(torch.uint8), q.view(torch.uint8))


def test_quantize_next_to_ties(ctx):
    """Quotients within a few units of the borders between codes, for scales of
    all kinds, the all-ones mantissa among them: bit for bit those of a true
    division."""
    rng = np.random.default_rng(5)
    v = np.arange(127, dtype=np.uint8)  # the magnitudes, and the borders between them
    mag = torch.from_numpy(v).view(torch.float8_e4m3fn).double().numpy()
    ties = (mag[1:] + mag[:-1]) / 2
    amax = [np.float32((3.5 - 2.0 ** -22) * 2.0 ** k) for k in range(-90, 120, 3)]
    amax += [np.float32(m * 2.0 ** k) for m, k in zip(rng.uniform(1, 2, 3000), rng.integers(-94, 126, 3000))]
    x = np.zeros((len(amax), 256), np.float32)
    for r, a in enumerate(amax):
        s = np.float32(a) / np.float32(448)
        near = (ties * np.float64(s)).astype(np.float32)
        x[r, :126], x[r, 128:254] = near, -near
        step = rng.integers(-2, 3, 256).astype(np.int32)
        x[r] = np.where(x[r] != 0, (x[r].view(np.int32) + step).view(np.float32), 0)
        x[r, 126:128], x[r, 254:] = (a, np.float32(2.0 ** -17) * a / np.float32(3.5)), (-a, -a * np.float32(2.0 ** -19))
    x = np.where(np.abs(x) > np.array(amax, np.float32)[:, None], np.array(amax, np.float32)[:, None], x)
    x[:70, 127], x[:70, 255] = [2.0 ** (k - 17) for k in range(-90, 120, 3)], [-(2.0 ** (k - 17)) for k in range(-90, 120, 3)]
    s = (np.array(amax, np.float32) / np.float32(448))[:, None]
    exp = torch.from_numpy(x / s).to(torch.float8_e4m3fn).view(torch.uint8)
    c, xd = Codes(len(amax), 256), torch.from_numpy(x).cuda()
    ctx.fp8_quantize(xd.data_ptr(), 0, 256, len(amax), 256, *c.args, stream=stream())
    assert torch.equal(c.scales().cpu(), torch.from_numpy(np.repeat(s.T, 2, 0)))
    bad = c.codes().view(torch.uint8).cpu() != exp
    assert not bad.any(), (bad.sum().item(), x[bad.numpy()][:4])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize_keeps_the_sign_of_zero(ctx, native, dtype):
    """Codes of zeros and of values that round to zero carry their sign, as a
    true division's do: from the quantiser and from the norm."""
    g = gen(77)
    x = torch.randn(40, 384, device="cuda", generator=g)
    x *= torch.randint(0, 2, x.shape, device="cuda", generator=g)  # zeros of either sign
    x[3] = 0.0
    x[4] = -0.0
    x[5, 1:] *= 2.0 ** -12
    x = x.to(DT[dtype][1])
    assert (x.double().signbit() & (x == 0)).any()
    s = torch.from_numpy(block_amax(x.float()).clamp_min(FLOOR).cpu().numpy() / np.float32(448)).cuda()
    exp = (x.float() / s.repeat_interleave(128, 1)).to(torch.float8_e4m3fn).view(torch.uint8)
    c, n = Codes(40, 384), Codes(40, 384)
    ctx.fp8_quantize(x.data_ptr(), DT[dtype][0], 384, 40, 384, *c.args, stream=stream())
    ctx.norm_residual(native.norm_args(rows=40, d=384, dtype=DT[dtype][0], h_dtype=DT[dtype][0], eps=0.0, h=x.data_ptr(), ldh=384, **n.fields),
                      stream=stream())
    assert torch.equal(c.scales(), s.t()) and torch.equal(n.scales(), s.t())
    assert torch.equal(c.codes().view(torch.uint8), exp)
    # the norm adds its absent branch: h + 1 * (+0), which makes -0 a +0
    zero = x == 0
    assert torch.equal(n.codes().view(torch.uint8)[~zero], exp[~zero]) and (n.codes().view(torch.uint8)[zero] == 0).all()


def test_quantize_special_blocks(ctx):
    """Zeros, the least and largest magnitudes, and blocks with an infinity or NaN: those read NaN whole, their neighbours are not touched by it."""
    x = torch.ones(8, 300, device="cuda")
    x[0] = 0
    x[1] = 1e-44
    x[2] = 3e38
    x[3, 5] = float("inf")
    x[4, 140] = float("nan")
    x[5, 299] = -float("inf")
    x[6] = -0.0
    x[7, :128] = 2.0 ** -97
    c = Codes(8, 300, padded=True)
    ctx.fp8_quantize(x.data_ptr(), 0, 300, 8, 300, *c.args, stream=stream())
    v, s = c.values(), c.scales()
    assert (v[0] == 0).all() and (s[:, 0].double() - FLOOR / 448).abs().max() <= U * FLOOR / 448
    assert (v[1] == 0).all() and (v[6] == 0).all()
    np.testing.assert_allclose(v[2].cpu(), np.float32(3e38), rtol=2.0 ** -22)
    assert v[3, :128].isnan().all() and s[0, 3].isnan() and (v[3, 128:] - 1).abs().max() <= 2.0 ** -22
    assert v[4, 128:256].isnan().all() and s[1, 4].isnan() and (v[4, :128] - 1).abs().max() <= 2.0 ** -22 and v[4, 256:].isfinite().all()
    assert v[5, 256:].isnan().all() and s[2, 5].isnan() and v[5, :256].isfinite().all()
    np.testing.assert_allclose(v[7, :128].cpu(), 2.0 ** -97, rtol=2.0 ** -22)  # 224 exactly, under the floored scale
    c.assert_rest_untouched()


# ----------------------------------------------------------------------- norm

def norm64(y, h, wp, gate, rpg, wn, bs, rs, norm_post, norm_pre, eps):
    """h', n and the errors of their f32 evaluation.  A sum of squares is a
    chain of at most 32 fma per thread and 10 joins (relative 42 U, halved by
    the root), then root, quotient and products: 28 U in all."""
    b = e = torch.zeros((), dtype=torch.float64, device="cuda")
    if y is not None:
        b = y
        if norm_post:
            b = y / torch.sqrt(y.square().mean(1, keepdim=True) + eps) * (1.0 if wp is None else wp)
        e = 28 * U * b.abs()
        if gate is not None:
            g = gate[torch.arange(y.shape[0], device="cuda") // rpg]
            b, e = b * g, e * g.abs()
    hh = h if h is not None else torch.zeros_like(y)
    out = rs * (hh + bs * b)
    e = abs(rs) * (abs(bs) * e + 4 * U * ((bs * b).abs() + hh.abs()))
    if not norm_pre:
        return out, out, e, e
    inv = 1 / torch.sqrt(out.square().mean(1, keepdim=True) + eps)
    w = 1.0 if wn is None else wn
    n = out * inv * w
    # the root mean square moves by at most the root mean square of e
    drift = torch.sqrt(e.square().mean(1, keepdim=True)) * inv
    wa = 1.0 if wn is None else wn.abs()
    return out, n, e, (e * inv * wa + n.abs() * (drift + 28 * U)) * (1 + 2.0 ** -10)


def run_norm(ctx, native, rows, d, dtype, res, pad, off, rpg, outs, seed, norm_post=1, norm_pre=1, has_y=True, has_h=True,
             weights=True, bs=0.5, rs=0.875, in_place=False):
    g = gen(seed)
    dt, rt = DT[dtype][1], DT[res][1]
    yb, y = rows_like(rows, d, pad, off, dt, g, 1.5)
    hb, h = rows_like(rows, d, pad, off, rt, g, 4.0)
    wp = 1 + 0.3 * torch.randn(d + 1, device="cuda", generator=g)[1 if off else 0:][:d]
    wn = 1 + 0.3 * torch.randn(d + 1, device="cuda", generator=g)[1 if off else 0:][:d]
    gates = None
    if rpg:
        gb, gates = rows_like(-(-rows // rpg), d, pad, off, dt, g)
    ref = norm64(y.double() if has_y else None, h.double() if has_h else None, wp.double() if weights else None,
                 None if gates is None else gates.double(), rpg, wn.double() if weights else None, bs, rs, norm_post, norm_pre, 1e-6)
    ho = torch.full((rows + 1, d + pad), 9.0, dtype=rt, device="cuda")
    no = torch.full((rows + 1, d + pad), 9.0, dtype=dt, device="cuda")
    c = Codes(rows, d, padded=pad > 0)
    a = dict(rows=rows, d=d, dtype=DT[dtype][0], h_dtype=DT[res][0], eps=1e-6, norm_post=norm_post, norm_pre=norm_pre,
             branch_scale=bs, res_scale=rs)
    if has_y:
        a.update(y=y.data_ptr(), ldy=d + pad, w_post=wp.data_ptr() if weights else 0)
    if has_h:
        a.update(h=h.data_ptr(), ldh=d + pad)
    if weights:
        a.update(w_pre=wn.data_ptr())
    if gates is not None:
        a.update(gate=gates.data_ptr(), ldg=d + pad, rows_per_gate=rpg)
    if "h" in outs:
        a.update(h_out=(h if in_place else ho).data_ptr(), ldh_out=d + pad)
    if "n" in outs:
        a.update(n_out=(y if in_place else no).data_ptr(), ldn=d + pad)
    if "c" in outs:
        a.update(**c.fields)
    ctx.norm_residual(native.norm_args(**a), stream=stream())
    torch.cuda.synchronize()
    eh, en, erh, ern = ref
    for what, got, exp, err, t in (("h", h if in_place else ho[:rows, :d], eh, erh, res), ("n", y if in_place else no[:rows, :d], en, ern, dtype)):
        if what in outs:
            bound = err * (1 + H[t]) + H[t] * exp.abs() + TINY[t]
            bad = (got.double() - exp).abs() > bound
            assert not bad.any(), (what, bad.sum().item(), got[bad][:4], exp[bad][:4], bound[bad][:4])
    if not in_place:
        for buf, used in ((ho, "h" in outs), (no, "n" in outs)):
            assert (buf[rows:] == 9).all() and (buf[:rows, d:] == 9).all() and (used or (buf == 9).all())
    if "c" in outs:
        assert_codes(c, en, ern)


@pytest.mark.parametrize("rows,d,pad,off", [(1, 1, 0, 0), (1, 1536, 0, 0), (3, 7, 0, 0), (5, 255, 1, 1), (64, 256, 8, 0),
                                            (130, 768, 0, 0), (19, 1155, 0, 0), (7, 4096, 16, 8), (3, 4100, 0, 0), (2, 8192, 0, 0),
                                            (2, 8200, 3, 1), (2, 16384, 0, 0), (1, 16383, 2, 0), (2311, 33, 0, 0)])
@pytest.mark.parametrize("dtype,res", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "bf16")])
def test_norm(ctx, native, rows, d, pad, off, dtype, res):
    run_norm(ctx, native, rows, d, dtype, res, pad, off, rpg=(rows + 2) // 3, outs="hnc", seed=rows + d)


@pytest.mark.parametrize("opts", [
    dict(outs="h"), dict(outs="n"), dict(outs="c"), dict(outs="hn"), dict(outs="hc"), dict(rpg=0), dict(rpg=1), dict(rpg=10 ** 12),
    dict(has_y=False, rpg=0), dict(has_h=False), dict(norm_post=0), dict(norm_pre=0), dict(norm_post=0, norm_pre=0, outs="hnc"),
    dict(weights=False), dict(bs=0.0), dict(rs=-2.0), dict(in_place=True, outs="hn"), dict(in_place=True, outs="hnc"),
])
@pytest.mark.parametrize("d", [96, 1000, 5000])
def test_norm_options(ctx, native, opts, d):
    run_norm(ctx, native, **{**dict(rows=37, d=d, dtype="bf16", res="bf16", pad=0, off=0, rpg=5, outs="hnc", seed=d), **opts})


@pytest.mark.parametrize("rows,d", [(9000, 1000), (9000, 1155), (4000, 4096), (700, 16384)])
def test_rows_that_blocks_walk(ctx, native, rows, d):
    """More rows than the grid holds at a time."""
    run_norm(ctx, native, rows, d, "bf16", "f32", 0, 0, rpg=1000, outs="hnc", seed=d)
    buf, x = rows_like(rows, 2 * d, 0, 0, torch.bfloat16, gen(d), 3.0)
    c = Codes(rows, d)
    ctx.fp8_quantize(x.data_ptr(), 1, 2 * d, rows, d, *c.args, act="silu", stream=stream())
    assert_codes(c, *act64(x.double(), d, "silu"))


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("d", [256, 1024, 4096, 8192])
def test_norm_one_sum_many_rows(ctx, native, post, d):
    """One of the two norms alone over many rows per block: consecutive sums
    of a block are then those of different rows.  Rows differ by powers of two
    up to 2^20, so a sum of another row shows."""
    rows = 20000
    g = gen(d + post)
    x = torch.randn(rows, d, device="cuda", generator=g)
    x *= torch.exp2(torch.randint(-10, 11, (rows, 1), device="cuda", generator=g).float())
    x = x.bfloat16()
    out = torch.empty_like(x)
    a = dict(rows=rows, d=d, dtype=DT["bf16"][0], h_dtype=DT["bf16"][0], eps=0.0)
    if post:
        a.update(y=x.data_ptr(), ldy=d, norm_post=1, h_out=out.data_ptr(), ldh_out=d)
    else:
        a.update(h=x.data_ptr(), ldh=d, norm_pre=1, n_out=out.data_ptr(), ldn=d)
    first = None
    for _ in range(10):
        out.zero_()
        ctx.norm_residual(native.norm_args(**a), stream=stream())
        if first is None:
            first = out.clone()
            for r in range(0, rows, 4000):
                v = x[r:r + 4000].double()
                exp = v / torch.sqrt(v.square().mean(1, keepdim=True))
                assert ((out[r:r + 4000].double() - exp).abs() <= (28 * U + H["bf16"] * (1 + 28 * U)) * exp.abs()).all()
        assert torch.equal(out, first)


def test_norm_rows_that_are_not_finite(ctx, native):
    """A row with a NaN or an infinity spoils itself alone; a row of zeros gives zeros (eps keeps the root above zero)."""
    d = 300
    h = torch.ones(5, d, device="cuda")
    h[1, 3] = float("nan")
    h[2, 3] = float("inf")
    h[3] = 0
    n = torch.empty_like(h)
    c = Codes(5, d)
    ctx.norm_residual(native.norm_args(rows=5, d=d, dtype=0, h_dtype=0, eps=1e-6, norm_pre=1, h=h.data_ptr(), ldh=d,
                                       n_out=n.data_ptr(), ldn=d, **c.fields), stream=stream())
    assert n[1].isnan().all() and n[2, 3].isnan() and (n[2, 4:] == 0).all()
    assert (n[3] == 0).all() and (c.values()[3] == 0).all()
    for r in (0, 4):
        assert (n[r].double() - 1 / math.sqrt(1 + 1e-6)).abs().max() <= 28 * U
        assert c.values()[r].isfinite().all()
    assert c.values()[1].isnan().all() and c.values()[2, :128].isnan().all()


# --------------------------------------------------------------------- linear

def linear_case(rows, i, o, seed, exact=False, padded=True):
    """An 8-bit operand and weights.  exact: codes of small integers and scales
    that are powers of two, so that every product and every sum is exact in
    f32 in any order and results can be compared bit for bit."""
    g = gen(seed)
    c = Codes(rows, i, padded)
    kb, nb = (i + 127) // 128, (o + 127) // 128
    if exact:
        x = torch.randint(-3, 4, (rows, i), device="cuda", generator=g).float()
        w = torch.randint(-3, 4, (o, i), device="cuda", generator=g).float()
        sx = 2.0 ** torch.randint(-2, 3, (kb, rows), device="cuda", generator=g).float()
        sw = 2.0 ** torch.randint(-2, 3, (nb, kb), device="cuda", generator=g).float()
    else:
        x = 60 * torch.randn(rows, i, device="cuda", generator=g)
        w = 60 * torch.randn(o, i, device="cuda", generator=g)
        sx = torch.exp(torch.randn(kb, rows, device="cuda", generator=g))
        sw = torch.exp(torch.randn(nb, kb, device="cuda", generator=g))
    c.buf[:] = 0x7F  # NaN wherever nothing should be read
    c.sbuf[:] = float("nan")
    c.buf[:rows, :i] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    c.sbuf[:kb, :rows] = sx
    wc = w.clamp(-448, 448).to(torch.float8_e4m3fn)
    bias = torch.randint(-8, 9, (o,), device="cuda", generator=g).float()
    return c, wc, sw, bias


def linear64(c, wc, sw, bias):
    """The sum and the sum of magnitudes."""
    ws = sw.double().repeat_interleave(128, 0)[:wc.shape[0]].repeat_interleave(128, 1)[:, :wc.shape[1]]
    x, w = c.values(), wc.double() * ws
    y, m = x @ w.t(), x.abs() @ w.abs().t()
    return (y, m) if bias is None else (y + bias.double(), m + bias.abs().double())


def run_linear(ctx, c, wc, sw, bias, dtype, pad=0, off=0, st=None):
    o, i = wc.shape
    lin = ctx.fp8_linear(wc.view(torch.uint8).cpu().numpy(), sw.cpu().numpy(), None if bias is None else bias.cpu().numpy())
    y = torch.full(((c.rows + 1) * (o + pad) + off,), 5.0, dtype=DT[dtype][1], device="cuda")
    lin.run(*c.args, c.rows, y[off:].data_ptr(), DT[dtype][0], o + pad, stream=stream() if st is None else st)
    torch.cuda.synchronize()
    lin.close()
    v = y[off:].view(c.rows + 1, o + pad)
    assert (v[:c.rows, o:] == 5).all() and (v[c.rows:] == 5).all() and (y[:off] == 5).all()
    return v[:c.rows, :o]


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 100, 37), (1, 1536, 6144), (3, 129, 257), (8, 2048, 1000), (15, 640, 255), (16, 768, 2304),
          (17, 768, 300), (31, 4000, 500), (33, 96, 1030), (64, 1024, 512), (65, 257, 129), (100, 512, 777), (127, 384, 640),
          (128, 1536, 1536), (129, 1024, 1537), (200, 130, 2050), (256, 4096, 256), (300, 1100, 1300), (511, 640, 384),
          (513, 768, 3000), (1000, 500, 999), (2304, 768, 2304), (4100, 1024, 520), (1, 5000, 11000), (300, 9000, 1300),
          (600, 4500, 2600), (40, 260, 20000)]


@pytest.mark.parametrize("rows,i,o", SHAPES)
def test_linear_exact(ctx, rows, i, o):
    """Sums that are exact in f32 (|sum| < 2^24 steps of 2^-4): bit for bit."""
    c, wc, sw, bias = linear_case(rows, i, o, rows + i + o, exact=True)
    y, m = linear64(c, wc, sw, bias)
    assert m.max() < 2.0 ** 20
    assert torch.equal(run_linear(ctx, c, wc, sw, bias, "f32").double(), y)
    for dtype in ("bf16", "f16"):
        got = run_linear(ctx, c, wc, sw, None, dtype, pad=3, off=1)
        assert torch.equal(got, linear64(c, wc, sw, None)[0].float().to(DT[dtype][1])), dtype


@pytest.mark.parametrize("rows,i,o", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear(ctx, rows, i, o, dtype):
    """A 128-column block is four tensor-core steps of 32 products; a step
    aligns its terms and the accumulator to the largest of them and drops what
    falls below f32's last place, at most 2^-23 of it for each of 33 terms:
    4 * 33 * 2^-23 of the block's magnitudes.  Each block then adds three
    roundings, of which the running total's can reach all earlier ones."""
    c, wc, sw, bias = linear_case(rows, i, o, 3 * rows + i + o)
    bias = bias if rows % 2 else None
    y, m = linear64(c, wc, sw, bias)
    got = run_linear(ctx, c, wc, sw, bias, dtype, pad=8).double()
    bound = m * (4 * 33 * 2.0 ** -23 + (3 + (i + 127) // 128) * U) + H[dtype] * y.abs()
    bad = (got - y).abs() > bound
    assert not bad.any(), (bad.sum().item(), got[bad][:4], y[bad][:4], bound[bad][:4])


@pytest.mark.parametrize("rows,i,o", [(33, 640, 40000), (70, 200, 9001), (90, 300, 37000), (150, 1300, 2561), (260, 100, 129), (390, 400, 9400),
                                      (2500, 256, 2600), (3000, 200, 2049), (2400, 384, 2176), (5000, 128, 1000)])
@pytest.mark.parametrize("dtype,pad,off", [("f32", 0, 0), ("f32", 1, 1), ("bf16", 8, 0), ("f16", 3, 1)])
def test_linear_last_tiles(ctx, rows, i, o, dtype, pad, off):
    """Numbers of 128 x 256 tiles below and above a multiple of the SMs, so
    that the last ones are whole, halved or quartered.  Exact in f32; rounded
    once otherwise."""
    c, wc, sw, bias = linear_case(rows, i, o, rows + o, exact=True)
    y = run_linear(ctx, c, wc, sw, bias, dtype, pad, off)
    exp, _ = linear64(c, wc, sw, bias)
    assert torch.equal(y, exp.to(DT[dtype][1]))


@pytest.mark.parametrize("rows,i,o", [(128 * 37, 640, 2048), (128 * 31, 300, 2001), (128 * 89, 384, 1024), (128 * 79 - 5, 700, 1001),
                                      (128 * 111, 100, 500)])
@pytest.mark.parametrize("dtype,pad,off", [("f32", 0, 0), ("f32", 7, 0), ("bf16", 7, 0), ("f16", 4, 4), ("bf16", 3, 1)])
def test_linear_several_tiles_each(ctx, rows, i, o, dtype, pad, off):
    """Two or more whole 128 x 256 tiles for a thread block (on 148 SMs), with
    a last round that is full, whole, halved and quartered; widths that end
    inside a 16-byte piece of rows with a stride of whole pieces.  Exact in
    f32; rounded once otherwise."""
    c, wc, sw, bias = linear_case(rows, i, o, rows + o, exact=True)
    y = run_linear(ctx, c, wc, sw, bias, dtype, pad, off)
    assert torch.equal(y, linear64(c, wc, sw, bias)[0].to(DT[dtype][1]))


@pytest.mark.parametrize("rows,i,o,dtype", [(128 * 700, 128, 1000, "f32"), (128 * 700, 128, 800, "bf16"), (128 * 300, 128, 2344, "f32"),
                                            (128 * 460, 100, 40, "f32"), (128 * 460, 128, 24, "f16"), (128 * 75, 128, 1032, "f32")])
def test_linear_odd_stores_then_more_tiles(ctx, rows, i, o, dtype):
    """Tiles whose last store blocks number odd (y ends inside the tile), each
    followed by further tiles of the same thread block with one column block
    of sums: the store that still reads a block of shared memory and the next
    tile's first write must not meet.  Exact sums, so any value of another
    tile shows; repeated, as an overlap is a matter of time."""
    c, wc, sw, bias = linear_case(rows, i, o, rows + o, exact=True, padded=False)
    lin = ctx.fp8_linear(wc.view(torch.uint8).cpu().numpy(), sw.cpu().numpy(), bias.cpu().numpy())
    y = torch.empty(rows, o, dtype=DT[dtype][1], device="cuda")
    exp = linear64(c, wc, sw, bias)[0].to(DT[dtype][1])
    for _ in range(8):
        y.fill_(5.0)
        for _ in range(3):
            lin.run(*c.args, rows, y.data_ptr(), DT[dtype][0], o, stream=stream())
        assert torch.equal(y, exp)
    lin.close()


def test_linear_nan_stays_in_its_row(ctx):
    """NaN codes, NaN and infinite scales reach only the rows (or the output blocks) they belong to."""
    for rows in (4, 200):
        c, wc, sw, _ = linear_case(rows, 300, 300, 5, exact=True)
        c.buf[1, 7] = 0x7F
        c.sbuf[2, 3] = float("nan")
        sw[1, 0] = float("inf")
        got = run_linear(ctx, c, wc, sw, None, "f32")
        ok = torch.ones(rows, dtype=torch.bool, device="cuda")
        ok[1] = ok[3] = False
        assert got[~ok].isnan().all()
        assert got[ok][:, :128].isfinite().all() and got[ok][:, 256:].isfinite().all()
        assert not got[ok][:, 128:256].isfinite().any()
        sw[1, 0] = 1.0
        c2, wc2, _, _ = linear_case(rows, 300, 300, 5, exact=True)
        assert torch.equal(got[ok][:, :128].double(), linear64(c2, wc2, sw, None)[0][ok][:, :128])


def test_linear_repeats_bit_for_bit(ctx):
    """No order of arrival decides a result: repeated calls agree bit for bit."""
    for rows, i, o in [(1, 4096, 1536), (24, 2048, 777), (700, 1024, 1000)]:
        c, wc, sw, bias = linear_case(rows, i, o, 9)
        first = run_linear(ctx, c, wc, sw, bias, "f32").clone()
        for _ in range(3):
            assert torch.equal(run_linear(ctx, c, wc, sw, bias, "f32"), first)


def test_linear_rows_do_not_depend_on_the_batch(ctx, native):
    """A row of exact sums has the same result alone and inside any batch."""
    c, wc, sw, bias = linear_case(600, 640, 520, 21, exact=True, padded=False)
    lin = ctx.fp8_linear(wc.view(torch.uint8).cpu().numpy(), sw.cpu().numpy(), bias.cpu().numpy())
    full = torch.empty(600, 520, device="cuda")
    lin.run(*c.args, 600, full.data_ptr(), 0, 520, stream=stream())
    for at, n in [(0, 1), (599, 1), (5, 16), (100, 40), (300, 129)]:
        y = torch.empty(n, 520, device="cuda")
        lin.run(c.buf[at].data_ptr(), c.buf.shape[1], c.sbuf.data_ptr() + 4 * at, c.lds, n, y.data_ptr(), 0, 520, stream=stream())
        assert torch.equal(y, full[at:at + n]), (at, n)
    lin.close()


# ----------------------------------------------------------------------- rope

def rope_angles(positions, f):
    """cos and sin in extended precision (64-bit mantissa)."""
    turns = np.asarray(positions, np.longdouble)[:, None] * (np.asarray(f, np.longdouble) / (2 * np.longdouble(math.pi) + np.longdouble(2.4492935982947064e-16)))
    a = (turns - np.round(turns)) * (2 * np.longdouble(math.pi) + np.longdouble(2.4492935982947064e-16))
    return torch.from_numpy(np.cos(a).astype(np.float64)).cuda(), torch.from_numpy(np.sin(a).astype(np.float64)).cuda()


def rope64(x, positions, f, m, interleaved):
    r = 2 * len(f)
    cos, sin = (t[:, None] for t in rope_angles(positions, f))
    x = x.double().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = x[..., a].clone(), x[..., b].clone()
    mag = torch.zeros_like(x)
    mag[..., a] = mag[..., b] = abs(m) * (u.abs() + v.abs())
    x[..., a], x[..., b] = m * (u * cos - v * sin), m * (v * cos + u * sin)
    return x, mag


def assert_rope(got, exp, mag, dtype, pmax):
    """cos and sin: the phase rounded to f32 (pi 2^-25 in the angle), the
    function's 2 units, the scale and three more roundings: under 2^-20 of
    |u| + |v|; the 64-bit frequency and the reference's extended product: the
    position times 2^-61."""
    bound = mag * (2.0 ** -20 + pmax * 2.0 ** -61) * (1 + H[dtype]) + torch.where(mag > 0, H[dtype] * exp.abs() + TINY[dtype], 0.0)
    bad = (got.double() - exp).abs() > bound
    assert not bad.any(), (bad.sum().item(), got[bad][:4], exp[bad][:4], bound[bad][:4])


@pytest.mark.parametrize("tokens,hq,hk,hd,rotary", [(1, 8, 1, 256, 256), (1, 1, 0, 2, 2), (3, 4, 2, 64, 32), (5, 3, 1, 80, 36),
                                                    (77, 12, 12, 64, 64), (130, 5, 2, 96, 16), (1021, 2, 1, 40, 40), (9, 70, 3, 128, 64),
                                                    (2, 1, 1, 1024, 1024), (700, 16, 4, 128, 128), (33, 3, 3, 66, 34), (64, 6, 2, 72, 48), (61, 4, 4, 33, 32), (40, 3, 3, 302, 302),
                                                    (25, 1, 2, 127, 2), (3, 9, 5, 1022, 1022), (2500, 4, 1, 30, 30)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rope(ctx, native, tokens, hq, hk, hd, rotary, interleaved, dtype):
    """q and k inside fused rows of q | k | v, to buffers of their own."""
    g = gen(tokens + hd)
    f, m = native.rope_frequencies(rotary, 10000.0, "yarn", factor=4.0, low=1.0, high=32.0, trained=4096)
    rope = ctx.rope(hd, f, interleaved, m)
    dt = DT[dtype][1]
    row = (hq + 2 * hk) * hd
    qkv = torch.randn(tokens, row, device="cuda", generator=g).to(dt)
    before = qkv.clone()
    pos = torch.randint(0, 1 << 20, (tokens,), device="cuda", generator=g)
    q, k = torch.full((tokens + 1, hq, hd), 3.0, dtype=dt, device="cuda"), torch.full((tokens + 1, max(hk, 1), hd), 3.0, dtype=dt, device="cuda")
    es = qkv.element_size()
    qv = native.rope_view(qkv.data_ptr(), row, hd, q.data_ptr(), hq * hd, hd, hq)
    kv = native.rope_view(qkv.data_ptr() + hq * hd * es, row, hd, k.data_ptr(), max(hk, 1) * hd, hd, hk)
    rope.run(qv, kv, DT[dtype][0], tokens, pos.data_ptr(), 64, stream=stream())
    assert torch.equal(qkv, before) and (q[tokens:] == 3).all() and (k[tokens:] == 3).all()
    heads = before[:, :(hq + hk) * hd].view(tokens, hq + hk, hd)
    exp, mag = rope64(heads, pos.cpu().numpy(), f, m, interleaved)
    got = torch.cat([q[:tokens], k[:tokens, :hk]], 1)
    assert_rope(got, exp, mag, dtype, 1 << 20)
    # in place, with 32-bit positions: the same bits, nothing else touched
    pos32 = pos.to(torch.int32)
    rope.run(native.rope_view(qkv.data_ptr(), row, hd, qkv.data_ptr(), row, hd, hq + hk), None, DT[dtype][0], tokens,
             pos32.data_ptr(), 32, stream=stream())
    assert torch.equal(qkv[:, :(hq + hk) * hd].view(tokens, -1, hd), got)
    assert torch.equal(qkv[:, (hq + hk) * hd:], before[:, (hq + hk) * hd:])
    rope.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rope_far_and_negative_positions(ctx, native, dtype):
    pos = torch.tensor([0, 1, -1, 131071, 1 << 24, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31), 1 << 33, -(1 << 40) + 7, (1 << 40) - 1], device="cuda")
    f, _ = native.rope_frequencies(64, 10000.0)
    f[-1] = 0.0   # a pair that does not turn
    f[-2] = -f[-2]
    x = torch.randn(len(pos), 2, 64, device="cuda", generator=gen(3)).to(DT[dtype][1])
    rope = ctx.rope(64, f)
    out = torch.empty_like(x)
    rope.run(native.rope_view(x.data_ptr(), 128, 64, out.data_ptr(), 128, 64, 2), None, DT[dtype][0], len(pos), pos.data_ptr(), stream=stream())
    exp, mag = rope64(x, pos.cpu().numpy(), f, 1.0, False)
    assert_rope(out, exp, mag, dtype, 1 << 40)
    assert torch.equal(out[0], x[0]) and torch.equal(out[:, :, 31], x[:, :, 31]) and torch.equal(out[:, :, 63], x[:, :, 63])
    rope.close()


@pytest.mark.parametrize("hd", [64, 1024])
def test_rope_runs_at_once_on_a_new_stream(ctx, native, hd):
    """Prepared and run without a pause, on a stream that does not wait for
    the legacy one, with the device busy there: the angles are complete."""
    s = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    pos = torch.arange(1, 6, device="cuda") * 1000
    x = torch.randn(5, 2, hd, device="cuda", generator=gen(hd))
    out = torch.empty_like(x)
    for k in range(12):
        f, _ = native.rope_frequencies(hd, 10000.0 + k)
        torch.cuda.synchronize()
        for _ in range(4):
            busy @ busy
        rope = ctx.rope(hd, f)
        rope.run(native.rope_view(x.data_ptr(), 2 * hd, hd, out.data_ptr(), 2 * hd, hd, 2), None, 0, 5, pos.data_ptr(), stream=s.cuda_stream)
        torch.cuda.synchronize()
        exp, mag = rope64(x, pos.cpu().numpy(), f, 1.0, False)
        assert_rope(out, exp, mag, "f32", 5000)
        rope.close()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_cosines_and_sines(ctx, native, interleaved):
    """Pairs (1, 0) come back as (cos, sin), each with a relative error: the
    phase less its nearest quarter turn rounded to f32 (2^-24 of an angle of at
    most pi/4: no more of its sine or cosine), and the function's unit in the
    last place (2^-23).  Absolute, what position and frequency leave in the
    phase: 2^20 positions * 2^-61 turns * 2 pi."""
    tokens, r = 4000, 128
    g = gen(31)
    pos = torch.randint(-(1 << 20), 1 << 20, (tokens,), device="cuda", generator=g)
    f, _ = native.rope_frequencies(r, 10000.0)
    # quarter turns, halves and what lies next to them
    f[:8] = 2 * math.pi * np.array([0.25, 0.5, 0.75, 0.125, 0.25 + 2.0 ** -40, 0.5 - 2.0 ** -40, 0.375, 2.0 ** -30])
    x = torch.zeros(tokens, r, device="cuda")
    x[:, 0::2 if interleaved else 1][:, :r // 2] = 1.0
    rope = ctx.rope(r, f, interleaved)
    out = torch.empty_like(x)
    rope.run(native.rope_view(x.data_ptr(), r, r, out.data_ptr(), r, r, 1), None, 0, tokens, pos.data_ptr(), stream=stream())
    cos, sin = rope_angles(pos.cpu().numpy(), f)
    got = (out[:, 0::2], out[:, 1::2]) if interleaved else (out[:, :r // 2], out[:, r // 2:])
    for v, exp in zip(got, (cos, sin)):
        bad = (v.double() - exp).abs() > exp.abs() * 3 * U + 2.0 ** 20 * 2.0 ** -61 * 2 * math.pi
        assert not bad.any(), (bad.sum().item(), v[bad][:4], exp[bad][:4])
    rope.close()


@pytest.mark.parametrize("hd,rotary", [(64, 64), (64, 48), (80, 20)])
def test_rope_strides(ctx, native, hd, rotary):
    """Heads-major input (tokens inside heads), odd offsets and a broadcast head (stride 0) to separate outputs."""
    f, _ = native.rope_frequencies(rotary, 10000.0)
    tokens, heads = 50, 3
    pos = torch.arange(tokens, device="cuda") * 3
    for interleaved in (False, True):
        rope = ctx.rope(hd, f, interleaved)
        buf = torch.randn(heads * tokens * (hd + 1) + 1, device="cuda", generator=gen(hd)).bfloat16()
        x = buf[1:].view(heads, tokens, hd + 1)[..., :hd].transpose(0, 1)
        out = torch.full((heads, tokens, hd + 3), 2.0, dtype=torch.bfloat16, device="cuda")
        rope.run(native.rope_view(x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), hd + 3, tokens * (hd + 3), heads), None, 1,
                 tokens, pos.data_ptr(), stream=stream())
        exp, mag = rope64(x, pos.cpu().numpy(), f, 1.0, interleaved)
        assert_rope(out.transpose(0, 1)[..., :hd], exp, mag, "bf16", 150)
        assert (out[..., hd:] == 2).all()
        rope.run(native.rope_view(x.data_ptr(), x.stride(0), 0, out.data_ptr(), hd + 3, tokens * (hd + 3), heads), None, 1, tokens,
                 pos.data_ptr(), stream=stream())
        exp, mag = rope64(x[:, :1].expand(-1, heads, -1), pos.cpu().numpy(), f, 1.0, interleaved)
        assert_rope(out.transpose(0, 1)[..., :hd], exp, mag, "bf16", 150)
        rope.close()


# -------------------------------------------------------- refusals, streams, graphs

def test_handles_refuse(ctx, native):
    L, by = native.lib(), ctypes.byref
    lin = ctx.fp8_linear(np.zeros((40, 100), np.uint8), np.ones((1, 1), np.float32))
    x = torch.zeros(4, 112, dtype=torch.uint8, device="cuda")
    s = torch.ones(1, 4, device="cuda")
    y = torch.full((4, 40), 5.0, device="cuda")

    def run(codes=x.data_ptr(), ldc=112, scales=s.data_ptr(), lds=4, rows=4, yp=y.data_ptr(), dt=0, ldy=40):
        return L.g4m_fp8_linear_run(lin._h, by(native.Fp8Rows(codes, ldc, scales, lds)), rows, yp, dt, ldy, stream())

    for bad, status in [(dict(codes=0), 1), (dict(scales=0), 1), (dict(yp=0), 1), (dict(rows=-1), 1), (dict(dt=3), 1),
                        (dict(codes=x.data_ptr() + 8), 1), (dict(ldc=104), 1), (dict(ldc=96), 2), (dict(lds=3), 2), (dict(ldy=39), 2),
                        (dict(yp=y.data_ptr() + 2), 1), (dict(scales=s.data_ptr() + 1), 1), (dict(rows=1 << 31, lds=1 << 31), 9)]:
        assert run(**bad) == status, (bad, native.last_error())
    assert run(rows=0, codes=0, yp=0) == 0
    torch.cuda.synchronize()
    assert (y == 5).all()
    with pytest.raises(native.G4MError):
        ctx.rope(64, np.full(32, np.nan))
    for hd, f, status in [(64, np.ones(33), 2), (2048, np.ones(4), 9), (64, [np.inf], 1)]:
        with pytest.raises(native.G4MError) as e:
            ctx.rope(hd, f)
        assert e.value.status == status
    rope = ctx.rope(8, [1.0, 0.5])
    xb = torch.zeros(256, device="cuda")
    pos = torch.zeros(8, dtype=torch.int64, device="cuda")

    def turn(xp=xb.data_ptr(), ts=16, hs=8, out=xb.data_ptr(), ots=16, ohs=8, heads=2, k=None, dt=0, tokens=4, pp=pos.data_ptr(), bits=64):
        return L.g4m_rope_run(rope._h, by(native.rope_view(xp, ts, hs, out, ots, ohs, heads)), k, dt, tokens, pp, bits, stream())

    other = xb.data_ptr() + 512
    for bad, status in [(dict(xp=0), 1), (dict(out=0), 1), (dict(heads=-1), 1), (dict(dt=7), 1), (dict(bits=16), 1), (dict(tokens=-1), 1),
                        (dict(pp=0), 1), (dict(pp=pos.data_ptr() + 4), 1), (dict(xp=xb.data_ptr() + 2), 1), (dict(ots=24), 1),
                        (dict(out=other, ots=12), 2), (dict(out=other, ohs=4), 2), (dict(out=other, ots=8, ohs=16), 2), (dict(out=other, ots=8, ohs=24), 2), (dict(out=other, ots=15, ohs=8), 2),
                        (dict(out=other, ohs=-8), 2), (dict(tokens=1 << 31), 9), (dict(heads=70000, out=other, ots=700000, tokens=1), 9)]:
        assert turn(**bad) == status, (bad, native.last_error())
    assert turn(tokens=0, pp=0, xp=0) == 0 and turn(heads=0, xp=0) == 0
    rope.close()
    assert turn() == 1  # a closed handle
    lin.close()
    assert run() == 1
    ctx2 = native.Context()
    kept = ctx2.fp8_linear(np.zeros((4, 4), np.uint8), np.ones((1, 1), np.float32))
    ctx2.close()
    with pytest.raises(native.G4MError):
        kept.run(*(0,) * 8)


class Layer:
    """The projections of one layer, as they chain: residual norm -> q | k | v
    -> rotary positions; residual norm -> gate | up -> gated activation ->
    down -> residual."""

    def __init__(self, ctx, native, rows, seed, d=640, heads=6, kv=2, hd=64, ff=1000):
        g = gen(seed)
        self.ctx, self.native, self.rows, self.d, self.heads, self.kv, self.hd, self.ff = ctx, native, rows, d, heads, kv, hd, ff
        self.weights = {}
        for name, o, i in (("qkv", (heads + 2 * kv) * hd, d), ("gu", 2 * ff, d), ("down", d, ff)):
            w = (40 * torch.randn(o, i, device="cuda", generator=g)).to(torch.float8_e4m3fn)
            sw = torch.exp(0.3 * torch.randn(-(-o // 128), -(-i // 128), device="cuda", generator=g)) / (40 * math.sqrt(i))
            self.weights[name] = (w, sw, ctx.fp8_linear(w.view(torch.uint8).cpu().numpy(), sw.cpu().numpy()))
        self.f, _ = native.rope_frequencies(hd, 10000.0)
        self.rope = ctx.rope(hd, self.f)
        self.y = torch.randn(rows, d, device="cuda", generator=g).bfloat16()
        self.h = torch.randn(rows, d, device="cuda", generator=g)
        self.norms = [1 + 0.1 * torch.randn(d, device="cuda", generator=g) for _ in range(4)]
        self.pos = torch.arange(rows, device="cuda") + 1000
        self.c1, self.c2, self.c3 = Codes(rows, d), Codes(rows, d), Codes(rows, ff)
        e = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        self.h1, self.h2, self.h3 = (e(rows, d, t=torch.float32) for _ in range(3))
        self.qkv, self.qk = e(rows, (heads + 2 * kv) * hd), e(rows, heads + kv, hd)
        self.gu, self.o = e(rows, 2 * ff), e(rows, d)

    def norm(self, y, h, h_out, wp, wn, codes):
        a = dict(rows=self.rows, d=self.d, dtype=1, h_dtype=0, eps=1e-6, y=y.data_ptr(), ldy=self.d, norm_post=1, w_post=wp.data_ptr(),
                 h=h.data_ptr(), ldh=self.d, h_out=h_out.data_ptr(), ldh_out=self.d, norm_pre=1, w_pre=wn.data_ptr())
        self.ctx.norm_residual(self.native.norm_args(**a, **(codes.fields if codes else {})), stream=stream())

    def linear(self, name, c, y):
        self.weights[name][2].run(*c.args, self.rows, y.data_ptr(), 1, y.shape[1], stream=stream())

    def run(self):
        n = self.norms
        self.norm(self.y, self.h, self.h1, n[0], n[1], self.c1)
        self.linear("qkv", self.c1, self.qkv)
        row = self.qkv.shape[1]
        self.rope.run(self.native.rope_view(self.qkv.data_ptr(), row, self.hd, self.qk.data_ptr(), (self.heads + self.kv) * self.hd, self.hd,
                                            self.heads + self.kv), None, 1, self.rows, self.pos.data_ptr(), stream=stream())
        self.norm(self.y, self.h1, self.h2, n[2], n[3], self.c2)
        self.linear("gu", self.c2, self.gu)
        self.ctx.fp8_quantize(self.gu.data_ptr(), 1, 2 * self.ff, self.rows, self.ff, *self.c3.args, act="gelu", stream=stream())
        self.linear("down", self.c3, self.o)
        self.norm(self.o, self.h2, self.h3, n[0], n[2], None)

    def outputs(self):
        return [t.clone() for t in (self.h1, self.c1.codes().view(torch.uint8), self.qkv, self.qk, self.h2, self.gu, self.c3.codes().view(torch.uint8), self.o, self.h3)]

    def check(self):
        """Each stage against 64 bits on the operands that it read."""
        n, rows = [w.double() for w in self.norms], self.rows
        stages = [(self.y, self.h, self.h1, n[0], n[1], self.c1), (self.y, self.h1, self.h2, n[2], n[3], self.c2), (self.o, self.h2, self.h3, n[0], n[2], None)]
        for y, h, out, wp, wn, c in stages:
            eh, en, erh, ern = norm64(y.double(), h.double(), wp, None, 1, wn, 1.0, 1.0, 1, 1, 1e-6)
            assert ((out.double() - eh).abs() <= erh * (1 + U) + U * eh.abs()).all()
            if c is not None:
                assert_codes(c, en, ern)
        for name, c, y in (("qkv", self.c1, self.qkv), ("gu", self.c2, self.gu), ("down", self.c3, self.o)):
            w, sw, _ = self.weights[name]
            exp, m = linear64(c, w, sw, None)
            bound = m * (4 * 33 * 2.0 ** -23 + (3 + (w.shape[1] + 127) // 128) * U) + H["bf16"] * exp.abs()
            assert ((y.double() - exp).abs() <= bound).all(), name
        exp, mag = rope64(self.qkv[:, :(self.heads + self.kv) * self.hd].view(rows, -1, self.hd), self.pos.cpu().numpy(), self.f, 1.0, False)
        assert_rope(self.qk, exp, mag, "bf16", 2000)
        assert_codes(self.c3, *act64(self.gu.double(), self.ff, "gelu"))


@pytest.mark.parametrize("rows", [1, 5, 40, 131, 700])
def test_layer_chain(ctx, native, rows):
    layer = Layer(ctx, native, rows, rows)
    layer.run()
    torch.cuda.synchronize()
    layer.check()
    layer.h.mul_(1.5)  # the same buffers again, with other inputs
    layer.run()
    torch.cuda.synchronize()
    layer.check()


def test_graphs_and_streams(ctx, native):
    """Two layers captured into graphs, replayed together on two streams with
    new inputs, against their eager runs; one linear called on two streams at once."""
    layers = [Layer(ctx, native, 3, 1), Layer(ctx, native, 150, 2)]
    layers[1].weights = {k: (w, sw, layers[0].weights[k][2]) for k, (w, sw, _) in layers[0].weights.items()}  # shared linears
    streams = [torch.cuda.Stream() for _ in layers]
    graphs = []
    for layer, s in zip(layers, streams):
        layer.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            layer.run()
        graphs.append(g)
    for k in range(3):
        want = []
        for layer in layers:
            layer.y.mul_(1.25)
            layer.run()
            torch.cuda.synchronize()
            want.append(layer.outputs())
        for layer in layers:
            for t in (layer.h1, layer.c1.buf, layer.qkv, layer.qk, layer.h2, layer.gu, layer.c3.buf, layer.o, layer.h3):
                t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for layer, w in zip(layers, want):
            for got, exp in zip(layer.outputs(), w):
                assert torch.equal(got, exp)
    for k in range(20):
        for layer, s in zip(layers, streams):
            with torch.cuda.stream(s):
                layer.linear("qkv", layer.c1, layer.qkv)
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        assert torch.equal(layer.qkv, w[2])


def test_offsets_past_32_bits(ctx, native):
    """Three rows each, spread over more than 4 GiB of input and of output."""
    a, b = (torch.empty(5_400_000_000, dtype=torch.uint8, device="cuda") for _ in range(2))
    d, rows, ld = 200, 3, 1_200_000_000
    x = a.view(torch.float16)[:2 * ld + d]
    pick = lambda t, stride, n: torch.stack([t[r * stride:r * stride + n] for r in range(rows)])  # noqa: E731
    g = gen(8)
    for r in range(rows):
        x[r * ld:r * ld + d] = torch.randn(d, device="cuda", generator=g).half()
    xs = pick(x, ld, d).clone()
    # quantise: codes 2.2e9 bytes apart, then the linear reads them there and writes rows 6e8 floats apart
    ldc = 2_200_000_000
    scales = torch.empty(2, rows, device="cuda")
    ctx.fp8_quantize(x.data_ptr(), 2, ld, rows, d, b.data_ptr(), ldc, scales.data_ptr(), rows, stream=stream())
    small = Codes(rows, d)
    ctx.fp8_quantize(xs.data_ptr(), 2, d, rows, d, *small.args, stream=stream())
    assert torch.equal(pick(b, ldc, d), small.buf[:rows, :d]) and torch.equal(scales, small.scales())
    _, wc, sw, _ = linear_case(rows, d, 300, 3)
    want = run_linear(ctx, small, wc, sw, None, "f32")
    lin = ctx.fp8_linear(wc.view(torch.uint8).cpu().numpy(), sw.cpu().numpy())
    y, ldy = a.view(torch.float32), 600_000_000
    lin.run(b.data_ptr(), ldc, scales.data_ptr(), rows, rows, y.data_ptr(), 0, ldy, stream=stream())
    assert torch.equal(pick(y, ldy, 300), want)
    lin.close()
    # norm and rotary positions, in place
    for r in range(rows):
        x[r * ld:r * ld + d] = xs[r]
    args = dict(rows=rows, d=d, dtype=2, h_dtype=2, eps=1e-6, norm_pre=1)
    ctx.norm_residual(native.norm_args(**args, h=x.data_ptr(), ldh=ld, n_out=b.data_ptr(), ldn=ld), stream=stream())
    n = torch.empty_like(xs)
    ctx.norm_residual(native.norm_args(**args, h=xs.data_ptr(), ldh=d, n_out=n.data_ptr(), ldn=d), stream=stream())
    assert torch.equal(pick(b.view(torch.float16), ld, d), n)
    pos = torch.tensor([5, 70000, 9], device="cuda")
    for rotary in (200, 48, 34):
        rope = ctx.rope(d, np.linspace(1, 0.01, rotary // 2))
        for t, stride in ((x, ld), (xs.view(-1), d)):
            rope.run(native.rope_view(t.data_ptr(), stride, d, t.data_ptr(), stride, d, 1), None, 2, rows, pos.data_ptr(), stream=stream())
        assert torch.equal(pick(x, ld, d), xs)
        rope.close()


def test_two_host_threads(ctx, native):
    """One linear, called from two threads on streams of their own."""
    import threading
    layers = [Layer(ctx, native, 20, 5), Layer(ctx, native, 300, 6)]
    layers[1].weights = layers[0].weights
    want = []
    for layer in layers:
        layer.run()
        torch.cuda.synchronize()
        want.append(layer.outputs())
    failed = []

    def work(layer, exp):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(50):
                    layer.run()
                s.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(layer.outputs(), exp)):
                    failed.append("outputs differ")
        except Exception as e:  # a thread's exception would be lost
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=a) for a in zip(layers, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("rows", [3, 700])
def test_an_expired_wait_is_reported(ctx, native, rows):
    """A wait that ran out in an earlier call: the linear's own sums stand all
    the same, and the next call that waits says so, once."""
    c, wc, sw, bias = linear_case(rows, 2048, 300, 4, exact=True)
    exp = linear64(c, wc, sw, bias)[0]
    ctx.synchronize(stream())
    assert native.lib().g4m_selftest_wait_timeout(ctx.h, 0, -200_000) == 0
    torch.cuda.synchronize()
    assert torch.equal(run_linear(ctx, c, wc, sw, bias, "f32").double(), exp)
    with pytest.raises(native.G4MError) as e:
        ctx.synchronize(stream())
    assert e.value.status == 5 and "kernel error code 1" in str(e.value)
    ctx.synchronize(stream())
    assert torch.equal(run_linear(ctx, c, wc, sw, bias, "f32").double(), exp)
    ctx.synchronize()


PER_LAYER = {"norm_residual": 3, "fp8_gemm": 3, "rope": 1, "fp8_quantize": 1}


def test_profile_leaves_captures_alone(ctx, native):
    """With per-launch timing on, a capture still works, and only the eager
    launches are timed."""
    layer = Layer(ctx, native, 5, 8)
    layer.run()
    torch.cuda.synchronize()
    ctx.profile_begin()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer.run()
    for _ in range(2):
        layer.run()
    g.replay()
    got = ctx.profile_end()
    assert {k: v[0] for k, v in got.items()} == {k: 2 * n for k, n in PER_LAYER.items()}
    assert all(0 < v[1] < 1e3 for v in got.values())
    torch.cuda.synchronize()
    layer.check()
    ctx.profile_begin()
    assert ctx.profile_end() == {}


def test_profile_counts_every_thread(ctx, native):
    """Launches of several threads are timed at once; timing that another
    thread ends and begins meanwhile loses some and breaks nothing."""
    import threading
    layers = [Layer(ctx, native, 3, 10 + k) for k in range(4)]
    for layer in layers:
        layer.run()
    torch.cuda.synchronize()
    failed = []

    def work(layer):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    layer.run()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # a thread's exception would be lost
            failed.append(repr(e))

    for switch in (False, True):
        ctx.profile_begin()
        threads = [threading.Thread(target=work, args=(layer,)) for layer in layers]
        for t in threads:
            t.start()
        while switch and any(t.is_alive() for t in threads):
            ctx.profile_end()
            ctx.profile_begin()
        for t in threads:
            t.join()
        got = {k: v[0] for k, v in ctx.profile_end().items()}
        assert not failed, failed
        if not switch:
            assert got == {k: 4 * 60 * n for k, n in PER_LAYER.items()}
    for layer in layers:
        layer.check()


def test_beside_a_tower_call(native, syn, tmp_path):
    """Layers on two streams while another thread embeds images with the same
    context: all give what they give alone."""
    import threading
    path = str(tmp_path / "v.safetensors")
    syn.write_safetensors(path, syn.vision_weights(0, layers=2))
    c = native.Context()
    try:
        c.load_weights(path)
        pix = [syn.image_pixels(k, 768, 768) for k in range(3)]
        layers = [Layer(c, native, 24, 40), Layer(c, native, 2000, 41)]
        outs, _ = c.vision_embed(pix, 256, 2)
        want = []
        for layer in layers:
            layer.run()
            torch.cuda.synchronize()
            want.append(layer.outputs())
        got, failed = [], []

        def tower():
            try:
                for _ in range(4):
                    got.append(c.vision_embed(pix, 256, 2)[0])
            except Exception as e:  # a thread's exception would be lost
                failed.append(repr(e))

        t = threading.Thread(target=tower)
        t.start()
        streams = [torch.cuda.Stream() for _ in layers]
        for _ in range(40):
            for layer, s in zip(layers, streams):
                with torch.cuda.stream(s):
                    layer.run()
        t.join()
        torch.cuda.synchronize()
        assert not failed, failed
        for layer, exp in zip(layers, want):
            assert all(torch.equal(p, q) for p, q in zip(layer.outputs(), exp))
        for again in got:
            assert all(np.array_equal(p, q) for p, q in zip(again, outs))
        c.synchronize()
    finally:
        c.close()


def test_default_stream_is_the_legacy_one(ctx):
    """Stream 0 orders with torch's default stream."""
    x = torch.zeros(64, 4096, device="cuda")
    c = Codes(64, 4096)
    for k in range(4):
        x.fill_(k + 1.0)
        ctx.fp8_quantize(x.data_ptr(), 0, 4096, 64, 4096, *c.args)
        assert (c.values() - (k + 1)).abs().max() <= (k + 1) * 2.0 ** -22


def test_current_device_is_kept(ctx, native):
    before = torch.cuda.current_device()
    layer = Layer(ctx, native, 2, 4)
    layer.run()
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before


def test_first_call_of_a_process_can_be_captured():
    """Kernels are loaded lazily; a capture may be the first to need them."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import sys; sys.path[:0] = [%r, %r]
import conftest, importlib, torch
import test_gpu_fp8_ops as T
native = importlib.import_module(conftest.PKG + "._native")
ctx = native.Context()
layer = T.Layer(ctx, native, 9, 3)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    layer.run()
g.replay()
torch.cuda.synchronize()
layer.check()
print("captured")
""" % (here, os.path.dirname(here))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
