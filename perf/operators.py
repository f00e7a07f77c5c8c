"""The 8-bit float operators of the g4m library, as cases to measure.

Four operators that a transformer layer chains around its projections:
  norm      RMSNorm after a block, gate and scale on its branch, residual add, RMSNorm before the next block
  quantize  rows to e4m3 codes with an f32 scale for each 128 columns, optionally after a gated activation
  linear    codes x e4m3 weights with an f32 scale for each 128 x 128 block, products summed in 32 bits
  rope      rotary positions on query and key heads

`run` computes them with elementary torch operations, or, where `own` is
true, through the library's public entry points on device pointers.
"""
import math

import numpy as np
import torch

own = False

PACKAGE = "gemma-4-webgpu-kernels-multimodal_b200"
BLOCK = 128               # columns (and weight rows) that share one scale
E4M3_MAX = 448.0          # largest finite e4m3 value
AMAX_FLOOR = 2.0 ** -96   # least block maximum: an all-zero block keeps a normal scale
EPS = 1e-6                # the towers' RMSNorm epsilon
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------- cases

def listed():
    return [
        # decode step: one token's residual update into the next 8-bit projection (embedding width 1536)
        {"name": "norm token", "op": "norm", "rows": 1, "d": 1536, "dtype": "bf16", "res": "bf16", "gate": 0, "out": "codes"},
        # a batch of clips with odd widths, one gate row for each clip
        {"name": "norm gated odd", "op": "norm", "rows": 1003, "d": 1155, "dtype": "f16", "res": "f16", "gate": 59, "out": "both"},
        # long prompt with the residual stream in f32, gate rows for blocks of 1024 tokens
        {"name": "norm long", "op": "norm", "rows": 16384, "d": 4096, "dtype": "bf16", "res": "f32", "gate": 1024, "out": "codes"},
        # decode batch of seven through a gated MLP
        {"name": "quantize few", "op": "quantize", "rows": 7, "d": 6144, "dtype": "bf16", "act": "silu"},
        # the gated MLP of a long prompt
        {"name": "quantize long", "op": "quantize", "rows": 8192, "d": 6144, "dtype": "bf16", "act": "gelu"},
        # decode step through the gate | up projection of an MLP on 1536-wide embeddings
        {"name": "linear token", "op": "linear", "rows": 1, "in": 1536, "out": 12288, "dtype": "bf16", "bias": False},
        # a decode batch, with input and output widths that end inside a scale block
        {"name": "linear few odd", "op": "linear", "rows": 37, "in": 4000, "out": 5000, "dtype": "f16", "bias": True},
        # the q | k | v projection of one 768 x 768 image (2304 patches)
        {"name": "linear image", "op": "linear", "rows": 2304, "in": 768, "out": 2304, "dtype": "f32", "bias": True},
        # prompt processing
        {"name": "linear long", "op": "linear", "rows": 8192, "in": 4096, "out": 8192, "dtype": "bf16", "bias": False},
        # decode step at a far position: 8 query heads, 1 key head, whole head, two halves
        {"name": "rope token", "op": "rope", "tokens": 1, "heads": 8, "kv": 1, "head_dim": 256, "rotary": 256, "layout": "half", "scaling": "none", "dtype": "bf16"},
        # odd token count, part of the head, frequencies stretched by bands, f32
        {"name": "rope odd part", "op": "rope", "tokens": 1021, "heads": 12, "kv": 3, "head_dim": 80, "rotary": 36, "layout": "half", "scaling": "banded", "dtype": "f32"},
        # long prompt, adjacent pairs, interpolated positions with an attention factor
        {"name": "rope long", "op": "rope", "tokens": 16384, "heads": 32, "kv": 8, "head_dim": 128, "rotary": 128, "layout": "interleaved", "scaling": "yarn", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "rope"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        d = _log(rng, 96, 8192)
        rows = _log(rng, 1, min(16384, 16384 * 4096 // (2 * d)))
        if rng.random() < 0.5:
            d = (d + 63) // 64 * 64
        gate = rng.choice([0, _log(rng, 1, rows)])
        return {"op": op, "rows": rows, "d": d, "dtype": dtype, "res": rng.choice([dtype, "f32"]), "gate": gate,
                "out": rng.choice(["codes", "rows", "both"])}
    if op == "quantize":
        d = _log(rng, 96, 12288)
        if rng.random() < 0.5:
            d = (d + 63) // 64 * 64
        rows = _log(rng, 1, min(16384, 8192 * 6144 // (2 * d)))
        return {"op": op, "rows": rows, "d": d, "dtype": dtype, "act": rng.choice(["none", "silu", "gelu"])}
    if op == "linear":
        i, o = _log(rng, 128, 8192), _log(rng, 128, 12288)
        if rng.random() < 0.6:
            i, o = (i + 127) // 128 * 128, (o + 127) // 128 * 128
        rows = _log(rng, 1, max(1, min(8192, 8192 * 4096 * 8192 // (2 * i * o))))
        return {"op": op, "rows": rows, "in": i, "out": o, "dtype": dtype, "bias": rng.random() < 0.5}
    hd = 2 * _log(rng, 32, 128)
    if rng.random() < 0.6:
        hd = (hd + 15) // 16 * 16
    rotary = hd if rng.random() < 0.5 else 2 * _log(rng, 8, hd // 2)
    kv = _log(rng, 1, 8)
    heads = kv * rng.choice([1, 2, 3, 4])
    tokens = _log(rng, 1, min(16384, 16384 * 40 * 128 // (2 * (heads + kv) * hd)))
    return {"op": op, "tokens": tokens, "heads": heads, "kv": kv, "head_dim": hd, "rotary": rotary,
            "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "banded", "yarn"]), "dtype": dtype}


def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    c = case
    if c["op"] == "norm":
        n, y, h = c["rows"] * c["d"], _size(c["dtype"]), _size(c["res"])
        out = (y if c["out"] != "codes" else 0) + (1 + 4 / BLOCK if c["out"] != "rows" else 0)
        gates = -(-c["rows"] // c["gate"]) * c["d"] * y if c["gate"] else 0
        return {"bytes": n * (y + 2 * h + out) + gates + 8 * c["d"], "flops": 10 * n}
    if c["op"] == "quantize":
        n = c["rows"] * c["d"]
        return {"bytes": n * (_size(c["dtype"]) * (1 if c["act"] == "none" else 2) + 1 + 4 / BLOCK), "flops": 10 * n}
    if c["op"] == "linear":
        kb, nb = -(-c["in"] // BLOCK), -(-c["out"] // BLOCK)
        return {"bytes": c["rows"] * (c["in"] + 4 * kb) + c["in"] * c["out"] + 4 * kb * nb + c["rows"] * c["out"] * _size(c["dtype"])
                + (4 * c["out"] if c["bias"] else 0), "flops": 2 * c["rows"] * c["in"] * c["out"]}
    n = c["tokens"] * (c["heads"] + c["kv"])
    return {"bytes": 2 * n * c["head_dim"] * _size(c["dtype"]) + 8 * c["tokens"], "flops": 3 * n * c["rotary"]}


# -------------------------------------------------------------------- inputs

def _pad16(d):
    return (d + 15) // 16 * 16


def _activations(g, rows, d):
    """Rows as a residual stream has them: unit noise, some channels far louder."""
    x = torch.randn(rows, d, device="cuda", generator=g)
    loud = torch.rand(d, device="cuda", generator=g) < 0.02
    return x * torch.where(loud, 20.0, 1.0) * torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))


def _to_codes(x, s):
    return (x / s).to(torch.float8_e4m3fn)


def _blocks(x):
    """[rows, d] -> [rows, blocks, 128], padded with zeros."""
    rows, d = x.shape
    return torch.nn.functional.pad(x, (0, -d % BLOCK)).view(rows, -1, BLOCK)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = _INPUTS[case["op"]](case, g)
    s["case"] = case
    if own:
        _HANDLES[case["op"]](case, s)
    return s


def _norm_inputs(c, g):
    dt, rt = DTYPES[c["dtype"]], DTYPES[c["res"]]
    s = {"y": (0.5 * _activations(g, c["rows"], c["d"])).to(dt), "h": (2 * _activations(g, c["rows"], c["d"])).to(rt)}
    for w in ("w_post", "w_pre"):
        s[w] = 1 + 0.2 * torch.randn(c["d"], device="cuda", generator=g)
    s["gate"] = None
    if c["gate"]:
        s["gate"] = torch.tanh(torch.randn(-(-c["rows"] // c["gate"]), c["d"], device="cuda", generator=g)).to(dt)
    # the branch and layer factors of a half-step residual with a layer scalar
    s["branch_scale"], s["res_scale"] = 0.5, 0.875
    return s


def _quantize_inputs(c, g):
    return {"x": _activations(g, c["rows"], c["d"] * (1 if c["act"] == "none" else 2)).to(DTYPES[c["dtype"]])}


def _linear_inputs(c, g):
    rows, i, o = c["rows"], c["in"], c["out"]
    x = _blocks(_activations(g, rows, i))
    xs = x.abs().amax(2).clamp_min(AMAX_FLOOR) / E4M3_MAX
    codes = torch.zeros(rows, _pad16(i), dtype=torch.uint8, device="cuda")
    codes[:, :i] = _to_codes(x, xs[:, :, None]).view(rows, -1)[:, :i].view(torch.uint8)
    w = torch.randn(o, i, device="cuda", generator=g) / math.sqrt(i)
    kb, nb = -(-i // BLOCK), -(-o // BLOCK)
    w = torch.nn.functional.pad(w, (0, kb * BLOCK - i, 0, nb * BLOCK - o)).view(nb, BLOCK, kb, BLOCK)
    w = w * torch.exp(0.5 * torch.randn(nb, 1, kb, 1, device="cuda", generator=g))
    ws = w.abs().amax((1, 3)).clamp_min(AMAX_FLOOR) / E4M3_MAX
    wc = _to_codes(w, ws[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:o, :i].contiguous()
    return {"codes": codes, "scales": xs.t().contiguous(), "w": wc, "w_scales": ws.contiguous(),
            "bias": torch.randn(o, device="cuda", generator=g) if c["bias"] else None}


def _rope_inputs(c, g):
    dt = DTYPES[c["dtype"]]
    # the heads as the projection leaves them: rows of q | k | v
    qkv = torch.randn(c["tokens"], (c["heads"] + 2 * c["kv"]) * c["head_dim"], device="cuda", generator=g).to(dt)
    first = torch.randint(0, 120000, (1,), device="cuda", generator=g)
    return {"qkv": qkv, "positions": first + torch.arange(c["tokens"], device="cuda")}


_INPUTS = {"norm": _norm_inputs, "quantize": _quantize_inputs, "linear": _linear_inputs, "rope": _rope_inputs}

# rotary settings of the cases: base, positions seen in training, and how they are stretched
THETA, TRAINED = 10000.0, 8192
LINEAR_FACTOR = 4.0
BANDED = {"factor": 8.0, "low": 1.0, "high": 4.0}
YARN = {"factor": 16.0, "fast": 32.0, "slow": 1.0}


# ---------------------------------------------------------------- plain form

def _rms(x):
    return torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)


def _quantized(v):
    """f32 rows -> e4m3 codes [rows, d] and scales [blocks, rows]."""
    b = _blocks(v)
    s = b.abs().amax(2).clamp_min(AMAX_FLOOR) / E4M3_MAX
    return _to_codes(b, s[:, :, None]).view(v.shape[0], -1)[:, :v.shape[1]], s.t()


def _norm_plain(c, s):
    y, h = s["y"].float(), s["h"].float()
    b = y * _rms(y) * s["w_post"]
    if s["gate"] is not None:
        b = b * s["gate"].float().repeat_interleave(c["gate"], 0)[:c["rows"]]
    h = s["res_scale"] * (h + s["branch_scale"] * b)
    n = h * _rms(h) * s["w_pre"]
    out = {"h": h.to(DTYPES[c["res"]])}
    if c["out"] != "codes":
        out["n"] = n.to(DTYPES[c["dtype"]])
    if c["out"] != "rows":
        out["codes"], out["scales"] = _quantized(n)
    return out


def _quantize_plain(c, s):
    x = s["x"].float()
    if c["act"] != "none":
        a, up = x[:, :c["d"]], x[:, c["d"]:]
        # gelu in its tanh form is a * sigmoid(2 u)
        u = a if c["act"] == "silu" else 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a)
        x = a * (1 / (1 + torch.exp(-u))) * up
    codes, scales = _quantized(x)
    return {"codes": codes, "scales": scales}


def _linear_plain(c, s):
    x = _blocks(s["codes"][:, :c["in"]].view(torch.float8_e4m3fn).float()) * s["scales"].t()[:, :, None]
    ws = s["w_scales"].repeat_interleave(BLOCK, 0)[:c["out"]]
    w = _blocks(s["w"].float()) * ws[:, :, None]
    y = x.view(c["rows"], -1) @ w.view(c["out"], -1).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[c["dtype"]])


def _frequencies(c):
    """Angle per position of each pair (64 bits) and the factor on cos and sin."""
    r = c["rotary"]
    f = THETA ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if c["scaling"] == "linear":
        return f / LINEAR_FACTOR, 1.0
    if c["scaling"] == "banded":
        # whole turns within the trained length: few are interpolated, many are kept, between them a blend
        turns = TRAINED * f / (2 * math.pi)
        keep = ((turns - BANDED["low"]) / (BANDED["high"] - BANDED["low"])).clamp(0, 1)
        return f * (keep + (1 - keep) / BANDED["factor"]), 1.0
    if c["scaling"] == "yarn":
        # pair index at which a given number of turns falls within the trained length
        at = [r * math.log(TRAINED / (2 * math.pi * b)) / (2 * math.log(THETA)) for b in (YARN["fast"], YARN["slow"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64, device="cuda") - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * ((1 - ramp) + ramp / YARN["factor"]), 0.1 * math.log(YARN["factor"]) + 1
    return f, 1.0


def _rope_plain(c, s):
    f, m = _frequencies(c)
    t, r, hd = c["tokens"], c["rotary"], c["head_dim"]
    a = s["positions"].double()[:, None] * f
    cos, sin = (torch.cos(a) * m).float()[:, None], (torch.sin(a) * m).float()[:, None]
    x = s["qkv"][:, :(c["heads"] + c["kv"]) * hd].reshape(t, -1, hd).float()
    if c["layout"] == "half":
        u, v = x[:, :, :r // 2], x[:, :, r // 2:r]
        x = torch.cat([u * cos - v * sin, v * cos + u * sin, x[:, :, r:]], 2)
    else:
        u, v = x[:, :, 0:r:2], x[:, :, 1:r:2]
        x = torch.cat([torch.stack([u * cos - v * sin, v * cos + u * sin], 3).flatten(2), x[:, :, r:]], 2)
    x = x.to(DTYPES[c["dtype"]])
    return {"q": x[:, :c["heads"]], "k": x[:, c["heads"]:]}


_PLAIN = {"norm": _norm_plain, "quantize": _quantize_plain, "linear": _linear_plain, "rope": _rope_plain}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["op"]](c, state)


# ------------------------------------------------------- the library's calls

_library = {}


def _lib():
    if not _library:
        import importlib
        _library["native"] = importlib.import_module(PACKAGE + "._native")
        _library["ctx"] = _library["native"].Context([0])
        _library["dtypes"] = {k: getattr(_library["native"], k.upper()) for k in DTYPES}
    return _library["native"], _library["ctx"], _library["dtypes"]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _fp8_out(rows, d):
    """Buffers of an 8-bit operand: padded rows of codes, scales [blocks, rows]."""
    return (torch.zeros(rows, _pad16(d), dtype=torch.uint8, device="cuda"),
            torch.empty(-(-d // BLOCK), rows, dtype=torch.float32, device="cuda"))


def _norm_handle(c, s):
    native, ctx, dts = _lib()
    rows, d = c["rows"], c["d"]
    s["h_out"] = torch.empty_like(s["h"])
    s["n_out"] = torch.empty_like(s["y"]) if c["out"] != "codes" else None
    s["codes_out"], s["scales_out"] = _fp8_out(rows, d) if c["out"] != "rows" else (None, None)
    s["args"] = native.norm_args(
        rows=rows, d=d, dtype=dts[c["dtype"]], h_dtype=dts[c["res"]], eps=EPS, y=s["y"].data_ptr(), ldy=d, norm_post=1,
        w_post=s["w_post"].data_ptr(), gate=s["gate"].data_ptr() if c["gate"] else 0, ldg=d, rows_per_gate=max(c["gate"], 1),
        branch_scale=s["branch_scale"], h=s["h"].data_ptr(), ldh=d, res_scale=s["res_scale"], h_out=s["h_out"].data_ptr(),
        ldh_out=d, w_pre=s["w_pre"].data_ptr(), norm_pre=1, n_out=s["n_out"].data_ptr() if s["n_out"] is not None else 0, ldn=d,
        codes=s["codes_out"].data_ptr() if s["codes_out"] is not None else 0, ldc=_pad16(d),
        scales=s["scales_out"].data_ptr() if s["scales_out"] is not None else 0, lds=rows)
    s["out"] = {"h": s["h_out"]}
    if s["n_out"] is not None:
        s["out"]["n"] = s["n_out"]
    if s["codes_out"] is not None:
        s["out"]["codes"], s["out"]["scales"] = s["codes_out"][:, :d].view(torch.float8_e4m3fn), s["scales_out"]


def _norm_own(c, s):
    _library["ctx"].norm_residual(s["args"], stream=_stream())
    return s["out"]


def _quantize_handle(c, s):
    _lib()
    s["codes_out"], s["scales_out"] = _fp8_out(c["rows"], c["d"])
    s["out"] = {"codes": s["codes_out"][:, :c["d"]].view(torch.float8_e4m3fn), "scales": s["scales_out"]}


def _quantize_own(c, s):
    _library["ctx"].fp8_quantize(s["x"].data_ptr(), _library["dtypes"][c["dtype"]], s["x"].shape[1], c["rows"], c["d"],
                                 s["codes_out"].data_ptr(), s["codes_out"].shape[1], s["scales_out"].data_ptr(), c["rows"],
                                 act=c["act"], stream=_stream())
    return s["out"]


def _linear_handle(c, s):
    native, ctx, _ = _lib()
    s["lin"] = ctx.fp8_linear(s["w"].view(torch.uint8).cpu().numpy(), s["w_scales"].cpu().numpy(),
                              None if s["bias"] is None else s["bias"].cpu().numpy())
    s["y"] = torch.empty(c["rows"], c["out"], dtype=DTYPES[c["dtype"]], device="cuda")


def _linear_own(c, s):
    s["lin"].run(s["codes"].data_ptr(), s["codes"].shape[1], s["scales"].data_ptr(), c["rows"], c["rows"], s["y"].data_ptr(),
                 _library["dtypes"][c["dtype"]], c["out"], stream=_stream())
    return s["y"]


def _rope_handle(c, s):
    native, ctx, _ = _lib()
    kw = {"none": {}, "linear": {"factor": LINEAR_FACTOR},
          "banded": {"factor": BANDED["factor"], "low": BANDED["low"], "high": BANDED["high"], "trained": TRAINED},
          "yarn": {"factor": YARN["factor"], "low": YARN["slow"], "high": YARN["fast"], "trained": TRAINED}}[c["scaling"]]
    f, m = native.rope_frequencies(c["rotary"], THETA, scaling=c["scaling"], **kw)
    s["rope"] = ctx.rope(c["head_dim"], f, interleaved=c["layout"] == "interleaved", attention_scale=m)
    hd, row = c["head_dim"], s["qkv"].shape[1]
    s["q"], s["k"] = (torch.empty(c["tokens"], h, hd, dtype=DTYPES[c["dtype"]], device="cuda") for h in (c["heads"], c["kv"]))
    at = s["qkv"].data_ptr()
    s["q_view"] = native.rope_view(at, row, hd, s["q"].data_ptr(), c["heads"] * hd, hd, c["heads"])
    s["k_view"] = native.rope_view(at + c["heads"] * hd * s["qkv"].element_size(), row, hd, s["k"].data_ptr(), c["kv"] * hd, hd, c["kv"])
    s["out"] = {"q": s["q"], "k": s["k"]}


def _rope_own(c, s):
    s["rope"].run(s["q_view"], s["k_view"], _library["dtypes"][c["dtype"]], c["tokens"], s["positions"].data_ptr(), pos_bits=64,
                  stream=_stream())
    return s["out"]


_HANDLES = {"norm": _norm_handle, "quantize": _quantize_handle, "linear": _linear_handle, "rope": _rope_handle}
_OWN = {"norm": _norm_own, "quantize": _quantize_own, "linear": _linear_own, "rope": _rope_own}


# ----------------------------------------------------------------- in 64 bits

def _e4m3_nearest(q):
    """The e4m3 value nearest to q, ties to the even code: 3 mantissa bits, least normal 2^-6, steps of 2^-9 below it."""
    _, e = torch.frexp(q)                               # q = m * 2^e, m in [0.5, 1)
    step = torch.ldexp(torch.ones_like(q), (e - 4).clamp_min(-9))
    return (torch.round(q / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _quantized64(v):
    rows, d = v.shape
    codes, scales = [], []
    for at in range(0, d, BLOCK):
        part = v[:, at:at + BLOCK]
        sc = torch.clamp(part.abs().max(1, keepdim=True).values, min=AMAX_FLOOR) / E4M3_MAX
        codes.append(_e4m3_nearest(part / sc))
        scales.append(sc[:, 0])
    return torch.cat(codes, 1), torch.stack(scales)


def _norm64(c, s):
    y, h = s["y"].double(), s["h"].double()
    branch = y / torch.sqrt((y * y).sum(1, keepdim=True) / c["d"] + EPS) * s["w_post"].double()
    if c["gate"]:
        branch = branch * s["gate"].double()[torch.arange(c["rows"], device="cuda") // c["gate"]]
    h = (h + branch * s["branch_scale"]) * s["res_scale"]
    n = h / torch.sqrt((h * h).sum(1, keepdim=True) / c["d"] + EPS) * s["w_pre"].double()
    out = {"h": h}
    if c["out"] in ("rows", "both"):
        out["n"] = n
    if c["out"] in ("codes", "both"):
        out["codes"], out["scales"] = _quantized64(n)
    return out


def _quantize64(c, s):
    x = s["x"].double()
    if c["act"] == "silu":
        gate, up = x.split(c["d"], 1)
        x = gate / (1 + torch.exp(-gate)) * up
    elif c["act"] == "gelu":
        gate, up = x.split(c["d"], 1)
        x = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
    codes, scales = _quantized64(x)
    return {"codes": codes, "scales": scales}


def _linear64(c, s):
    y = torch.zeros(c["rows"], c["out"], dtype=torch.float64, device="cuda")
    per_out = torch.arange(c["out"], device="cuda") // BLOCK
    for b, at in enumerate(range(0, c["in"], BLOCK)):
        x = s["codes"][:, at:min(at + BLOCK, c["in"])].view(torch.float8_e4m3fn).double()
        y += (x @ s["w"][:, at:at + BLOCK].double().t()) * s["scales"][b].double()[:, None] * s["w_scales"][per_out, b].double()
    return y if s["bias"] is None else y + s["bias"].double()


def _rope64(c, s):
    r, hd = c["rotary"], c["head_dim"]
    j = np.arange(r // 2, dtype=np.float64)
    f, m = THETA ** (-2.0 * j / r), 1.0
    if c["scaling"] == "linear":
        f = f / LINEAR_FACTOR
    elif c["scaling"] == "banded":
        wave = 2 * np.pi / f
        blend = (TRAINED / wave - BANDED["low"]) / (BANDED["high"] - BANDED["low"])
        mixed = (1 - blend) * f / BANDED["factor"] + blend * f
        f = np.where(wave > TRAINED / BANDED["low"], f / BANDED["factor"], np.where(wave < TRAINED / BANDED["high"], f, mixed))
    elif c["scaling"] == "yarn":
        where = lambda turns: r * np.log(TRAINED / (turns * 2 * np.pi)) / (2 * np.log(THETA))  # noqa: E731
        lo, hi = max(np.floor(where(YARN["fast"])), 0), min(np.ceil(where(YARN["slow"])), r - 1)
        inter = np.clip((j - lo) / max(hi - lo, 0.001), 0, 1)
        f, m = f / YARN["factor"] * inter + f * (1 - inter), 1 + 0.1 * np.log(YARN["factor"])
    turn = torch.polar(torch.full((c["tokens"], r // 2), float(m), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * torch.from_numpy(f).cuda())
    x = s["qkv"].view(c["tokens"], -1, hd)[:, :c["heads"] + c["kv"]].double().clone()
    a, b = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
    x[..., a], x[..., b] = z.real, z.imag
    return {"q": x[:, :c["heads"]], "k": x[:, c["heads"]:]}


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return {"norm": _norm64, "quantize": _quantize64, "linear": _linear64, "rope": _rope64}[case["op"]](
        case, _INPUTS[case["op"]](case, g))
