"""The microscaled formats as cases that can be timed and checked: MXFP4 weights (4 bits), MXFP8 rows of activations
(8 bits), and what a layer does with them.

Both formats cut a row into blocks of 32. A block has one scale, a power of two held as its exponent plus 127 in a byte,
and an element each of e2m1 (two to a byte, the even one in the low nibble) or e4m3: the exponent is that of the largest
magnitude less the largest exponent of the element's type (2 or 8), elements are rounded to nearest, ties to even, and
magnitudes beyond the type's largest become that.

`own` false: the operators in elementary torch operations. `own` true: the library's calls.
"""
import functools
import importlib
import math

import torch

own = False
BLOCK = 32
GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)         # magnitudes of e2m1
EPS = 1e-6
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_lib = None


def listed():
    return [
        # A model file's rows on their way to MXFP4, with the values that they then stand for: a small model's gate
        # projection as f16, and a large one's as bf16, the row count odd.
        dict(name="load-f16-4864x896", kind="load", type="f16", rows=4864, k=896),
        dict(name="load-bf16-18957x3584", kind="load", type="bf16", rows=18957, k=3584),
        # The attention's output of a prompt chunk on its way into the output projection.
        dict(name="rows-512x3584", kind="rows", rows=512, k=3584),
        # The norm ahead of a projection: one token of a small model, where the launch counts; a ragged chunk whose
        # sublayer output comes as the parts of a product that was split over K.
        dict(name="norm-1x896", kind="norm", rows=1, n=896, parts=1),
        dict(name="norm-301x3584-parts", kind="norm", rows=301, n=3584, parts=3),
        # One token: a small model's down projection, and a large one's head, the longest read of a decode step.
        dict(name="token-896x4864", kind="token", n=896, k=4864),
        dict(name="token-152064x3584", kind="token", n=152064, k=3584),
        # Few rows (tokens of several drafts), an ordinary question, a full prompt chunk through the down projection.
        dict(name="product-7x4608x3584", kind="product", m=7, n=4608, k=3584),
        dict(name="product-77x896x4864", kind="product", m=77, n=896, k=4864),
        dict(name="product-512x3584x18944", kind="product", m=512, n=3584, k=18944),
        # Gate and up projection with the gated activation: a ragged chunk, and a document read in large chunks.
        dict(name="gated-301x4864x896", kind="gated", m=301, ff=4864, k=896),
        dict(name="gated-2048x18944x3584", kind="gated", m=2048, ff=18944, k=3584),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _blocks(rng, lo, hi):
    """A multiple of the block, spread like _log."""
    return BLOCK * _log(rng, lo // BLOCK, hi // BLOCK)


def draw(rng):
    kind = rng.choice(["load", "rows", "norm", "token", "product", "product", "gated"])
    if kind == "load":
        k = _blocks(rng, 32, 18944)
        return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), rows=_log(rng, 1, min(38000, 18957 * 3584 // k)), k=k)
    if kind == "rows":
        return dict(kind=kind, rows=_log(rng, 1, 2048), k=_blocks(rng, 32, 18944))
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 2048), n=_blocks(rng, 64, 8192), parts=rng.randint(0, 7))
    if kind == "token":
        k = _blocks(rng, 32, 18944)
        return dict(kind=kind, n=_log(rng, 1, min(152064, 152064 * 3584 // k)), k=k)
    m, k = _log(rng, 1, 2048), _blocks(rng, 32, 18944)
    most = min(37888, 2048 * 37888 * 3584 // (m * k))          # no more work than the largest listed case
    if kind == "product":
        return dict(kind=kind, m=m, n=_log(rng, 1, most), k=k)
    return dict(kind=kind, m=m, ff=_blocks(rng, 32, most // 2), k=k)


# ---- what a program holds before the call -----------------------------------------------------------
class _Buffer:
    """Device memory as the library's calls take it (ptr, nbytes); it lives as long as its tensor."""

    def __init__(self, t):
        self.t = t.contiguous()
        self.ptr, self.nbytes = self.t.data_ptr(), self.t.numel() * self.t.element_size()


def _empty(*shape, dtype=torch.float32):
    return _Buffer(torch.empty(shape, dtype=dtype, device="cuda"))


def _codes8(rows, k):
    """Room for MXFP8 rows: elements and scales."""
    return _empty(rows, k, dtype=torch.uint8), _empty(rows, k // BLOCK, dtype=torch.uint8)


def _activations(rows, k, g):
    """Rows as they leave a layer: most columns of order one, some of them an order larger."""
    gain = 1.0 + 12.0 * (torch.rand(k, generator=g, device="cuda") < 0.01)
    return torch.randn(rows, k, generator=g, device="cuda") * gain


def _weight(n, k, g):
    """An MXFP4 weight: packed codes and scales."""
    codes, scales = _to_mxfp4(torch.randn(n, k, generator=g, device="cuda").mul_(0.02))
    return _Buffer(_packed(codes)), _Buffer(scales)


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if kind == "load":
        s["src"] = _Buffer((torch.randn(c["rows"], c["k"], generator=g, device="cuda") * 0.02).to(_TYPES[c["type"]]))
        s["codes"], s["scales"] = _empty(c["rows"], c["k"] // 2, dtype=torch.uint8), _empty(c["rows"], c["k"] // BLOCK, dtype=torch.uint8)
        s["values"] = _empty(c["rows"], c["k"], dtype=torch.bfloat16)
    elif kind == "rows":
        s["src"] = _Buffer(_activations(c["rows"], c["k"], g))
        s["codes"], s["scales"] = _codes8(c["rows"], c["k"])
    elif kind == "norm":
        n, rows = c["n"], c["rows"]
        s["x"] = _Buffer(_activations(rows, n, g))
        s["parts"] = _Buffer(torch.randn(max(c["parts"], 1), rows, n, generator=g, device="cuda") * 0.5)
        s["w"] = _Buffer(1.0 + 0.1 * torch.randn(n, generator=g, device="cuda"))
        s["xout"] = _empty(rows, n)
        s["codes"], s["scales"] = _codes8(rows, n)
    elif kind == "token":
        s["wc"], s["ws"] = _weight(c["n"], c["k"], g)
        s["x"] = _Buffer(_activations(1, c["k"], g))
        s["out"] = _empty(c["n"])
    else:
        rows = c["n"] if kind == "product" else 2 * c["ff"]
        s["wc"], s["ws"] = _weight(rows, c["k"], g)
        codes, scales = _to_mxfp8(_activations(c["m"], c["k"], g))
        s["ac"], s["as"] = _Buffer(codes.to(torch.float8_e4m3fn).view(torch.uint8)), _Buffer(scales)
        if kind == "product":
            s["out"] = _empty(c["m"], c["n"])
        else:
            s["codes"], s["scales"] = _codes8(c["m"], c["ff"])
            s["values"] = _empty(c["m"], c["ff"], dtype=torch.bfloat16)
    torch.cuda.synchronize()
    return s


# ---- plain forms --------------------------------------------------------------------------------------
def _exponents(x, largest):
    """Scale bytes of the blocks of x [..., blocks, 32] f32, and 2^(127 - byte)."""
    field = (x.abs().amax(-1).view(torch.int32) >> 23) & 255
    s = (field - largest).clamp(min=0)
    s = torch.where(field == 255, field, s)
    return s.to(torch.uint8), ((254 - s.clamp(max=253)) << 23).view(torch.float32)


def _to_mxfp4(x):
    """e2m1 codes (a byte each) and scale bytes of rows of f32."""
    b = x.view(x.shape[0], -1, BLOCK)
    s, up = _exponents(b, 2)
    v = b * up[..., None]
    a = v.abs()
    # borders between neighbouring magnitudes; a tie goes to the code that is even
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code | (torch.signbit(v).to(torch.uint8) << 3)).view(x.shape), s


def _packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _to_mxfp8(x):
    """e4m3 elements (as f32 numbers) and scale bytes of rows of f32."""
    b = x.view(x.shape[0], -1, BLOCK)
    s, up = _exponents(b, 8)
    v = (b * up[..., None]).clamp(-448.0, 448.0)
    return v.to(torch.float8_e4m3fn).to(torch.float32).view(x.shape), s


def _times_scales(v, scales):
    bits = scales.to(torch.int32) << 23
    f = torch.where(scales == 0, torch.full_like(bits, 0x00400000), bits).view(torch.float32)
    return (v.view(*scales.shape, BLOCK) * f[..., None]).view(v.shape)


def _values4(codes, scales):
    """f32 values of an MXFP4 weight of packed codes."""
    table = torch.tensor(GRID4 + tuple(-v for v in GRID4), device="cuda")
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return _times_scales(table[both.to(torch.int32)], scales)


def _values8(codes, scales):
    return _times_scales(codes.view(torch.float8_e4m3fn).to(torch.float32), scales)


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "load":
        code, scales = _to_mxfp4(s["src"].t.to(torch.float32))
        return {"values": _values4(_packed(code), scales).to(torch.bfloat16), "scales": scales}
    if kind == "rows":
        v, scales = _to_mxfp8(s["src"].t)
        return {"codes": v.to(torch.float8_e4m3fn), "scales": scales}
    if kind == "norm":
        x = s["x"].t
        if c["parts"]:
            x = x + functools.reduce(torch.add, s["parts"].t)      # the order in which a product's parts are added up
        d = x.to(torch.float64)               # 64 bits: elements next to the border between two codes
        h = d * (1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)) * s["w"].t.to(torch.float64)
        v, scales = _to_mxfp8(h.to(torch.float32))
        return {"xout": x, "codes": v.to(torch.float8_e4m3fn), "scales": scales}
    w = _values4(s["wc"].t, s["ws"].t)
    if kind == "token":
        return s["x"].t[0] @ w.T
    y = _values8(s["ac"].t, s["as"].t) @ w.T
    if kind == "product":
        return y
    gate, up = y[:, :c["ff"]], y[:, c["ff"]:]
    v, scales = _to_mxfp8(gate * torch.sigmoid(gate) * up)
    return _times_scales(v, scales).to(torch.bfloat16)


# ---- the library's calls ------------------------------------------------------------------------------
def _run_own(s):
    global _lib
    if _lib is None:
        _lib = importlib.import_module("cpp-tensorlib_amd").load()
    lib, c, kind = _lib, s["case"], s["case"]["kind"]
    if kind == "load":
        src_type = {"f32": lib.T_F32, "f16": lib.T_F16, "bf16": lib.T_BF16}[c["type"]]
        lib.quantize_mxfp4(s["src"], src_type, s["codes"], s["scales"], c["rows"], c["k"])
        lib.dequantize_mxfp4(s["codes"], s["scales"], s["values"], lib.T_BF16, c["rows"], c["k"])
        return {"values": s["values"].t, "scales": s["scales"].t}
    if kind == "rows":
        lib.quantize_mxfp8(s["src"], s["codes"], s["scales"], c["rows"], c["k"])
        return {"codes": s["codes"].t.view(torch.float8_e4m3fn), "scales": s["scales"].t}
    if kind == "norm":
        lib.rmsnorm_res_mxfp8(s["x"], s["parts"], c["parts"], s["w"], s["xout"], s["codes"], s["scales"], c["n"], EPS, c["rows"])
        return {"xout": s["xout"].t, "codes": s["codes"].t.view(torch.float8_e4m3fn), "scales": s["scales"].t}
    if kind == "token":
        lib.gemv_mxfp4(s["x"], s["wc"], s["ws"], s["out"], c["n"], c["k"])
        return s["out"].t
    if kind == "product":
        lib.gemm_mxfp4_nt(s["ac"], s["as"], s["wc"], s["ws"], s["out"], c["m"], c["n"], c["k"])
        return s["out"].t
    lib.gemm_mxfp4_nt_swiglu(s["ac"], s["as"], s["wc"], s["ws"], s["codes"], s["scales"], c["m"], c["ff"], c["k"])
    lib.dequantize_mxfp8(s["codes"], s["scales"], s["values"], lib.T_BF16, c["m"], c["ff"])
    return s["values"].t


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    mx4, mx8 = 0.5 + 1 / BLOCK, 1 + 1 / BLOCK              # bytes an element with its share of the scale
    if kind == "load":                                      # written, and read again for the values
        n = c["rows"] * c["k"]
        return {"bytes": n * ({"f32": 4, "f16": 2, "bf16": 2}[c["type"]] + 2 * mx4 + 2), "flops": 0}
    if kind == "rows":
        return {"bytes": c["rows"] * c["k"] * (4 + mx8), "flops": 0}
    if kind == "norm":
        return {"bytes": c["rows"] * c["n"] * (4 * (2 + c["parts"]) + mx8) + 4 * c["n"], "flops": 6 * c["rows"] * c["n"]}
    if kind == "token":
        return {"bytes": c["n"] * c["k"] * mx4 + 4 * (c["n"] + c["k"]), "flops": 2 * c["n"] * c["k"]}
    m, k = c["m"], c["k"]
    rows = c["n"] if kind == "product" else 2 * c["ff"]
    # the gated activation's values are read back from what was written
    out = 4 * m * c["n"] if kind == "product" else m * c["ff"] * (2 * mx8 + 2)
    return {"bytes": m * k * mx8 + rows * k * mx4 + out, "flops": 2 * m * rows * k}


# ---- the definitions in 64 bits -----------------------------------------------------------------------
D64 = torch.float64


def _nearest(x, mantissa, lowest, largest_exp, largest):
    """Blocks of x rounded to elements of `mantissa` bits, exponents lowest .. largest_exp and magnitudes up to `largest`
    under their scale: (values, scales, elements)."""
    b = x.to(D64).view(*x.shape[:-1], -1, BLOCK)
    big = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(big.clamp(min=2.0 ** -126))) - largest_exp
    scale = torch.pow(torch.full_like(big, 2.0), e.clamp(min=-127.0))
    v = b / scale
    step = torch.pow(torch.full_like(v, 2.0), torch.floor(torch.log2(v.abs().clamp(min=2.0 ** lowest))).clamp(min=lowest) - mantissa)
    v = (torch.round(v / step) * step).clamp(-largest, largest)
    return (v * scale).view(x.shape), scale, v.view(x.shape)


def _real4(codes, scales, i):
    """Rows i .. i + 4096 of an MXFP4 weight: sign, two bits of exponent, one of mantissa."""
    p = codes[i:i + 4096]
    q = torch.stack([p.remainder(16), p.div(16, rounding_mode="floor")], -1).flatten(1).to(D64)
    e, m, sign = q.div(2, rounding_mode="floor").remainder(4), q.remainder(2), 1.0 - 2.0 * (q >= 8)
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2.0, e - 1)) * sign
    return (v.view(len(p), -1, BLOCK) * torch.pow(2.0, scales[i:i + 4096].to(D64) - 127)[..., None]).flatten(1)


def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    if kind == "load":
        return {"values": _nearest(s["src"].t, 1, 0, 2, 6.0)[0], "scales": None}
    if kind == "rows":
        return {"codes": _nearest(s["src"].t, 3, -6, 8, 448.0)[2], "scales": None}
    if kind == "norm":
        x = s["x"].t.to(D64)
        if c["parts"]:
            x = x + s["parts"].t.to(D64).sum(0)
        h = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["n"] + EPS) * s["w"].t.to(D64)
        return {"xout": x, "codes": _nearest(h, 3, -6, 8, 448.0)[2], "scales": None}
    wc, ws = s["wc"].t, s["ws"].t
    if kind == "token":
        a = s["x"].t.to(D64)
    else:
        a = s["ac"].t.view(torch.float8_e4m3fn).to(D64).view(c["m"], -1, BLOCK)
        a = (a * torch.pow(2.0, s["as"].t.to(D64) - 127)[..., None]).flatten(1)
    y = torch.cat([a @ _real4(wc, ws, i).T for i in range(0, len(wc), 4096)], 1)
    if kind == "token":
        return y[0]
    if kind == "product":
        return y
    gate, up = y[:, :c["ff"]], y[:, c["ff"]:]
    return _nearest(gate / (1 + torch.exp(-gate)) * up, 3, -6, 8, 448.0)[0]
