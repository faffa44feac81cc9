"""What the operators for 8-bit operands with a scale per token and per channel are timed on, from one token to a data-set shard:

  norm    RMS norm with the residual's addition, quantised: to int8 or e4m3 with a scale for each row, or ("static") to e4m3
          with a scale that a calibrated model has for the whole tensor
  rows    quantisation of an activation, a scale for each row
  linear  the product of two such operands, scales for each token and output channel, bias, optionally GELU

``run`` computes them in elementary torch operations, or (``own``) through ``siglip_b200.Engine``.  int8 codes come back as the
values they stand for (bf16), beside their scales; e4m3 codes as the float8 numbers that they are, beside theirs.  Sizes are those of the
encoders the repository is configured for (768 wide; 1152 / 4304 at 729 tokens an image) and generic ones.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

EPS = 1e-6
STATIC_SCALE = 8.0 / 448.0      # a calibrated model: norm outputs within +-8
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
SMALLEST = 2.0 ** -126          # no scale is smaller


def listed() -> list:
    return [
        # one token's residual stream in front of a projection: launches and latency
        dict(name="norm_1", kind="norm", rows=1, cols=1152, dtype="bf16", residual=True, codes="int8"),
        # seven images packed to the tokens that a mask left over
        dict(name="norm_ragged", kind="norm", rows=5003, cols=1152, dtype="bf16", residual=True, codes="e4m3"),
        # a long prompt through a wider model
        dict(name="norm_wide", kind="norm", rows=16384, cols=4096, dtype="bf16", residual=True, codes="int8"),
        # 64 images, a model that keeps its residual stream in fp32 and has calibrated scales
        dict(name="norm_static", kind="norm", rows=64 * 729, cols=1152, dtype="f32", residual=False, codes="static"),
        # GELU outputs of a few tokens in front of FC2
        dict(name="rows_8", kind="rows", rows=8, cols=4304, dtype="bf16", codes="int8"),
        # fp32 activations of an odd width: rows that start on no 16-byte boundary
        dict(name="rows_odd", kind="rows", rows=3001, cols=1155, dtype="f32", codes="e4m3"),
        # GELU outputs of 64 images
        dict(name="rows_64", kind="rows", rows=64 * 729, cols=4304, dtype="bf16", codes="int8"),
        # FC2 for one token: 5 MB of weights that stay in L2
        dict(name="linear_1", kind="linear", rows=1, n=1152, k=4304, codes="int8", gelu=False, bias="bf16"),
        # sixteen sequences, a token each, through a wide layer: 64 MB of weights
        dict(name="linear_16", kind="linear", rows=16, n=8192, k=8192, codes="int8", gelu=False, bias="none"),
        # FC1 + GELU of one image
        dict(name="linear_729", kind="linear", rows=729, n=4304, k=1152, codes="e4m3", gelu=True, bias="bf16"),
        # FC2 of seven images packed
        dict(name="linear_ragged", kind="linear", rows=5003, n=1152, k=4304, codes="int8", gelu=False, bias="f32"),
        # FC1 + GELU of 64 images
        dict(name="linear_64", kind="linear", rows=64 * 729, n=4304, k=1152, codes="int8", gelu=True, bias="bf16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "rows", "linear", "linear"])
    if kind == "linear":
        # widths of the two encoders, or of no model's; K need not be a whole number of vectors
        n, k = rng.choice([(1152, 4304), (4304, 1152), (768, 768), (16 * _log(rng, 8, 512), _log(rng, 100, 9000)), (16 * _log(rng, 8, 512), _log(rng, 100, 9000))])
        rows = _log(rng, 1, max(2, min(60_000, 64 * 729 * 4304 * 1152 // (n * k))))
        return dict(kind=kind, rows=rows, n=n, k=k, codes=rng.choice(["int8", "int8", "e4m3"]), gelu=rng.random() < 0.4,
                    bias=rng.choice(["bf16", "f32", "none"]))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    cols = rng.choice([768, 1152, 4304, 8 * _log(rng, 4, 2048), _log(rng, 32, 16384)])
    rows = _log(rng, 1, max(2, min(100_000, 150_000_000 // cols // (2 if dtype == "f32" else 1))))
    if kind == "rows":
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, codes=rng.choice(["int8", "e4m3"]))
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7, codes=rng.choice(["int8", "e4m3", "static"]))


def _type(name: str) -> torch.dtype:
    return {"bf16": torch.bfloat16, "f32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn, "static": torch.float8_e4m3fn}[name]


def _pitched(rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """A buffer of 8-bit codes: rows on 128-byte lines."""
    return torch.zeros((rows, (cols + 127) // 128 * 128), dtype=torch.uint8, device="cuda").view(dtype)[:, :cols]


def _operand(x: torch.Tensor, codes: str):
    """Codes and scales of an operand as a program holds them, made in slices so that a large one fits beside itself."""
    q, scales = _pitched(*x.shape, _type(codes)), torch.empty(x.shape[0], device="cuda")
    for r in range(0, x.shape[0], 8192):
        v = x[r:r + 8192].float()
        s = v.abs().amax(1) / CODE_MAX[codes]
        v = v / s[:, None]
        q[r:r + 8192] = v.round().to(torch.int8) if codes == "int8" else v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        scales[r:r + 8192] = s
    return q, scales


def prepare(case: dict, seed: int) -> dict:
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = dict(kind=c["kind"], codes=c["codes"])
    if c["kind"] == "linear":
        rows, n, k = c["rows"], c["n"], c["k"]
        # activations: channels of different size, a few of them large, tokens of different size
        x = (normal(rows, k) * torch.exp(0.5 * normal(k)) * torch.exp(0.3 * normal(rows, 1))).to(torch.bfloat16)
        s["A"], s["scale_a"] = _operand(x, c["codes"])
        s["W"], s["scale_w"] = _operand(normal(n, k) * (1.0 / math.sqrt(k)), c["codes"])
        s["bias"] = None if c["bias"] == "none" else (normal(n) * 0.1).to(_type(c["bias"]))
        s.update(gelu=c["gelu"], D=torch.empty((rows, n), dtype=torch.bfloat16, device="cuda"))
        return s
    rows, cols = c["rows"], c["cols"]
    size = torch.exp(0.5 * normal(cols))
    s["x"] = (normal(rows, cols) * size).to(_type(c["dtype"]))
    if c["kind"] == "norm":
        s["gamma"] = 1 + 0.1 * normal(cols)
        s["residual"] = (3 * normal(rows, cols) * size).to(_type(c["dtype"])) if c["residual"] else None
        s["summed"] = torch.empty_like(s["x"]) if c["residual"] else None
        s["scale"] = torch.tensor([STATIC_SCALE], device="cuda")
    # the buffers of a serving loop
    s["q"] = _pitched(rows, cols, _type(c["codes"]))
    if c["codes"] != "static":
        s["scales"] = torch.empty(rows, device="cuda")
    if c["codes"] == "int8":
        s["values"] = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    return s


@functools.lru_cache(maxsize=None)
def _engine():
    from siglip_b200 import Engine
    return Engine(0)          # a program keeps one handle per GPU


def _run_own(s: dict):
    eng = _engine()
    if s["kind"] == "linear":
        from siglip_b200 import lib
        return eng.linear_scaled(s["A"], s["W"], s["scale_a"], s["scale_w"], s["bias"], out=s["D"], flags=lib.SL8_FLAG_GELU if s["gelu"] else 0)
    if s["codes"] == "static":
        out = eng.rmsnorm_quantize(s["x"], s["gamma"], EPS, s["scale"], residual=s["residual"], summed=s["summed"], out=s["q"])
        return out if s["residual"] is not None else (out,)
    if s["kind"] == "rows":
        q, scales = eng.quantize_rows(s["x"], s["q"].dtype, out=s["q"], scales=s["scales"])
        rest = ()
    else:
        q, scales, *rest = eng.rmsnorm_quantize_rows(s["x"], s["gamma"], EPS, s["q"].dtype, residual=s["residual"], summed=s["summed"],
                                                     out=s["q"], scales=s["scales"])
    return (_values(q, scales, s), scales, *rest)


def _values(q: torch.Tensor, scales: torch.Tensor, s: dict) -> torch.Tensor:
    """What int8 codes stand for; float8 codes are numbers as they are."""
    return torch.mul(q, scales[:, None], out=s["values"]) if s["codes"] == "int8" else q


def run(s: dict):
    if own:
        return _run_own(s)
    if s["kind"] == "linear":
        y = s["A"].float() @ s["W"].float().T * s["scale_a"][:, None] * s["scale_w"]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["gelu"]:
            y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
        return y.to(torch.bfloat16)
    y, rest = s["x"].float(), ()
    if s["kind"] == "norm":
        if s["residual"] is not None:
            y = y + s["residual"].float()
            rest = (y.to(s["x"].dtype),)
        y = y * s["gamma"] * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    if s["codes"] == "static":
        return ((y / s["scale"]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), *rest)
    amax = y.abs().amax(1)
    scales = torch.where(amax == 0, torch.ones_like(amax), (amax / CODE_MAX[s["codes"]]).clamp(min=SMALLEST))
    y = y / scales[:, None]
    q = y.round().to(torch.int8) if s["codes"] == "int8" else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (_values(q, scales, s), scales, *rest)


def work(case: dict) -> dict:
    """Inputs once, outputs once (codes and scales, not the values that ``run`` makes of int8 codes to be compared)."""
    c = case
    if c["kind"] == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": m * k + n * k + 4 * m + 4 * n + {"bf16": 2, "f32": 4, "none": 0}[c["bias"]] * n + 2 * m * n, "flops": 2 * m * n * k}
    m, n, t = c["rows"], c["cols"], 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "rows":
        return {"bytes": m * n * (t + 1) + 4 * m, "flops": 3 * m * n}
    return {"bytes": m * n * ((3 if c["residual"] else 1) * t + 1) + 4 * n + (0 if c["codes"] == "static" else 4 * m), "flops": 7 * m * n}


def _nearest_e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number of each value in 64 bits, ties to the even one: three bits behind the leading one, a step of 2^-9 below 2^-6."""
    v = torch.clip(v, -448.0, 448.0)
    step = torch.ldexp(torch.ones_like(v), torch.clip(torch.frexp(v).exponent - 4, min=-9))
    return torch.round(v / step) * step


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s["kind"] == "linear":
        out = torch.empty((case["rows"], case["n"]), dtype=torch.float64, device="cuda")
        w = s["W"].double().T.contiguous() * s["scale_w"].double()
        for r in range(0, case["rows"], 4096):
            p = torch.matmul(s["A"][r:r + 4096].double(), w) * s["scale_a"][r:r + 4096, None].double()
            if s["bias"] is not None:
                p += s["bias"].double()
            if s["gelu"]:         # x (1 + tanh u) / 2 is x / (1 + exp(-2 u))
                p /= 1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3))
            out[r:r + 4096] = p
        return out
    parts = []
    for r in range(0, case["rows"], 4096):
        h, rest = s["x"][r:r + 4096].double(), []
        if s["kind"] == "norm":
            if s["residual"] is not None:
                h = h + s["residual"][r:r + 4096].double()
                rest = [h]
            h = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["cols"] + EPS) * s["gamma"].double()
        if s["codes"] == "static":
            parts.append([_nearest_e4m3(h / s["scale"].double()), *rest])
            continue
        largest = torch.linalg.vector_norm(h, ord=math.inf, dim=1)
        scale = torch.where(largest > 0, largest / CODE_MAX[s["codes"]], 1.0)
        q = h / scale[:, None]
        parts.append([torch.round(q) * scale[:, None] if s["codes"] == "int8" else _nearest_e4m3(q), scale, *rest])
    return [torch.cat(p) for p in zip(*parts)]
