"""The operators of a layer whose matrix products run in 8-bit integers: what each is timed on, in plain form and as the
framework's calls.

Kinds of case (one dict of plain values each; sizes from the repository's tests and benchmark, or generic):

  norm      rmsnorm_i8: the residual's addition, the root-mean-square norm and its rows in 8 bits with a scale each
  quantize  quantize_i8: rows in 8 bits with a scale each (attention output, SwiGLU output, a matrix's channels)
  gemm      gemm_i8: product of 8-bit rows with 8-bit channels, scaled per token and channel, SwiGLU as its epilogue where asked

8 bits are whole numbers of -127 .. 127, the same in both forms: the norm's factor belongs to the scale, so that no sum's order
reaches them. They are returned as they are, with their scales beside them.
"""
import importlib.util
import math
import os
import sys

import torch

own = False
DEV = "cuda"
EPS = 1e-5
_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"none": 0, "f32": 4, "f16": 2, "bf16": 2}


def _int8():
    """The package's directory name carries a hyphen: load it by path under its import name."""
    name = "llm_infer_b200"
    if name not in sys.modules:
        here = os.path.join(os.getcwd(), "llm-infer_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from llm_infer_b200 import int8
    return int8


# ------------------------------------------------------------------------------------------------------------ cases
def _norm(rows, dim, dtype, delta):
    return dict(kind="norm", rows=rows, dim=dim, dtype=dtype, delta=delta)


def _quantize(rows, dim, dtype):
    return dict(kind="quantize", rows=rows, dim=dim, dtype=dtype)


def _gemm(m, k, n, swiglu, out):
    return dict(kind="gemm", m=m, k=k, n=n, swiglu=swiglu, out=out)


def listed():
    return [
        # a generation step of one sequence: residual, norm and quantisation of one row; launch latency
        dict(_norm(1, 4096, "f32", "f32"), name="norm_step"),
        # a serving batch of a model of odd width that keeps its residual stream in bf16
        dict(_norm(61, 5003, "bf16", "bf16"), name="norm_b61_d5003"),
        # every token of eight prompts between two projections
        dict(_norm(9184, 4096, "f32", "f32"), name="norm_prompt_9184"),
        # the hidden activations of a generation step in front of the down projection
        dict(_quantize(8, 14336, "bf16"), name="quantize_b8_d14336"),
        # attention output of a prompt in front of the output projection
        dict(_quantize(1003, 4096, "f32"), name="quantize_1003_d4096"),
        # hidden activations of every token of eight prompts
        dict(_quantize(9184, 14336, "bf16"), name="quantize_prompt_9184"),
        # stacked q, k and v projection of one sequence's step: the weights are read once, latency counts
        dict(_gemm(1, 4096, 6144, False, "f32"), name="gemm_step_qkv"),
        # gate and up projection of eight sequences, SwiGLU
        dict(_gemm(8, 4096, 14336, True, "bf16"), name="gemm_b8_swiglu"),
        # odd everything: a short prompt in a model whose widths are no multiples of anything
        dict(_gemm(203, 1011, 4099, False, "f16"), name="gemm_203_k1011_n4099"),
        # classifier over the last tokens of a batch
        dict(_gemm(61, 4096, 128256, False, "f32"), name="gemm_b61_classifier"),
        # down projection of one prompt
        dict(_gemm(1003, 14336, 4096, False, "f32"), name="gemm_1003_down"),
        # gate and up projection of every token of eight prompts, SwiGLU
        dict(_gemm(9184, 4096, 14336, True, "bf16"), name="gemm_prompt_9184_swiglu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quantize", "gemm", "gemm", "gemm"])
    grain = rng.choice([1, 1, 8, 64])  # widths that are odd, or multiples of what models have

    def width(lo, hi):
        return max(grain, _log(rng, lo, hi) // grain * grain)

    if kind == "norm":
        dim = width(64, 16384)
        return _norm(_log(rng, 1, min(16384, 9184 * 4096 // dim)), dim, rng.choice(["f32", "f16", "bf16"]),
                     rng.choice(["none", "f32", "f16", "bf16"]))
    if kind == "quantize":
        dim, dtype = width(64, 28672), rng.choice(["f32", "f16", "bf16"])
        return _quantize(_log(rng, 1, min(16384, 9184 * 14336 * 3 // (dim * (_BYTES[dtype] + 1)))), dim, dtype)
    swiglu = rng.random() < 0.4
    k, n = width(64, 14336), width(64, 14336)
    m = _log(rng, 1, min(16384, 9184 * 4096 * 14336 // (k * n)))
    return _gemm(m, k, n, swiglu, rng.choice(["f32", "f16", "bf16"]))


# ----------------------------------------------------------------------------------------------------------- inputs
def _rows(g, rows, dim, spread=1.0):
    """Activations: normal, with every 97th channel eight times as large, as trained models have them."""
    x = torch.randn((rows, dim), generator=g, device=DEV) * spread
    x[:, 5::97] *= 8.0
    return x


def _bytes_of(x):
    """8-bit rows of x and their scales, the rows 16 bytes apart or a multiple of that, as the entry points lay them out."""
    rows, dim = x.shape
    top = x.abs().amax(1)
    q = torch.empty((rows, (dim + 15) // 16 * 16), dtype=torch.int8, device=DEV)[:, :dim]
    q.copy_(torch.round(x * (127.0 / top)[:, None]))
    return q, top / 127.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    c = dict(case)
    if c["kind"] == "gemm":
        c["a"], c["a_scale"] = _bytes_of(_rows(g, c["m"], c["k"]))
        w_rows = c["n"] * (2 if c["swiglu"] else 1)
        c["w"], c["w_scale"] = _bytes_of(torch.randn((w_rows, c["k"]), generator=g, device=DEV) * c["k"] ** -0.5)
        return c
    c["x"] = _rows(g, c["rows"], c["dim"]).to(_T[c["dtype"]])
    if c["kind"] == "norm":
        c["weight"] = 1.0 + 0.1 * torch.randn(c["dim"], generator=g, device=DEV)
        if c["delta"] != "none":
            c["d"] = _rows(g, c["rows"], c["dim"], 0.5).to(_T[c["delta"]])
            c["x_out"] = torch.empty_like(c["x"])
    return c


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_rows(z, factor):
    """Rows z (32 bits) as whole numbers of -127 .. 127 and their scales; ``factor`` [rows] belongs to the scales."""
    top = z.abs().amax(1)
    inverse = torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))
    return torch.round(z * inverse[:, None]).to(torch.int8), factor * top * (1.0 / 127.0)


def _plain_norm(s):
    h = s["x"].float()
    if s["delta"] != "none":
        h = h + s["d"].float()
    factor = 1.0 / torch.sqrt(h.square().mean(1) + EPS)
    q, scale = _plain_rows(h * s["weight"], factor)
    return (q, scale, h.to(s["x"].dtype)) if s["delta"] != "none" else (q, scale)


def _plain_gemm(s):
    # (whole numbers: a sum of 32 bits is exact up to 2^24 and off by 2^-24 of itself above)
    y = (s["a"].float() @ s["w"].float().t()) * s["a_scale"][:, None] * s["w_scale"]
    if s["swiglu"]:
        gate, up = y[:, :s["n"]], y[:, s["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(_T[s["out"]])


def run(s):
    if own:
        i8 = _int8()
        if s["kind"] == "gemm":
            return i8.gemm_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], out_dtype=_T[s["out"]], swiglu=s["swiglu"])
        if s["kind"] == "quantize":
            return i8.quantize_i8(s["x"])
        if s["delta"] == "none":
            return i8.rmsnorm_i8(s["x"], s["weight"], EPS)
        q, scale = i8.rmsnorm_i8(s["x"], s["weight"], EPS, delta=s["d"], x_out=s["x_out"])
        return q, scale, s["x_out"]
    if s["kind"] == "gemm":
        return _plain_gemm(s)
    if s["kind"] == "quantize":
        x = s["x"].float()
        return _plain_rows(x, torch.ones_like(x[:, 0]))
    return _plain_norm(s)


# ------------------------------------------------------------------------------------------------------ work, exact
def work(case):
    if case["kind"] == "gemm":
        m, k, n = case["m"], case["k"], case["n"]
        w_rows = n * (2 if case["swiglu"] else 1)
        return {"bytes": m * k + w_rows * k + 4 * (m + w_rows) + m * n * _BYTES[case["out"]], "flops": 2 * m * w_rows * k}
    count, size = case["rows"] * case["dim"], _BYTES[case["dtype"]]
    if case["kind"] == "quantize":
        return {"bytes": count * (size + 1) + 4 * case["rows"], "flops": 4 * count}
    delta = _BYTES[case["delta"]]
    return {"bytes": count * (size + delta + (size if delta else 0) + 1) + 4 * (case["rows"] + case["dim"]), "flops": 8 * count}


def exact(case, seed):
    """From the definitions, in 64 bits: y = x / sqrt(mean(x^2) + eps) * weight; scale = max|y| / 127, q = the whole number next to
    y / scale; out = sum over the inner dimension of the values that q and scale stand for."""
    s = prepare(case, seed)
    if case["kind"] == "gemm":
        a = s["a"].double() * s["a_scale"].double()[:, None]
        out = torch.matmul(a, (s["w"].double() * s["w_scale"].double()[:, None]).transpose(0, 1))
        if case["swiglu"]:
            gate, up = out.split(case["n"], dim=1)
            out = gate * torch.sigmoid(gate) * up
        return out
    x = s["x"].double()
    if case["kind"] == "quantize":
        y, rest = x, ()
    else:
        if case["delta"] != "none":
            x = x + s["d"].double()
        y = x * torch.rsqrt((x * x).sum(1, keepdim=True) / case["dim"] + EPS) * s["weight"].double()
        rest = (x,) if case["delta"] != "none" else ()
    scale = y.abs().amax(1) / 127.0
    return (torch.round(y / scale[:, None]).to(torch.int8), scale) + rest
