"""The operators of a server with long contexts: what each is timed on, in plain form and as the framework's calls.

Kinds of case (one dict of plain values each; sizes from the repository's tests and benchmark, or generic):

  rope    rope_positions: rotary embedding of the tokens' q and k (interleaved or half layout, part of the head, scaled
          frequencies) and the insert of k and v into the caches
  shared  attn_decode_shared: one token's attention of a batch over a prefix that all its sequences share and the rows of
          their own caches
  scored  the same, which also adds the weight that each own row received to an accumulator per kv head
  evict   kv_evict: the rows of largest accumulated weight (with the first and the last ones) move from a prompt's cache
          into a smaller one

Ragged lengths are a function of the case, so that a case's work is known without its inputs.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
GOLDEN = 0.6180339887498949
_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _context():
    """The package's directory name carries a hyphen: load it by path under its import name."""
    name = "llm_infer_b200"
    if name not in sys.modules:
        here = os.path.join(os.getcwd(), "llm-infer_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from llm_infer_b200 import context
    return context


# ------------------------------------------------------------------------------------------------------------ cases
def _shared(kind, batch, prefix, rows, heads, kv_heads, dim, dtype, out):
    return dict(kind=kind, batch=batch, prefix=prefix, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, out=out)


def _evict(batch, rows, keep, sink, recent, kv_heads, dim, dtype):
    return dict(kind="evict", batch=batch, rows=rows, keep=keep, sink=sink, recent=recent, kv_heads=kv_heads, dim=dim, dtype=dtype)


def _rope(batch, tokens, first, heads, kv_heads, dim, rotary, layout, scaling, dtype, q_out, cache):
    return dict(kind="rope", batch=batch, tokens=tokens, first=first, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                layout=layout, scaling=scaling, dtype=dtype, q_out=q_out, cache=cache)


def listed():
    return [
        # a generation step's rotary embedding: eight sequences, one token each, late positions; launch latency
        dict(_rope(8, 1, 100000, 32, 8, 128, 128, "half", "llama3", "f32", "f16", "f16"), name="rope_step_b8"),
        # all tokens of eight prompts of a model that rotates part of the head, scaled positions
        dict(_rope(8, 1148, 0, 32, 8, 128, 64, "interleaved", "yarn", "bf16", "bf16", "bf16"), name="rope_prompt_9184"),
        # two users behind one short system prompt, 1.1B-shaped: the smallest attention call
        dict(_shared("shared", 2, 512, 64, 32, 4, 64, "f16", "f16"), name="shared_b2_p512_d64"),
        # a serving batch of an 8B-shaped layer behind a few pages of instructions, ragged answers
        dict(_shared("shared", 16, 4096, 512, 32, 8, 128, "f16", "f16"), name="shared_b16_p4096"),
        # many users over one document, the attention of the prefix is a matrix product for each kv head
        dict(_shared("shared", 64, 16384, 1024, 32, 8, 128, "bf16", "bf16"), name="shared_b64_p16384"),
        # few users over one very long document (512 MiB of prefix), odd batch and lengths
        dict(_shared("shared", 7, 131072, 333, 32, 8, 128, "f16", "f16"), name="shared_b7_p131072"),
        # one sequence under a cache budget, no prefix, fp32 result for the engine's fp32 activations
        dict(_shared("scored", 1, 0, 1000, 32, 4, 64, "f16", "f32"), name="scored_b1_t1000_d64"),
        # the headline decode shape, accumulating weights
        dict(_shared("scored", 16, 0, 4096, 32, 8, 128, "f16", "f16"), name="scored_b16_t4096"),
        # prefix and accumulated weights at once, twelve heads to a kv head, bf16
        dict(_shared("scored", 9, 2048, 1777, 24, 2, 128, "bf16", "bf16"), name="scored_b9_p2048_g12"),
        # the smallest eviction: one sequence back to its budget
        dict(_evict(1, 1024, 256, 4, 64, 8, 128, "f16"), name="evict_b1_t1024"),
        # a batch of ragged prompts into budget-sized caches
        dict(_evict(16, 4096, 1999, 4, 256, 8, 128, "bf16"), name="evict_b16_t4096"),
        # one very long prompt down to an eighth
        dict(_evict(1, 131072, 16384, 4, 1024, 8, 128, "f16"), name="evict_b1_t131072"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "shared", "shared", "shared", "scored", "scored", "evict", "evict"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 4, 64), (32, 8, 128), (8, 2, 128), (16, 16, 64), (64, 8, 128), (24, 2, 128)])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "rope":
        batch = _log(rng, 1, 16)
        tokens = rng.choice([1, _log(rng, 1, 8192 // batch)])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rope(batch, tokens, _log(rng, 1, 120000), heads, kv_heads, dim, rotary, rng.choice(["interleaved", "half"]),
                     rng.choice(["none", "linear", "yarn", "llama3"]), rng.choice(["f32", dtype]), rng.choice(["f32", dtype]), dtype)
    if kind == "evict":
        batch = _log(rng, 1, 32)
        rows = _log(rng, 128, max(129, min(131072, 131072 * 8 // (batch * kv_heads))))
        keep = _log(rng, max(16, rows // 16), max(17, rows * 15 // 16))
        return _evict(batch, rows, keep, rng.choice([0, 4, 7]), rng.randint(0, keep // 4), kv_heads, dim, dtype)
    batch = _log(rng, 1, 64)
    # no more key rows in all, and no more products with the prefix, than the largest listed cases
    prefix = _log(rng, 64, max(65, min(131072, 131072 * 8 // kv_heads, 64 * 16384 * 32 // (batch * heads))))
    rows = _log(rng, 16, max(17, min(4096, 16 * 4096 * 8 // (batch * kv_heads))))
    if kind == "scored" and rng.random() < 0.5:
        prefix = 0
    return _shared(kind, batch, prefix, rows, heads, kv_heads, dim, dtype, rng.choice([dtype, dtype, "f32"]))


def _lengths(case):
    """Ragged lengths of the batch, spread over the upper part of the caches: a function of the case alone."""
    lo, hi = max(1, case["rows"] // 4), case["rows"]
    if case["batch"] == 1:
        return [hi]
    return [lo + int((hi - lo + 1) * ((i + 1) * GOLDEN % 1.0)) for i in range(case["batch"])]


# ----------------------------------------------------------------------------------------------------------- inputs
def _frequencies(rotary, scaling):
    """Scaled frequencies of the pairs and the factor on cos and sin, in 64 bits: the published formulas (base 500000,
    trained length 8192, eight times longer contexts)."""
    base, trained, scale = 500000.0, 8192.0, 8.0
    half = rotary // 2
    i = np.arange(half, dtype=np.float64)
    f = base ** (-2.0 * i / rotary)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / scale, 1.0
    if scaling == "llama3":  # long waves divided by the scale, short ones kept, a ramp between
        smooth = np.clip((trained * f / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return (1.0 - smooth) * f / scale + smooth * f, 1.0
    turn = lambda n: rotary * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rotary - 1)
    ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
    return f / scale * ramp + f * (1.0 - ramp), 0.1 * math.log(scale) + 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    normal = lambda *s, dtype, std=1.0: (torch.randn(s, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)  # noqa: E731
    st = dict(case=case)
    if case["kind"] == "rope":
        B, n, H, Hkv, D, T = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"], _T[case["dtype"]]
        N = B * n
        # the stacked projection's output: a token's q, k and v side by side
        qkv = normal(N, H + 2 * Hkv, D, dtype=T)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        f, factor = _frequencies(case["rotary"], case["scaling"])
        st["inv_freq"], st["factor"] = torch.from_numpy(f).to(torch.float32).to(DEV), factor
        seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(n)
        step = torch.arange(n, dtype=torch.int32, device=DEV).repeat(B)
        shift = torch.randint(0, 64, (B,), generator=g, device=DEV, dtype=torch.int32)
        st["seq"], st["row"] = seq, step + (shift % 3)[seq.long()]  # the cache row is not the position: rows were evicted before
        st["pos"] = case["first"] + shift[seq.long()] + step
        st["k_cache"] = torch.zeros((B, n + 5, Hkv, D), dtype=_T[case["cache"]], device=DEV)
        st["v_cache"] = torch.zeros_like(st["k_cache"])
        if own:
            st["context"] = _context()
        return st
    T = _T[case["dtype"]]
    B, R, Hkv, D = case["batch"], case["rows"], case["kv_heads"], case["dim"]
    st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    st["k"] = normal(B, R, Hkv, D, dtype=T)
    st["v"] = normal(B, R, Hkv, D, dtype=T)
    if case["kind"] == "evict":
        # accumulated weights: heavy-tailed, some rows never attended to (ties at zero)
        s = torch.exp(1.5 * torch.randn((B, Hkv, R), generator=g, device=DEV)) * 0.01
        st["scores"] = torch.where(torch.rand((B, Hkv, R), generator=g, device=DEV) < 0.1, torch.zeros_like(s), s)
        if own:
            st["context"] = _context()
            st["k_out"] = torch.zeros((B, case["keep"], Hkv, D), dtype=T, device=DEV)
            st["v_out"] = torch.zeros_like(st["k_out"])
            st["scores_out"] = torch.zeros((B, Hkv, case["keep"]), device=DEV)
        return st
    H, P = case["heads"], case["prefix"]
    st["q"] = normal(B, H, D, dtype=T, std=1.5)
    st["kp"] = normal(P, Hkv, D, dtype=T) if P else None
    st["vp"] = normal(P, Hkv, D, dtype=T) if P else None
    scored = case["kind"] == "scored"
    if scored:
        st["scores"] = torch.rand((B, Hkv, R), generator=g, device=DEV)
    if own:
        st["context"] = _context()
        st["workspace"] = st["context"].SharedWorkspace(B, H, Hkv, D, rows=R if scored else 0)
        if scored:
            st["scores_out"] = torch.zeros((B, Hkv, R), device=DEV)
    return st


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_rope(st):
    c, half = st["case"], st["case"]["rotary"] // 2
    # the angle alone in 64 bits: at position 100000 a product rounded to 32 bits is wrong by 4e-3
    turns = st["pos"].double()[:, None] * (st["inv_freq"].double() / (2 * math.pi))[None, :]
    angle = ((turns - torch.floor(turns)) * (2 * math.pi)).float()
    cos, sin = (torch.cos(angle) * st["factor"])[:, None, :], (torch.sin(angle) * st["factor"])[:, None, :]

    def rotate(x):
        x = x.float()
        y = x.clone()
        if c["layout"] == "half":
            a, b = x[..., :half], x[..., half:2 * half]
            y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
        return y

    seq, row = st["seq"].long(), st["row"].long()
    st["k_cache"][seq, row] = rotate(st["k"]).to(st["k_cache"].dtype)
    st["v_cache"][seq, row] = st["v"].float().to(st["v_cache"].dtype)
    return [rotate(st["q"]).to(_T[c["q_out"]]), st["k_cache"], st["v_cache"]]


def _plain_decode(st):
    c = st["case"]
    B, H, Hkv, D, P, R = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["prefix"], c["rows"]
    q = st["q"].float().view(B, Hkv, H // Hkv, D) / math.sqrt(D)
    valid = (torch.arange(R, device=DEV)[None, :] < st["lens"][:, None])[:, None, None, :]
    s = torch.matmul(q, st["k"].float().permute(0, 2, 3, 1))
    s = torch.where(valid, s, torch.full_like(s, -math.inf))
    if P:
        rows = q.permute(1, 0, 2, 3).reshape(Hkv, -1, D)
        sp = torch.matmul(rows, st["kp"].float().permute(1, 2, 0)).view(Hkv, B, H // Hkv, P).permute(1, 0, 2, 3)
        s = torch.cat([sp, s], dim=3)
    p = torch.exp(s - torch.amax(s, dim=3, keepdim=True))
    p = p / torch.sum(p, dim=3, keepdim=True)
    o = torch.matmul(p[..., P:], st["v"].float().permute(0, 2, 1, 3))
    if P:
        rows = p[..., :P].permute(1, 0, 2, 3).reshape(Hkv, -1, P)
        o = o + torch.matmul(rows, st["vp"].float().permute(1, 0, 2)).view(Hkv, B, H // Hkv, D).permute(1, 0, 2, 3)
    out = o.reshape(B, H, D).to(_T[c["out"]])
    if c["kind"] == "shared":
        return [out]
    weight = torch.sum(p[..., P:], dim=2)
    return [out, torch.where(valid[:, 0], st["scores"] + weight, torch.zeros_like(weight))]


def _plain_evict(st):
    c, lens, s = st["case"], st["lens"], st["scores"]
    B, R, keep, Hkv, D = c["batch"], c["rows"], c["keep"], c["kv_heads"], c["dim"]
    row = torch.arange(R, device=DEV)[None, None, :]
    n = lens[:, None, None]
    key = torch.where((row < c["sink"]) | (row >= n - c["recent"]), torch.full_like(s, math.inf), s)
    key = torch.where(row < n, key, torch.full_like(s, -1.0))
    picked = torch.sort(key, dim=2, descending=True, stable=True).indices[..., :keep]
    picked = torch.sort(torch.where(picked < n, picked, torch.full_like(picked, R)), dim=2).values
    there = picked < R
    at = torch.where(there, picked, torch.zeros_like(picked))
    index = at.permute(0, 2, 1)[..., None].expand(B, keep, Hkv, D)
    mask = there.permute(0, 2, 1)[..., None]
    k = torch.where(mask, torch.gather(st["k"], 1, index), torch.zeros((), dtype=st["k"].dtype, device=DEV))
    v = torch.where(mask, torch.gather(st["v"], 1, index), torch.zeros((), dtype=st["v"].dtype, device=DEV))
    scores = torch.where(there, torch.gather(s, 2, at), torch.zeros_like(s[..., :keep]))
    kept = torch.where(there, picked, torch.full_like(picked, -1)).to(torch.int32)
    return [k, v, scores, kept, torch.clamp(lens, max=keep)]


# ---------------------------------------------------------------------------------------------------------- one pass
def run(st):
    c = st["case"]
    if not own:
        return {"rope": _plain_rope, "shared": _plain_decode, "scored": _plain_decode, "evict": _plain_evict}[c["kind"]](st)
    ctx = st["context"]
    if c["kind"] == "rope":
        q = ctx.rope_positions(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["pos"], st["row"], seq=st["seq"],
                               inv_freq=st["inv_freq"], factor=st["factor"], layout=c["layout"], q_out_dtype=_T[c["q_out"]])
        return [q, st["k_cache"], st["v_cache"]]
    if c["kind"] == "evict":
        kept, lens = ctx.kv_evict(st["k"], st["v"], st["scores"], st["lens"], c["keep"], sink=c["sink"], recent=c["recent"],
                                  out=(st["k_out"], st["v_out"], st["scores_out"]))
        return [st["k_out"], st["v_out"], st["scores_out"], kept, lens]
    if c["kind"] == "scored":
        out = ctx.attn_decode_shared(st["q"], st["kp"], st["vp"], st["k"], st["v"], st["lens"], out_dtype=_T[c["out"]],
                                     scores=st["scores"], scores_out=st["scores_out"], workspace=st["workspace"])
        return [out, st["scores_out"]]
    return [ctx.attn_decode_shared(st["q"], st["kp"], st["vp"], st["k"], st["v"], st["lens"], out_dtype=_T[c["out"]],
                                   workspace=st["workspace"])]


def work(case):
    if case["kind"] == "rope":
        N = case["batch"] * case["tokens"]
        width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        moved = N * width * _BYTES[case["dtype"]] + N * case["heads"] * case["dim"] * _BYTES[case["q_out"]]
        moved += N * 2 * case["kv_heads"] * case["dim"] * _BYTES[case["cache"]] + 12 * N + 2 * case["rotary"]
        return {"bytes": moved, "flops": N * (case["heads"] + case["kv_heads"]) * case["rotary"] * 3}
    lens = _lengths(case)
    row = case["kv_heads"] * case["dim"] * 2 * 2  # K and V of one row, 16 bits
    if case["kind"] == "evict":
        after = sum(min(n, case["keep"]) for n in lens)
        moved = sum(lens) * case["kv_heads"] * 4 + after * row * 2 + case["batch"] * (case["kv_heads"] * case["keep"] * 8 + 8)
        return {"bytes": moved, "flops": sum(lens) * case["kv_heads"]}
    qo = case["batch"] * case["heads"] * case["dim"]
    moved = (case["prefix"] + sum(lens)) * row + qo * (2 + _BYTES[case["out"]]) + 4 * case["batch"]
    if case["kind"] == "scored":
        moved += sum(lens) * case["kv_heads"] * 8
    return {"bytes": moved, "flops": 4 * case["dim"] * case["heads"] * (case["batch"] * case["prefix"] + sum(lens))}


# ------------------------------------------------------------------------------------------------ in 64 bits, by itself
def _exact_rope(st):
    c, R = st["case"], st["case"]["rotary"]
    theta = torch.outer(st["pos"].double(), st["inv_freq"].double())
    z = torch.polar(torch.full_like(theta, st["factor"]), theta)[:, None, :]

    def turned(x):
        x = x.double()
        head, tail = x[..., :R], x[..., R:]
        if c["layout"] == "half":
            w = torch.complex(head[..., :R // 2].contiguous(), head[..., R // 2:].contiguous()) * z
            return torch.cat([w.real, w.imag, tail], dim=-1)
        w = torch.view_as_complex(head.reshape(*head.shape[:-1], R // 2, 2).contiguous()) * z
        return torch.cat([torch.view_as_real(w).flatten(-2), tail], dim=-1)

    kc, vc = torch.zeros_like(st["k_cache"], dtype=torch.float64), torch.zeros_like(st["v_cache"], dtype=torch.float64)
    at = (st["seq"].long(), st["row"].long())
    kc.index_put_(at, turned(st["k"]))
    vc.index_put_(at, st["v"].double())
    return [turned(st["q"]), kc, vc]


def _exact_decode(st):
    c = st["case"]
    G = c["heads"] // c["kv_heads"]
    out = torch.empty((c["batch"], c["heads"], c["dim"]), dtype=torch.float64, device=DEV)
    weights = torch.zeros((c["batch"], c["kv_heads"], c["rows"]), dtype=torch.float64, device=DEV)
    for h in range(c["kv_heads"]):
        kp = st["kp"][:, h].double() if c["prefix"] else None
        vp = st["vp"][:, h].double() if c["prefix"] else None
        for b, n in enumerate(_lengths(c)):
            q = st["q"][b, h * G:(h + 1) * G].double()
            s = q @ st["k"][b, :n, h].double().T
            if kp is not None:
                s = torch.cat([q @ kp.T, s], dim=1)
            s = s * c["dim"] ** -0.5
            lse = torch.logsumexp(s, dim=1, keepdim=True)
            p = torch.exp(s - lse)
            o = p[:, c["prefix"]:] @ st["v"][b, :n, h].double()
            if vp is not None:
                o = o + p[:, :c["prefix"]] @ vp
            out[b, h * G:(h + 1) * G] = o
            if c["kind"] == "scored":
                weights[b, h, :n] = st["scores"][b, h, :n].double() + p[:, c["prefix"]:].sum(0)
    return [out] if c["kind"] == "shared" else [out, weights]


def _exact_evict(st):
    c, lens = st["case"], _lengths(st["case"])
    B, Hkv, keep = c["batch"], c["kv_heads"], c["keep"]
    s = st["scores"].cpu().numpy().astype(np.float64)
    kept = np.full((B, Hkv, keep), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        if n <= keep:
            kept[b, :, :n] = np.arange(n)
            continue
        always = np.zeros(n, dtype=bool)
        always[:min(c["sink"], n)] = True
        always[max(0, n - c["recent"]):] = True
        free = np.flatnonzero(~always)
        room = keep - int(always.sum())
        for h in range(Hkv):
            best = free[np.lexsort((free, -s[b, h, free]))[:room]]
            kept[b, h] = np.sort(np.concatenate([np.flatnonzero(always), best]))
    index = torch.from_numpy(kept).to(DEV).long()
    k = torch.zeros((B, keep, Hkv, c["dim"]), dtype=torch.float64, device=DEV)
    v, scores = torch.zeros_like(k), torch.zeros((B, Hkv, keep), dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        m = min(n, keep)
        for h in range(Hkv):
            k[b, :m, h] = st["k"][b, index[b, h, :m], h].double()
            v[b, :m, h] = st["v"][b, index[b, h, :m], h].double()
            scores[b, h, :m] = st["scores"][b, h, index[b, h, :m]].double()
    return [k, v, scores, torch.from_numpy(kept).to(DEV), torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device=DEV)]


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "shared": _exact_decode, "scored": _exact_decode, "evict": _exact_evict}[case["kind"]](st)
