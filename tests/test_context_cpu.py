"""Long-context operators without a device: what they refuse, the tables of scaled frequencies, the dealing of tiles."""
import ctypes as C
import math

import pytest
import torch


@pytest.fixture(scope="module")
def ctx(built_lib, pkg):
    from llm_infer_b200 import context
    return context


def _evict_args(b):
    a = b.AttnKvEvictArgs()
    for i, n in enumerate("k v k_out v_out scores scores_out kept kv_len_out".split()):
        setattr(a, n, (i + 1) << 20)
    a.batch, a.n_kv_heads, a.head_dim, a.rows, a.out_rows, a.keep = 1, 2, 64, 100, 50, 50
    return a


def _shared_args(b):
    a = b.AttnDecodeSharedArgs()
    for i, n in enumerate("o q k_prefix v_prefix k v workspace".split()):
        setattr(a, n, (i + 1) << 20)
    a.o_dtype = a.dtype = b.DTYPE_F16
    a.batch, a.n_heads, a.n_kv_heads, a.head_dim, a.prefix_len, a.kv_capacity = 2, 8, 2, 64, 10, 10
    a.kv_batch_stride = 10 * 2 * 64
    return a


def _rope_args(b):
    a = b.AttnRopePositionsArgs()
    for i, n in enumerate("q_out q k v k_cache v_cache inv_freq pos row seq".split()):
        setattr(a, n, (i + 1) << 20)
    a.tokens, a.n_heads, a.n_kv_heads, a.head_dim, a.n_seqs, a.cache_rows = 4, 8, 2, 64, 2, 10
    a.kv_batch_stride = 10 * 2 * 64
    a.in_dtype = a.q_out_dtype = a.kv_dtype = b.DTYPE_F16
    return a


@pytest.mark.parametrize("entry,make,changes,code", [
    ("attn_rope_positions", _rope_args, dict(inv_freq=None), -1),
    ("attn_rope_positions", _rope_args, dict(tokens=0), -1),
    ("attn_rope_positions", _rope_args, dict(rotary_dim=66), -1),
    ("attn_rope_positions", _rope_args, dict(rotary_dim=31), -1),
    ("attn_rope_positions", _rope_args, dict(head_dim=63), -1),
    ("attn_rope_positions", _rope_args, dict(layout=2), -1),
    ("attn_rope_positions", _rope_args, dict(in_dtype=3), -1),
    ("attn_rope_positions", _rope_args, dict(kv_dtype=0), -2),
    ("attn_rope_positions", _rope_args, dict(seq=None), -1),             # four tokens, two sequences
    ("attn_rope_positions", _rope_args, dict(kv_batch_stride=0), -1),
    ("attn_rope_positions", _rope_args, dict(kv_row_stride=64), -1),     # rows would overlap
    ("attn_rope_positions", _rope_args, dict(q=(2 << 20) + 1), -3),
    ("attn_decode_shared", _shared_args, dict(q=None), -1),
    ("attn_decode_shared", _shared_args, dict(k_prefix=None), -1),
    ("attn_decode_shared", _shared_args, dict(v=None), -1),
    ("attn_decode_shared", _shared_args, dict(n_heads=9), -1),
    ("attn_decode_shared", _shared_args, dict(batch=0), -1),
    ("attn_decode_shared", _shared_args, dict(dtype=0), -2),
    ("attn_decode_shared", _shared_args, dict(o_dtype=2), -2),           # bf16 out of fp16 inputs
    ("attn_decode_shared", _shared_args, dict(kv_batch_stride=0), -1),
    ("attn_decode_shared", _shared_args, dict(scores=8 << 20), -1),      # weights in, none out
    ("attn_decode_shared", _shared_args, dict(kv_row_stride=132), -3),
    ("attn_decode_shared", _shared_args, dict(prefix_row_stride=64), -1),
    ("attn_decode_shared", _shared_args, dict(k=(5 << 20) + 8), -3),
    ("attn_decode_shared", _shared_args, dict(scores_out=9 << 20, score_out_stride=9), -1),
    ("attn_kv_evict", _evict_args, dict(kept=None), -1),
    ("attn_kv_evict", _evict_args, dict(keep=0), -1),
    ("attn_kv_evict", _evict_args, dict(keep=51), -1),                   # more than the output caches hold
    ("attn_kv_evict", _evict_args, dict(sink=30, recent=21), -1),
    ("attn_kv_evict", _evict_args, dict(head_dim=60), -2),
    ("attn_kv_evict", _evict_args, dict(batch=2), -1),                   # no batch stride
    ("attn_kv_evict", _evict_args, dict(k=(1 << 20) + 2), -3),
    ("attn_kv_evict", _evict_args, dict(k_out=1 << 20), -1),             # K in place, V elsewhere
    ("attn_kv_evict", _evict_args, dict(k_out=(1 << 20) + 256), -1),     # overlap
    ("attn_kv_evict", _evict_args, dict(scores_out=(5 << 20) + 4), -1),
    ("attn_kv_evict", _evict_args, dict(k_out=1 << 20, v_out=2 << 20, scores_out=5 << 20), -1),  # in place with fewer rows
])
def test_refusals_of_the_c_abi(built_lib, pkg, entry, make, changes, code):
    a = make(pkg.binding)
    for name, value in changes.items():
        setattr(a, name, value)
    assert getattr(built_lib, entry)(C.byref(a), None) == code
    assert getattr(built_lib, entry)(None, None) == -1


def test_cpu_tensors_are_refused(ctx):
    q, kv = torch.zeros(1, 4, 64).half(), torch.zeros(1, 8, 2, 64).half()
    with pytest.raises(ValueError, match="CUDA"):
        ctx.attn_decode_shared(q, None, None, kv, kv.clone())
    with pytest.raises(ValueError, match="CUDA"):
        ctx.kv_evict(kv, kv.clone(), torch.zeros(1, 2, 8), None, 4)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ctx.rope_positions(q, kv[:, 0], kv[:, 0], kv, kv.clone(), i, i, inv_freq=torch.ones(32))


def test_rope_frequencies(ctx):
    base, factor = ctx.rope_frequencies(128, 500000.0)
    assert factor == 1.0 and base.dtype == torch.float32 and base.shape == (64,)
    for i in (0, 1, 31, 63):
        assert float(base[i]) == pytest.approx(500000.0 ** (-2 * i / 128), rel=2 ** -23)
    linear, _ = ctx.rope_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(linear, base / 4, rtol=2 ** -22, atol=0)
    ntk, _ = ctx.rope_frequencies(128, 500000.0, {"type": "ntk", "factor": 8.0})
    assert float(ntk[0]) == 1.0 and float(ntk[-1]) == pytest.approx(float(base[-1]) / 8, rel=1e-6)
    llama3, _ = ctx.rope_frequencies(128, 500000.0, {"type": "llama3", "factor": 8.0, "original": 8192})
    wave = 2 * math.pi / base.double()
    assert torch.equal(llama3[wave < 8192 / 4], base[wave < 8192 / 4])
    assert torch.allclose(llama3[wave > 8192], base[wave > 8192] / 8, rtol=2 ** -22, atol=0)
    between = (wave >= 8192 / 4) & (wave <= 8192)
    assert between.any() and ((llama3 <= base) & (llama3 >= base / 8 * (1 - 1e-6)))[between].all()
    yarn, factor = ctx.rope_frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0, "original": 4096})
    base = ctx.rope_frequencies(64, 10000.0)[0]
    turns = 4096 * base.double() / (2 * math.pi)
    assert factor == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert torch.equal(yarn[turns > 34], base[turns > 34])
    assert torch.allclose(yarn[turns < 0.7], base[turns < 0.7] / 16, rtol=2 ** -22, atol=0)
    assert (yarn[1:] < yarn[:-1]).all()
    for bad in ({"type": "dynamic", "factor": 2.0}, {"type": "linear", "factor": 0.5}, {"type": "llama3", "factor": 2.0, "original": 1, "high_freq_factor": 1.0}):
        with pytest.raises(ValueError):
            ctx.rope_frequencies(64, 10000.0, bad)
    with pytest.raises(ValueError):
        ctx.rope_frequencies(63, 10000.0)


def test_the_mirrors_of_the_argument_structures_have_the_librarys_sizes(built_lib, pkg):
    b = pkg.binding
    for index, mirror in ((10, b.AttnRopePositionsArgs), (11, b.AttnDecodeSharedArgs), (12, b.AttnKvEvictArgs)):
        assert built_lib.attn_abi_struct_size(index) == C.sizeof(mirror)


def test_packed_arguments_lie_where_the_mirrors_have_them(ctx, pkg):
    b = pkg.binding
    for packer, mirror in ((ctx.ROPE_ARGS, b.AttnRopePositionsArgs), (ctx.SHARED_ARGS, b.AttnDecodeSharedArgs), (ctx.EVICT_ARGS, b.AttnKvEvictArgs)):
        assert packer.size == C.sizeof(mirror)
        fields = mirror._fields_
        values = [float(i + 1) if kind is C.c_float else i + 1 for i, (_, kind) in enumerate(fields)]
        got = mirror.from_buffer_copy(packer.pack(*values))
        assert [getattr(got, name) for name, _ in fields] == values
