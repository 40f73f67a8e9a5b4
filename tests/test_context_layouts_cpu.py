"""What the long-context operators make of their operands' layouts, without a device: tensors of the host stand in, and what would be
handed to the library is looked at instead."""
import types

import pytest
import torch


@pytest.fixture
def ctx(built_lib, pkg, monkeypatch):
    from llm_infer_b200 import context
    calls = []
    monkeypatch.setattr(context, "_one_device", lambda *tensors: 0)
    monkeypatch.setattr(context, "_enqueue", lambda entry, index, stream, packed: calls.append((entry, packed)))
    return types.SimpleNamespace(context=context, calls=calls)


B, T, HKV, D = 2, 6, 3, 64


def _cache(b=B, t=T):
    return torch.zeros((b, t, HKV, D), dtype=torch.float16)


def _one_row(b=B, t=T):  # every row of a sequence is the same memory
    return torch.zeros((b, 1, HKV, D), dtype=torch.float16).expand(b, t, HKV, D)


def _scores(kind, b=B, t=T):
    return {"heads": lambda: torch.zeros((b, 1, t)).expand(b, HKV, t),
            "all": lambda: torch.zeros(t).expand(b, HKV, t),
            "sequences": lambda: torch.zeros((1, HKV, t)).expand(b, HKV, t),
            "overlapping": lambda: torch.zeros(t + b * HKV).as_strided((b, HKV, t), (HKV, 1, 1))}[kind]()


def _decode(ctx, b=B, k=None, v=None, prefix=None, scores=None, scores_out=None):
    q = torch.zeros((b, 6, D), dtype=torch.float16)
    k = _cache(b) if k is None else k
    ws = types.SimpleNamespace(key=(b, 6, HKV, D, 0), rows=T, ptr=1 << 20, nbytes=1 << 20, status_ptr=0)
    return ctx.context.attn_decode_shared(q, prefix, prefix, k, k if v is None else v, scores=scores, scores_out=scores_out, workspace=ws)


@pytest.mark.parametrize("kind,batch", [("heads", 1), ("heads", 2), ("all", 1), ("all", 2), ("sequences", 2), ("overlapping", 1), ("overlapping", 2)])
def test_scores_whose_runs_share_memory_are_refused(ctx, kind, batch):
    k = _cache(batch)
    with pytest.raises(ValueError, match="scores"):
        ctx.context.kv_evict(k, k.clone(), _scores(kind, batch), None, 3)
    with pytest.raises(ValueError, match="scores"):
        ctx.context.kv_evict(k, k.clone(), torch.zeros((batch, HKV, T)), None, 3, out=(_cache(batch, 4), _cache(batch, 4), _scores(kind, batch, 4)))
    with pytest.raises(ValueError, match="scores"):
        _decode(ctx, batch, scores=_scores(kind, batch))
    with pytest.raises(ValueError, match="scores"):
        _decode(ctx, batch, scores=_scores(kind, batch), scores_out=torch.zeros((batch, HKV, T)))
    with pytest.raises(ValueError, match="scores"):
        _decode(ctx, batch, scores_out=_scores(kind, batch))
    assert not ctx.calls


@pytest.mark.parametrize("make", [_one_row, lambda b=B, t=T: torch.zeros(b * T * HKV * D, dtype=torch.float16).as_strided((b, t, HKV, D), (T * HKV * D, D, D, 1))],
                         ids=["one row", "overlapping rows"])
def test_caches_and_prefixes_whose_rows_share_memory_are_refused(ctx, make):
    f16 = torch.float16
    with pytest.raises(ValueError, match="row"):
        _decode(ctx, k=make())
    with pytest.raises(ValueError, match="row"):
        _decode(ctx, 1, k=make(1))
    with pytest.raises(ValueError, match="row"):
        _decode(ctx, prefix=make(1)[0])
    s = torch.zeros((B, HKV, T))
    with pytest.raises(ValueError, match="row"):
        ctx.context.kv_evict(make(), make(), s, None, 3)
    with pytest.raises(ValueError, match="row"):
        ctx.context.kv_evict(make(), make(), s, None, 3, out=(_cache(t=4), _cache(t=4), torch.zeros((B, HKV, 4))))
    with pytest.raises(ValueError, match="row"):
        ctx.context.kv_evict(_cache(), _cache(), s, None, 3, out=(make(t=4), make(t=4), torch.zeros((B, HKV, 4))))
    i = torch.zeros(B, dtype=torch.int32)
    with pytest.raises(ValueError, match="row"):
        ctx.context.rope_positions(torch.zeros((B, 6, D), dtype=f16), torch.zeros((B, HKV, D), dtype=f16), torch.zeros((B, HKV, D), dtype=f16),
                                   make(), make(), i, i, inv_freq=torch.ones(D // 2))
    assert not ctx.calls


def test_a_single_run_or_row_may_have_any_stride(ctx):
    """Strides of dimensions of one element mean nothing: such operands are taken, their strides are not."""
    odd = torch.zeros(4 * HKV * D, dtype=torch.float16).as_strided((1, 1, HKV, D), (0, 0, D, 1))
    ctx.context.kv_evict(odd, odd.clone().as_strided((1, 1, HKV, D), (0, 0, D, 1)), torch.zeros((1, HKV, 1)), None, 1)
    _decode(ctx, 1, k=odd, prefix=odd[0])
    _decode(ctx, 1, scores=torch.zeros((1, HKV, T)).as_strided((1, HKV, T), (0, T, 1)))
    q, kv, i = torch.zeros((1, 6, D), dtype=torch.float16), torch.zeros((1, HKV, D), dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    ctx.context.rope_positions(q, kv, kv, odd, odd, i, i, inv_freq=torch.ones(D // 2))
    assert [entry for entry, _ in ctx.calls] == ["attn_kv_evict", "attn_decode_shared", "attn_decode_shared", "attn_rope_positions"]
