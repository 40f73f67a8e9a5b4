"""The launches of a generation step in 8-bit products without a GPU: model.Llama's step with recorders in the place of the kernels."""
import pytest
import torch

LAYER = ["rmsnorm_i8", "gemm_i8", "rope_positions", "attn_decode", "quantize_i8", "gemm_i8", "rmsnorm_i8", "gemm_i8", "quantize_i8", "gemm_i8"]


@pytest.fixture
def model(pkg, monkeypatch):
    """A Llama of two layers whose kernels are recorders, and their list of (entry, arguments, keyword arguments)."""
    from llm_infer_b200 import model as M
    calls = []

    def recorder(name, result):
        return lambda *args, **kwargs: (calls.append((name, args, kwargs)), result(args, kwargs))[1]

    monkeypatch.setattr(M.A, "embed_f16", recorder("embed_f16", lambda a, k: None))
    monkeypatch.setattr(M.A, "attn_decode", recorder("attn_decode", lambda a, k: k["out"]))
    monkeypatch.setattr(M.A, "argmax", recorder("argmax", lambda a, k: None))
    monkeypatch.setattr(M.X, "rope_positions", recorder("rope_positions", lambda a, k: k["q_out"]))
    monkeypatch.setattr(M.I, "rmsnorm_i8", recorder("rmsnorm_i8", lambda a, k: (k["out"], k["scale"])))
    monkeypatch.setattr(M.I, "quantize_i8", recorder("quantize_i8", lambda a, k: (k["out"], k["scale"])))
    monkeypatch.setattr(M.I, "gemm_i8", recorder("gemm_i8", lambda a, k: k["out"]))
    c = M.ModelConfig(dim=48, hidden_dim=80, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16, vocab_size=32, max_seq_len=300)
    m = M.Llama.__new__(M.Llama)
    z = torch.zeros
    m.cfg, m.batch, m.weight_type, m.kv_early, m.device = c, 3, "i8", True, torch.device("cpu")
    m._own_rope, m._inv_freq, m._rope_factor, m._rope_layout, m.workspace = True, None, 1.0, "interleaved", None
    m.w = {"embed": None, "rms_att": z(2, 48), "rms_ffn": z(2, 48), "rms_final": z(48)}
    m.wg = m.w
    m.w8 = {n: [(f"{n}{l}", f"scale of {n}{l}") for l in range(2)] for n in ("wqkv", "wo", "w13", "w2")}
    m.w8["wcls"] = ("wcls", "scale of wcls")
    m._rows8 = m._int8_rows(3)
    m.q, m.k, m.v = m._heads(m._rows8["qkv"])
    m.q_turned, m.att, m.x, m.logits = z(3, 4, 16), z(3, 4, 16), z(3, 48), z(3, 32)
    m.tokens, m.next_token, m.status, m.pos, m.kv_pos, m.kv_len = (z(3, dtype=torch.int32) for _ in range(6))
    m.k_cache, m.v_cache = z(2, 3), z(2, 3)
    return m, calls


@pytest.mark.parametrize("logits", [False, True])
def test_a_steps_launches(model, logits):
    m, calls = model
    m._launch_step(0, logits)
    assert [name for name, _, _ in calls] == ["embed_f16"] + 2 * LAYER + (["rmsnorm_i8", "gemm_i8", "argmax"] if logits else [])
    gemms = [(a[2], k) for name, a, k in calls if name == "gemm_i8"]
    assert [w for w, _ in gemms][:4] == ["wqkv0", "wo0", "w130", "w20"] and all(k["w_early"] for _, k in gemms)
    assert [bool(k.get("swiglu")) for w, k in gemms] == [w.startswith("w13") for w, _ in gemms]


def test_every_output_is_added_to_the_residual_stream_once(model):
    """The output and the down projection leave what the next norm adds; only the first norm has nothing to add."""
    m, calls = model
    m._launch_step(0, True)
    norms = [k for name, _, k in calls if name == "rmsnorm_i8"]
    assert [k.get("delta") is None for k in norms] == [True, False, False, False, False]
    assert all(k["delta"] is m._rows8["delta"] for k in norms[1:])


def test_attention_reads_the_turned_queries(model):
    m, calls = model
    m._launch_step(0, False)
    for name, args, kw in calls:
        if name == "rope_positions":
            assert args[0] is m.q and kw["q_out"] is m.q_turned
        if name == "attn_decode":
            assert args[0] is m.q_turned and kw["two_pass"]


def test_projections_outputs_are_views_of_one_buffer(model):
    m, _ = model
    m._rows8["qkv"].copy_(torch.arange(3 * 128).view(3, 128))
    assert m.q.shape == (3, 4, 16) and m.k.shape == m.v.shape == (3, 2, 16)
    assert float(m.q[1, 0, 0]) == 128 and float(m.k[1, 0, 0]) == 128 + 64 and float(m.v[1, 1, 15]) == 128 + 127
