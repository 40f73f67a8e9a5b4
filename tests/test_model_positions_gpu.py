"""Generation behind a shared prefix: what its results must not depend on, and the angles of its rows."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M(built_lib, pkg):
    from llm_infer_b200 import model
    return model


def _config(M, **kw):
    return M.ModelConfig(**{**dict(dim=512, hidden_dim=1024, n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, vocab_size=500,
                                   max_seq_len=160, rope_theta=10000.0), **kw})


# the last: many sequences behind a long prefix, whose kernel had 128 CTAs when few tokens were asked for and 100 for many
@pytest.mark.parametrize("P,B,n_heads,most,budget", [(1, 3, 8, 130, 0), (70, 3, 8, 130, 0), (70, 3, 8, 130, 16), (16000, 8, 32, 900, 0)])
def test_results_do_not_depend_on_how_many_tokens_are_asked_for(M, P, B, n_heads, most, budget):
    cfg = _config(M, n_heads=n_heads, n_layers=1, max_seq_len=most + 30)
    w = M.random_weights(cfg, 5)
    rng = np.random.default_rng(P)
    prefix = rng.integers(0, cfg.vocab_size, P).tolist()
    prompts = [rng.integers(0, cfg.vocab_size, 1 + i % 9).tolist() for i in range(B)]
    llama = M.Llama(cfg, w, batch=B)
    prefix = llama.encode_prefix(prefix)
    kw = dict(budget=budget, evict_every=5, sink=2, want_logits=True)
    tokens, logits = llama.generate_shared(prefix, prompts, most, **kw)
    for n in (1, 3, 12, 50):
        few, few_logits = llama.generate_shared(prefix, prompts, n, **kw)
        assert torch.equal(few, tokens[:, :n]) and torch.equal(few_logits, logits[:, :n])


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}])
def test_keys_of_a_long_prefix_are_turned_by_the_angles_of_the_own_rows(M, scaling):
    """Late positions of layer 0 against 64-bit angles: fp16 rounding of the keys (2^-11) and what the projection's sums of 512 products may
    be off by, 64 instructions that cut off 2^-23 of the products' magnitudes each. An angle whose product was rounded to fp32 is off
    by up to 2^-8 here."""
    cfg = _config(M, n_layers=1)
    w = M.random_weights(cfg, 9)
    from llm_infer_b200 import context
    P = 65536 + 3
    tokens = np.random.default_rng(3).integers(0, cfg.vocab_size, P)
    llama = M.Llama(cfg, w, batch=1, rope_scaling=scaling)
    k, _ = llama.encode_prefix(tokens.tolist())
    f, factor = context.rope_frequencies(cfg.head_dim, cfg.rope_theta, scaling)
    at = torch.arange(P - 2000, P)
    x = w["embed"].cpu().double()[torch.from_numpy(tokens)[at]]
    x = x / torch.sqrt((x * x).mean(1, keepdim=True) + cfg.norm_eps) * w["rms_att"][0].cpu().double()
    wk = w["wk"][0].cpu().double().T
    y, size = ((p @ q).view(len(at), cfg.n_kv_heads, cfg.head_dim // 2, 2) for p, q in ((x, wk), (x.abs(), wk.abs())))
    a = at.double()[:, None] * f.double()[None]
    c, s = (torch.cos(a) * factor)[:, None], (torch.sin(a) * factor)[:, None]
    want = torch.stack([y[..., 0] * c - y[..., 1] * s, y[..., 0] * s + y[..., 1] * c], -1)
    size = size.sum(-1, keepdim=True) * factor
    got = k[0, at.to(k.device)].double().cpu().view(want.shape)
    assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -17 * size).all())


def test_models_that_clamp_q_k_and_v_agree_with_the_ordinary_path(M):
    cfg = _config(M, qkv_clip=0.75)
    w = M.random_weights(cfg, 4)
    rng = np.random.default_rng(8)
    prefix = rng.integers(0, cfg.vocab_size, 40).tolist()
    prompts = [rng.integers(0, cfg.vocab_size, 6).tolist() for _ in range(2)]
    llama = M.Llama(cfg, w, batch=2)
    tokens, logits = llama.generate_shared(prefix, prompts, 5, want_logits=True)
    want_tokens, want = llama.generate([prefix + p for p in prompts], 5, want_logits=True)
    for b in range(2):
        for i in range(5):
            bound = 2e-3 + 1e-2 * float(want[b, i].pow(2).mean().sqrt())
            assert float((logits[b, i] - want[b, i]).abs().max()) <= bound
            if int(tokens[b, i]) != int(want_tokens[b, i]):
                top = torch.sort(want[b, i]).values
                assert float(top[-1] - top[-2]) <= 2 * bound
                break


def test_scaled_positions_past_the_cache_are_refused_before_anything_runs(M):
    cfg = _config(M)
    w = M.random_weights(cfg, 5)
    with pytest.raises(ValueError, match="layout"):
        M.Llama(cfg, w, batch=1, rope_layout="halves")
    for mode in ("token", "batched"):
        llama = M.Llama(cfg, w, batch=1, rope_layout="half")
        launches = M.X._b.load().attn_kernel_launch_count()
        with pytest.raises(ValueError, match="slide"):
            llama.generate([[1, 2, 3]], cfg.max_seq_len - 1, prompt_mode=mode)  # the last token's position is max_seq_len
        with pytest.raises(ValueError, match="slide"):
            llama.forward(torch.tensor([1], dtype=torch.int32), cfg.max_seq_len)
        assert M.X._b.load().attn_kernel_launch_count() == launches
    assert llama.generate([[1, 2, 3]], cfg.max_seq_len - 2, prompt_mode="token").shape == (1, cfg.max_seq_len - 2)
    assert math.isfinite(float(llama.logits.sum()))
