"""Generation behind a shared prefix: what its results must not depend on."""
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
