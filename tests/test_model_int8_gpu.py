"""Llama(weight_type="i8"): the whole forward pass in 8-bit products against a plain one, and its paths against each other.

How far two correct runs may be apart: a row's step is max|y| / 127, about 0.03 of its root mean square. Values that differ a little ahead of
a rounding (order of the attention's sums, queries in fp16) land on neighbouring steps here and there; at worst the two roundings
are independent, which is step^2 / 6 in the mean square, 1.2 % of the row. Nine roundings lie in a row in two layers and the classifier,
the gated product doubles what reaches it: sqrt(9) x 1.2 % x 2 = 7.4 % of the logits' norm. A missing or misplaced step is of order one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
FAR = 0.075


@pytest.fixture(scope="module")
def M(built_lib, pkg):
    from llm_infer_b200 import model
    return model


def _config(M, **kw):
    return M.ModelConfig(**{**dict(dim=512, hidden_dim=1000, n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, vocab_size=1003,
                                   max_seq_len=64, norm_eps=1e-5, rope_theta=10000.0), **kw})


def _rows8(y):
    """The value of a row in 8 bits, in 64 bits."""
    scale = y.abs().amax(-1, keepdim=True) / 127.0
    return torch.round(y / scale.clamp_min(1e-300)) * scale


def plain_logits(c, w, tokens, half_layout=False):
    """Logits of every token of one sequence, from the definition (weights fp16 on the host)."""
    w = {k: v.double() for k, v in w.items()}
    D, H, G, n = c.head_dim, c.n_heads, c.n_heads // c.n_kv_heads, len(tokens)

    def norm(x, weight):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + c.norm_eps) * weight

    def product(y, matrix):
        return _rows8(y) @ _rows8(matrix).t()

    angle = torch.arange(n, dtype=torch.float64)[:, None] * c.rope_theta ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = (x[..., :D // 2], x[..., D // 2:]) if half_layout else (x[..., 0::2], x[..., 1::2])
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-2 if half_layout else -1)
        return y.reshape(x.shape)

    x = w["embed"][tokens]
    mask = torch.full((n, n), -torch.inf, dtype=torch.float64).triu(1)
    for l in range(c.n_layers):
        qkv = product(norm(x, w["rms_att"][l]), torch.cat([w["wq"][l], w["wk"][l], w["wv"][l]]))
        q, k, v = qkv.split([H * D, H // G * D, H // G * D], 1)
        q, k, v = turn(q.view(n, H, D)), turn(k.reshape(n, -1, D)).half().double(), v.reshape(n, -1, D).half().double()
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) / D ** 0.5 + mask, -1)
        x = x + product(torch.einsum("hij,jhd->ihd", p, v).reshape(n, H * D), w["wo"][l])
        gate, up = product(norm(x, w["rms_ffn"][l]), torch.cat([w["w1"][l], w["w3"][l]])).split(c.hidden_dim, 1)
        x = x + product(gate * torch.sigmoid(gate) * up, w["w2"][l])
    return product(norm(x, w["rms_final"]), w["wcls"])


def _apart(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float(((a - b).norm(dim=-1) / b.norm(dim=-1)).max())


@pytest.mark.parametrize("batch", [1, 3, 12])
@pytest.mark.parametrize("kw", [{}, dict(head_dim=128, n_heads=4, n_kv_heads=4, dim=384, hidden_dim=777), dict(vocab_size=257, n_layers=1)])
@pytest.mark.parametrize("mode", ["token", "batched"])
def test_logits_of_every_path_are_the_plain_models(M, batch, kw, mode):
    """A ragged batch, more sequences than the GEMVs of other weight types take among them; widths that are no multiples of 16."""
    c = _config(M, **kw)
    w = M.random_weights(c, seed=3)
    rng = np.random.default_rng(batch)
    prompts = [rng.integers(0, c.vocab_size, size=int(n)).tolist() for n in rng.integers(1, 20, size=batch)]
    llama = M.Llama(c, w, batch=batch, weight_type="i8")
    tokens, logits = llama.generate(prompts, 6, want_logits=True, prompt_mode=mode)
    for b, prompt in enumerate(prompts):
        want = plain_logits(c, w, prompt + tokens[b].tolist())
        assert _apart(logits[b], want[len(prompt) - 1:len(prompt) + 5]) < FAR
        assert torch.equal(logits[b].argmax(-1).int(), tokens[b])


def test_a_captured_step_gives_the_same_bits(M):
    c = _config(M)
    w = M.random_weights(c, seed=4)
    prompts = [[5, 6, 7], [900], list(range(20, 41))]
    runs = []
    for capture in (False, True):
        llama = M.Llama(c, w, batch=3, weight_type="i8")
        if capture:
            llama.capture()
        runs.append([llama.generate(prompts, 8, want_logits=True, prompt_mode=mode) for mode in ("token", "batched", "token")])
    for a, b in zip(*runs):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(runs[0][0][1], runs[0][2][1])


def test_scaled_and_half_paired_positions(M):
    c = _config(M)
    w = M.random_weights(c, seed=5)
    prompts = [[5, 6, 7, 8, 9], [900, 3]]
    llama = M.Llama(c, w, batch=2, weight_type="i8", rope_layout="half")
    for mode in ("token", "batched"):
        tokens, logits = llama.generate(prompts, 5, want_logits=True, prompt_mode=mode)
        for b, prompt in enumerate(prompts):
            want = plain_logits(c, w, prompt + tokens[b].tolist(), half_layout=True)
            assert _apart(logits[b], want[len(prompt) - 1:len(prompt) + 4]) < FAR


@pytest.mark.parametrize("budget", [0, 16])
def test_generation_behind_a_shared_prefix(M, budget):
    c = _config(M)
    w = M.random_weights(c, seed=6)
    rng = np.random.default_rng(1)
    prefix = rng.integers(0, c.vocab_size, size=33).tolist()
    prompts = [rng.integers(0, c.vocab_size, size=n).tolist() for n in (4, 1, 9)]
    llama = M.Llama(c, w, batch=3, weight_type="i8")
    tokens, logits = llama.generate_shared(prefix, prompts, 10, budget=budget, want_logits=True, evict_every=4)
    for b, prompt in enumerate(prompts):
        last = 10 if budget == 0 else max(0, budget - len(prompt))  # (up to the first eviction)
        want = plain_logits(c, w, prefix + prompt + tokens[b].tolist())[len(prefix) + len(prompt) - 1:]
        assert _apart(logits[b, :min(last, 10)], want[:min(last, 10)]) < FAR


def test_gguf_files_and_refusals(M, pkg, tmp_path):
    from llm_infer_b200 import gguf
    c = _config(M, hidden_dim=1024, vocab_size=512)
    path = str(tmp_path / "m.gguf")
    w = M.random_weights(c, seed=7)
    gguf.write_gguf(path, c, {k: v.numpy() for k, v in w.items()})
    prompts = [[1, 2, 3], [4]]
    a = M.Llama.from_gguf(path, 2, int8=True).generate(prompts, 4, want_logits=True)
    b = M.Llama(c, w, 2, weight_type="i8").generate(prompts, 4, want_logits=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError, match="clamp"):
        M.Llama(_config(M, qkv_clip=8.0), M.random_weights(c, seed=7), 1, weight_type="i8")
    llama = M.Llama(_config(M, max_seq_len=16), M.random_weights(_config(M), seed=7), 1, weight_type="i8")
    with pytest.raises(ValueError, match="slide"):
        llama.generate([[1, 2, 3]], 15)
    with pytest.raises(ValueError, match="weight embed"):
        M.Llama(c, M.random_weights(c, seed=7, weight_type="q8_0"), 1, weight_type="i8")
    q8 = str(tmp_path / "q8.gguf")
    gguf.write_gguf(q8, c, {k: v.numpy() for k, v in M.random_weights(c, seed=7, weight_type="q8_0").items()}, weight_type="q8_0")
    with pytest.raises(ValueError, match="F16"):
        M.Llama.from_gguf(q8, 1, int8=True)
