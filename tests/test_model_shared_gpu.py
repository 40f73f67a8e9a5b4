"""Generation behind a shared prefix, with scaled positions and with evicting caches, against the forward pass in 64 bits.

The model is small and random; the definition below runs one token of one sequence at a time over lists of keys and values. Logits
are compared as in the other model tests (2e-3 + 1e-2 of the row's RMS: fp16 caches and queries), tokens where the definition's own
top-2 margin exceeds twice that bound."""
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


class Definition:
    """One sequence: feed(token, position) -> logits. Own caches per layer and kv head as lists of (k, v, weight)."""

    def __init__(self, cfg, weights, inv_freq, factor, layout):
        self.c = cfg
        self.w = {k: v.double() for k, v in weights.items()}
        self.f, self.factor, self.layout = inv_freq.double(), factor, layout
        self.prefix = [[[] for _ in range(cfg.n_kv_heads)] for _ in range(cfg.n_layers)]
        self.own = [[[] for _ in range(cfg.n_kv_heads)] for _ in range(cfg.n_layers)]

    def _rotate(self, x, pos):
        a = pos * self.f
        c, s = torch.cos(a) * self.factor, torch.sin(a) * self.factor
        y, R = x.clone(), 2 * len(self.f)
        i0, i1 = (slice(0, R // 2), slice(R // 2, R)) if self.layout == "half" else (slice(0, R, 2), slice(1, R, 2))
        y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
        return y

    def feed(self, token, pos, into_prefix=False):
        c, w = self.c, self.w
        norm = lambda x, g: x / torch.sqrt((x * x).mean() + c.norm_eps) * g  # noqa: E731
        x = w["embed"][token]
        for l in range(c.n_layers):
            h = norm(x, w["rms_att"][l])
            q = self._rotate((w["wq"][l] @ h).view(c.n_heads, -1), pos)
            k = self._rotate((w["wk"][l] @ h).view(c.n_kv_heads, -1), pos)
            v = (w["wv"][l] @ h).view(c.n_kv_heads, -1)
            G, out = c.n_heads // c.n_kv_heads, []
            for g in range(c.n_kv_heads):
                (self.prefix if into_prefix else self.own)[l][g].append([k[g], v[g], 0.0])
                rows = self.prefix[l][g] + self.own[l][g]
                s = q[g * G:(g + 1) * G] @ torch.stack([r[0] for r in rows]).T / math.sqrt(c.head_dim)
                p = torch.softmax(s, 1)
                out.append(p @ torch.stack([r[1] for r in rows]))
                for r, weight in zip(rows, p.sum(0)):
                    r[2] += float(weight)
            x = x + w["wo"][l] @ torch.cat(out).view(-1)
            h = norm(x, w["rms_ffn"][l])
            gate = w["w1"][l] @ h
            x = x + w["w2"][l] @ (gate * torch.sigmoid(gate) * (w["w3"][l] @ h))
        return w["wcls"] @ norm(x, w["rms_final"])


def _check(tokens, logits, want):
    """False once the two may legitimately have picked different tokens."""
    bound = 2e-3 + 1e-2 * float(want.pow(2).mean().sqrt())
    assert (logits.double() - want).abs().max() <= bound
    top = torch.sort(want).values
    if float(top[-1] - top[-2]) > 2 * bound:
        assert int(tokens) == int(want.argmax())
    return int(tokens) == int(want.argmax())


CASES = [("interleaved", None, 40, (5, 9, 1)), ("half", {"type": "llama3", "factor": 8.0, "original": 64}, 33, (3, 1)),
         ("half", {"type": "yarn", "factor": 4.0, "original": 64}, 1, (7,)),
         ("interleaved", {"type": "linear", "factor": 2.0}, 70, (2, 2, 6, 4, 11))]


@pytest.mark.parametrize("layout,scaling,P,lens", CASES)
def test_generation_behind_a_shared_prefix(M, layout, scaling, P, lens):
    cfg = _config(M)
    w = M.random_weights(cfg, 5)
    rng = np.random.default_rng(P)
    prefix = rng.integers(0, cfg.vocab_size, P).tolist()
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in lens]
    llama = M.Llama(cfg, w, batch=len(prompts), rope_layout=layout, rope_scaling=scaling)
    tokens, logits = llama.generate_shared(prefix, prompts, 6, want_logits=True)
    again = llama.generate_shared(llama.encode_prefix(prefix), prompts, 6)
    assert torch.equal(tokens, again)
    from llm_infer_b200 import context
    inv_freq, factor = context.rope_frequencies(cfg.head_dim, cfg.rope_theta, scaling)
    for b, prompt in enumerate(prompts):
        d = Definition(cfg, w, inv_freq, factor, layout)
        for i, t in enumerate(prefix):
            d.feed(t, i, into_prefix=True)
        for i, t in enumerate(prompt):
            want = d.feed(t, P + i)
        for i in range(6):
            if not _check(tokens[b, i], logits[b, i], want):
                break
            want = d.feed(int(tokens[b, i]), P + len(prompt) + i)


@pytest.mark.parametrize("layout,scaling", [("half", {"type": "ntk", "factor": 4.0}), ("interleaved", None)])
def test_every_other_path_has_the_scaled_positions_too(M, layout, scaling):
    """prefill, token-at-a-time steps and the captured step of one model agree with the definition."""
    cfg = _config(M)
    w = M.random_weights(cfg, 6)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in (12, 30)]
    from llm_infer_b200 import context
    inv_freq, factor = context.rope_frequencies(cfg.head_dim, cfg.rope_theta, scaling)
    for mode in ("batched", "token"):
        llama = M.Llama(cfg, w, batch=2, rope_layout=layout, rope_scaling=scaling)
        if mode == "token":
            llama.capture()
        tokens, logits = llama.generate(prompts, 4, want_logits=True, prompt_mode=mode)
        for b, prompt in enumerate(prompts):
            d = Definition(cfg, w, inv_freq, factor, layout)
            for i, t in enumerate(prompt):
                want = d.feed(t, i)
            for i in range(4):
                if not _check(tokens[b, i], logits[b, i], want):
                    break
                want = d.feed(int(tokens[b, i]), len(prompt) + i)


def test_generation_under_a_cache_budget(M, monkeypatch):
    """Eviction every few tokens. The definition follows the rows that were kept, after checking that they are the right ones: the sink,
    the recent rows, and no evicted row with a larger weight than a kept one (weights within 1e-3 of the definition's count as equal)."""
    from llm_infer_b200 import context
    cfg = _config(M)
    w = M.random_weights(cfg, 7)
    rng = np.random.default_rng(2)
    P, lens, budget, every, sink, recent = 25, (13, 20), 16, 5, 2, 6
    prefix = rng.integers(0, cfg.vocab_size, P).tolist()
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in lens]
    calls = []
    evict = context.kv_evict

    def recorded(k, v, scores, kv_len, keep, **kw):
        before = kv_len.tolist()
        kept, after = evict(k, v, scores, kv_len, keep, **kw)
        calls.append((before, kept.cpu().clone(), after.tolist()))
        return kept, after

    monkeypatch.setattr(context, "kv_evict", recorded)
    n_new = 9
    llama = M.Llama(cfg, w, batch=2)
    tokens, logits = llama.generate_shared(prefix, prompts, n_new, budget=budget, evict_every=every, sink=sink, recent=recent, want_logits=True)
    assert len(calls) >= 2 * cfg.n_layers and len(calls) % cfg.n_layers == 0
    rounds = [calls[i:i + cfg.n_layers] for i in range(0, len(calls), cfg.n_layers)]
    assert all(max(r[0][0]) == budget + every and max(r[0][2]) <= budget for r in rounds)
    inv_freq, factor = context.rope_frequencies(cfg.head_dim, cfg.rope_theta)
    longest = max(lens)
    for b, prompt in enumerate(prompts):
        d = Definition(cfg, w, inv_freq, factor, "interleaved")
        for i, t in enumerate(prefix):
            d.feed(t, i, into_prefix=True)
        held, pending, same = 0, list(rounds), True
        for step in range(longest + n_new - 1):
            if pending and max(pending[0][0][0]) == budget + every and _at(step, lens, budget, every, len(rounds) - len(pending)):
                before = pending[0][0][0][b]
                for l, (_, kept, _) in enumerate(pending.pop(0)):
                    if step <= longest - len(prompt):
                        continue  # this sequence has not started
                    assert before == held
                    for h in range(cfg.n_kv_heads):
                        rows = [r for r in kept[b, h].tolist() if r >= 0]
                        own = d.own[l][h]
                        assert rows == sorted(set(rows)) and len(rows) == min(held, budget)
                        if held > budget:
                            assert rows[:sink] == list(range(sink)) and rows[-recent:] == list(range(held - recent, held))
                            free = set(range(sink, held - recent))
                            out_rows = free - set(rows)
                            worst = min(own[r][2] for r in free & set(rows))
                            assert all(own[r][2] <= worst + 2e-3 for r in out_rows)
                        d.own[l][h] = [own[r] for r in rows]
                held = min(held, budget)
            i = step - (longest - len(prompt))
            if i < 0:
                continue
            token = prompt[i] if i < len(prompt) else int(tokens[b, i - len(prompt)])
            want = d.feed(token, P + i)
            held += 1
            if i >= len(prompt) - 1 and not _check(tokens[b, i - len(prompt) + 1], logits[b, i - len(prompt) + 1], want):
                same = False
                break
        assert same or step > longest  # (a near-tie may end the comparison, but not before the first evictions)


def _at(step, lens, budget, every, done):
    """Whether the eviction numbered `done` happens in front of `step`: the fullest cache holds budget + every rows there."""
    longest = max(lens)
    held = [0] * len(lens)
    n = 0
    for s in range(step + 1):
        if max(held) == budget + every:
            if n == done:
                return s == step
            n += 1
            held = [min(x, budget) for x in held]
        held = [0 if s <= longest - len_ else x for x, len_ in zip(held, lens)]
        held = [x + 1 for x in held]
    return False


def test_refusals(M):
    cfg = _config(M)
    llama = M.Llama(cfg, M.random_weights(cfg, 5), batch=1)
    for bad in (dict(prompts=[[]]), dict(prompts=[[1], [2]]), dict(prefix=[]), dict(n_new=200), dict(budget=8, recent=6), dict(budget=8, evict_every=0)):
        with pytest.raises(ValueError):
            llama.generate_shared(**{**dict(prefix=[1, 2], prompts=[[3]], n_new=20), **bad})
    with pytest.raises(ValueError):
        M.Llama(_config(M, qkv_clip=1.0), M.random_weights(cfg, 5), batch=1, rope_layout="half")
