"""Which operands of an eviction may lie how in memory, by what the C entry answers without a device: ATTN_ERR_INVALID_ARG (-1) for
operands that share bytes where they must not, and something else (no device here) for those that do not."""
import ctypes as C
import random

import pytest
import torch

no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: calls that are accepted must not be launched")
INVALID = -1
NAMES = "k v k_out v_out scores scores_out kept kv_len kv_len_out".split()


def _args(b, **kw):
    """K, V [2, 6, 2, 8] and outputs [2, 4, 2, 8], all dense and far apart; keep = 4."""
    a = b.AttnKvEvictArgs()
    for i, n in enumerate(NAMES):
        setattr(a, n, (i + 1) << 20)
    a.batch, a.n_kv_heads, a.head_dim, a.rows, a.out_rows, a.keep = 2, 2, 8, 6, 4, 4
    a.kv_batch_stride, a.out_batch_stride = 6 * 16, 4 * 16
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def _code(lib, a):
    return lib.attn_kv_evict(C.byref(a), None)


def _bytes(base, batch, batch_stride, rows, row_stride, width):
    return {base + 2 * (b * batch_stride + t * row_stride + i) for b in range(batch) for t in range(rows) for i in range(width)}


@no_device
@pytest.mark.parametrize("seed", range(8))
def test_caches_are_refused_exactly_when_they_share_bytes(built_lib, pkg, seed):
    """Inputs and outputs of one buffer with the same strides in every interleaving: sequences, rows or both."""
    rng = random.Random(seed)
    seen = {True: 0, False: 0}
    for _ in range(400):
        batch, rows = rng.choice([1, 2, 3]), rng.choice([1, 2, 4])
        width = 16
        row_stride = width * rng.choice([1, 2, 3, 4])
        batch_stride = row_stride * rows * rng.choice([1, 2, 3]) + width * rng.choice([0, 0, 1])
        if rng.random() < 0.3 and batch > 1:  # rows outermost
            batch_stride, row_stride = width * rng.choice([1, 2, 4]), width * rng.choice([1, 2, 4]) * 4 * batch
        base = [(1 << 20) + 2 * 8 * rng.randrange(0, 60) for _ in range(4)]
        sets = [_bytes(p, batch, batch_stride, rows, row_stride, width) for p in base]
        a = _args(pkg.binding, batch=batch, rows=rows, out_rows=rows, keep=rows, kv_row_stride=row_stride, out_row_stride=row_stride,
                  kv_batch_stride=batch_stride, out_batch_stride=batch_stride, k=base[0], v=base[1], k_out=base[2], v_out=base[3],
                  **{n: (i + 8) << 20 for i, n in enumerate(NAMES[4:])})
        # (inputs may share, and the three in place may be the outputs, but then with the scores in place too)
        wrong = any(not sets[i].isdisjoint(sets[j]) for i in (0, 1) for j in (2, 3))
        between_outputs = not sets[2].isdisjoint(sets[3])
        if between_outputs and not wrong:
            continue
        seen[wrong] += 1
        assert (_code(built_lib, a) == INVALID) == wrong, (batch, rows, batch_stride, row_stride, base)
    assert min(seen.values()) > 30


@no_device
def test_scores_of_one_buffer_may_interleave(built_lib, pkg):
    b, at = pkg.binding, 19 << 20
    both = dict(score_stride=10, score_out_stride=10)
    assert _code(built_lib, _args(b, scores=at, scores_out=at + 4 * 6, **both)) != INVALID
    assert _code(built_lib, _args(b, scores=at, scores_out=at + 4 * 5, **both)) == INVALID
    assert _code(built_lib, _args(b, scores=at, scores_out=at + 4 * 7, **both)) == INVALID  # its fourth column is the next run's first
    assert _code(built_lib, _args(b, scores=at + 4 * 4, scores_out=at, **both)) != INVALID


@no_device
def test_outputs_may_not_share_memory_with_each_other_or_with_what_is_read(built_lib, pkg):
    """A CTA would read or write what another one writes."""
    b = pkg.binding
    cache, scores, kept, lens = 2 * 4 * 16 * 2, 2 * 2 * 4 * 4, 2 * 2 * 4 * 4, 2 * 4  # bytes of the outputs
    assert _code(built_lib, _args(b)) != INVALID
    at = lambda name: (NAMES.index(name) + 1) << 20  # noqa: E731
    sizes = dict(k=2 * 6 * 16 * 2, v=2 * 6 * 16 * 2, scores=2 * 2 * 6 * 4, kv_len=lens, k_out=cache, v_out=cache, scores_out=scores, kept=kept, kv_len_out=lens)
    written = ["k_out", "v_out", "scores_out", "kept", "kv_len_out"]
    for i, x in enumerate(written):
        step = 16 if x in ("k_out", "v_out") else 4
        for y in ["k", "v", "scores", "kv_len"] + written[:i]:
            other = at(y) - at(y) % 16
            for where in (other - sizes[x] + step, other, -(-(other + sizes[y] - step) // step) * step):
                if (x, y) == ("kv_len_out", "kv_len") and where == other:
                    continue  # the new lengths may take the old ones' place
                assert _code(built_lib, _args(b, **{x: where})) == INVALID, (x, y, where - other)
            assert _code(built_lib, _args(b, **{x: other + (sizes[y] + 15) // 16 * 16})) != INVALID, (x, y)
    assert _code(built_lib, _args(b, kv_len_out=at("kv_len"))) != INVALID


@no_device
def test_keys_that_are_their_own_values_cannot_be_compacted_in_place(built_lib, pkg):
    """k == v in place: two CTAs would move the same rows."""
    b, at = pkg.binding, 1 << 20
    place = dict(rows=6, out_rows=6, kv_batch_stride=6 * 16, out_batch_stride=6 * 16, scores=9 << 20, scores_out=9 << 20)
    names = dict(kept=11 << 20, kv_len=12 << 20, kv_len_out=13 << 20)
    assert _code(built_lib, _args(b, k=at, v=at, k_out=at, v_out=at, **place, **names)) == INVALID
    assert _code(built_lib, _args(b, k=at, v=2 << 20, k_out=at, v_out=2 << 20, **place, **names)) != INVALID
    assert _code(built_lib, _args(b, k=at, v=at)) != INVALID  # read twice, written apart
