"""Llama(weight_type="i8") with more sequences than other weight types' steps take."""
import numpy as np
import pytest
import torch

from test_model_int8_gpu import FAR, M, _apart, _config, plain_logits  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [33, 64, 80])
@pytest.mark.parametrize("mode", ["token", "batched"])
def test_logits_of_large_batches_are_the_plain_models(M, batch, mode):  # noqa: F811
    c = _config(M)
    w = M.random_weights(c, seed=8)
    rng = np.random.default_rng(batch)
    prompts = [rng.integers(0, c.vocab_size, size=int(n)).tolist() for n in rng.integers(1, 12, size=batch)]
    llama = M.Llama(c, w, batch=batch, weight_type="i8")
    llama.capture()
    tokens, logits = llama.generate(prompts, 4, want_logits=True, prompt_mode=mode)
    for b in range(0, batch, 5):
        want = plain_logits(c, w, prompts[b] + tokens[b].tolist())
        assert _apart(logits[b], want[len(prompts[b]) - 1:len(prompts[b]) + 3]) < FAR
        assert torch.equal(logits[b].argmax(-1).int(), tokens[b])
