"""The ends of SmolLMB200.generate: prompts it cannot embed, the last position, rows without a usable logit."""
import math

import pytest
import torch

from test_paged_sequences import tiny


@pytest.mark.parametrize("prompts", [[[1, 50]], [[3], [-1, 2]], [[10 ** 12]]])
def test_tokens_outside_the_vocabulary_are_refused(prompts):
    """On the host, before anything is indexed with them (the model has 50)."""
    model = tiny(torch.device("cpu"))
    with pytest.raises(ValueError, match="vocabulary"):
        model.generate(prompts, 2)


@pytest.mark.gpu
def test_the_last_position_can_be_used(cuda_dev):
    """The last new token is not stored, so a prompt of n tokens and m new ones take n + m - 1 positions (of 64)."""
    from npu_b200 import device_error

    model = tiny(cuda_dev)
    prompts = [[t % 50 for t in range(64)], [5] * 60]
    short = model.generate([p[-1:] for p in prompts], 1)  # any first call
    assert short.shape == (2, 1)
    assert model.generate(prompts, 1).shape == (2, 1)
    whole = model.generate([prompts[1]], 5)
    assert whole.shape == (1, 5) and torch.equal(whole[:, :1], model.generate(prompts, 1)[1:])
    with pytest.raises(ValueError):
        model.generate(prompts, 2)
    cache = model.new_paged_cache(4, 16)  # 64 tokens, all of them
    assert torch.equal(model.generate([prompts[1]], 5, cache=cache), whole)
    assert device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("settings", [{}, dict(temperature=0.8, top_k=20)])
def test_a_row_without_a_usable_logit_ends(cuda_dev, settings, monkeypatch):
    """The second prompt's logits are NaN once (at the first token, at a later one): -1 from there on, and the other
    prompts' tokens as without it."""
    from npu_b200 import device_error

    model = tiny(cuda_dev)
    prompts = [[1, 2, 3], [4], [5, 6, 7, 8, 9]]

    def run():
        return model.generate(prompts, 6, generator=torch.Generator(device=cuda_dev).manual_seed(1), **settings)

    clean = run()
    assert (clean >= 0).all()
    for name, first in [("prefill_packed", 0), ("decode_packed", 3)]:
        step, calls = getattr(model, name), []

        def once(*args):
            logits = step(*args)
            calls.append(0)
            if len(calls) == max(first, 1):
                logits[1] = math.nan
            return logits

        with monkeypatch.context() as patched:
            patched.setattr(model, name, once)
            out = run()
        assert torch.equal(out[[0, 2]], clean[[0, 2]])
        assert torch.equal(out[1, :first], clean[1, :first]) and (out[1, first:] == -1).all()
    assert device_error() == 0
