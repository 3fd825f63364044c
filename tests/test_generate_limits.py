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
