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
