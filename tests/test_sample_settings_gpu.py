"""What sample takes as a setting and as a place for its result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(dev, R=3, V=1000):
    g = torch.Generator(device=dev).manual_seed(R)
    return torch.randn(R, V, generator=g, device=dev), torch.empty(R, V, device=dev).exponential_(generator=g)


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("value", ["many", None, [1.0]])
def test_a_setting_that_is_no_number_is_refused(cuda_dev, name, value):
    from npu_b200 import sample

    with pytest.raises(ValueError, match=f"{name} must be a number"):
        sample(*rows(cuda_dev), **{name: value})


def test_a_top_k_that_is_not_a_number_is_refused(cuda_dev):
    from npu_b200 import sample

    x, e = rows(cuda_dev)
    with pytest.raises(ValueError, match="top_k must not be NaN"):
        sample(x, e, top_k=math.nan)
    whole = sample(x, e)
    for k in (0, -3, 10 ** 12, -10 ** 12, math.inf, 1000, 5000):
        assert torch.equal(sample(x, e, top_k=k), whole)


def test_the_result_of_one_row_goes_into_a_column(cuda_dev):
    """tokens[:, step] of a [1, steps] buffer: one element, whatever its stride."""
    from npu_b200 import sample

    x, e = rows(cuda_dev, 1)
    tokens = torch.full((1, 5), -9, dtype=torch.long, device=cuda_dev)
    sample(x, e, out=tokens[:, 2])
    assert tokens.tolist() == [[-9, -9, sample(x, e).item(), -9, -9]]
    x, e = rows(cuda_dev, 2)
    with pytest.raises(ValueError, match="out must be"):
        sample(x, e, out=tokens.expand(2, 5)[:, 2])
    with pytest.raises(ValueError, match="out must be"):
        sample(x, e, out=torch.zeros(2, 5, dtype=torch.long, device=cuda_dev)[:, 2])
