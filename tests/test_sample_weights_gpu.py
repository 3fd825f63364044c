"""The weights that decide a draw between two tokens.

With T = 1 (or a power of two) z = (x - max) / T is exact, so a token's ratio w / e is off by the exponential's and the
quotient's error only: 2 units in the last place each (2^-22 of the value at most), and e is rounded to fp32 (2^-24).
Two such ratios compare as in 64 bits if they differ by 2^-19."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1.0, 0.25, 8.0])
@pytest.mark.parametrize("V,at", [(16, 8), (16, 9), (5000, 4001), (40_000, 39_000)])
def test_two_tokens_whose_ratios_nearly_agree(cuda_dev, T, V, at):
    """Token 0 has the maximum, token `at` (another thread's) lies z below it; its noise puts its ratio 2^-18 above
    or below token 0's."""
    from npu_b200 import sample

    z = torch.cat([torch.linspace(-80, -1, 150), -torch.logspace(-6, 0, 50)]).float()
    R = len(z)
    x = torch.full((2 * R, V), -math.inf)
    x[:, 0] = 3.0
    x[:, at] = 3.0 + T * z.repeat(2)
    exact = (x[:, at].double() - 3.0) / T  # what the rounding of x left
    assert torch.equal(exact.float().double(), exact)
    e = torch.ones(2 * R, V)
    closer = torch.cat([torch.full((R,), -1.0), torch.full((R,), 1.0)]).double()
    e[:, at] = (torch.exp(exact) * (1 + closer * 2 ** -18)).float()
    assert (e[:, at] > 1e-36).all()
    got = sample(x.to(cuda_dev), e.to(cuda_dev), temperature=T).cpu()
    assert torch.equal(got, torch.where(closer < 0, at, 0))
