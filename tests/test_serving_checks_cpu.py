"""Further refusals of the serving operators, without a GPU: nothing is launched."""
import pytest
import torch

from npu_b200 import _lib
from test_serving_cpu import FAKE, append


@pytest.mark.parametrize("start,out", [(FAKE, FAKE), (FAKE, FAKE + 4), (FAKE + 4, FAKE)])
def test_positions_and_lengths_in_one_place_are_refused(start, out):
    """Two sequences, so 8 bytes each: the lengths would be written while other blocks read the positions there."""
    assert append(spb=start, so=out) == _lib.B2A_ERR_INVALID_ARG


def test_positions_and_lengths_side_by_side_are_not():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: the call would launch")
    assert append(spb=FAKE, so=FAKE + 8) in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)
    assert append(spb=FAKE, so=None) in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)
