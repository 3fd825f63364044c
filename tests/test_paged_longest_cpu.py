"""The longest tables that single-token attention over a paged cache takes, without a GPU: lengths, rounded up to whole
tiles of keys, are 32-bit numbers."""
import pytest
import torch

from npu_b200 import _lib

FAKE = 0x10000  # aligned, never read: nothing is launched without a device
LL2, LL3 = _lib.ll2, _lib.ll3


def decode(form, keys):
    lib, w = _lib.load(), keys // 16
    tail = (None, FAKE, 2, 8, 2, 20, 16, 128, LL2(1024, 128), LL3(4096, 2048, 128), LL3(4096, 2048, 128), LL2(1024, 128),
            LL2(1024, 128), 1, 0.1, 1, FAKE, 1 << 30, None)
    if form == "bf16":
        return lib.b2a_decode_paged(FAKE, FAKE, FAKE, FAKE, w, w, FAKE, *tail)
    if form == "shared":
        return lib.b2a_decode_paged_shared(FAKE, FAKE, FAKE, FAKE, w, w, FAKE, FAKE, None, 1, -1, *tail)
    return lib.b2a_decode_paged_e4m3(FAKE, FAKE, FAKE, FAKE, FAKE, LL2(32, 16), LL2(32, 16), FAKE, w, w, FAKE, *tail)


@pytest.mark.parametrize("form,longest", [("bf16", 2 ** 31 - 80), ("shared", 2 ** 31 - 80), ("e4m3", 2 ** 31 - 144)])
def test_longest_table(form, longest):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: valid calls would be launched")
    for keys in (longest - 48, longest):
        assert decode(form, keys) in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)
    assert decode(form, longest + 16) == _lib.B2A_ERR_INVALID_ARG
