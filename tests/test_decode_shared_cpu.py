"""Refusals of single-token attention over a shared prefix, without a GPU: nothing is launched."""
import pytest
import torch

from npu_b200 import _lib, api

FAKE = 0x10000  # aligned, never read: the checks fail first
LL2, LL3 = _lib.ll2, _lib.ll3
INVALID, ALIGNMENT = _lib.B2A_ERR_INVALID_ARG, _lib.B2A_ERR_ALIGNMENT


def call(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, t=FAKE, ld=80, w=80, sl=FAKE, pre=FAKE, cu=FAKE, n=2, least=-1, gate=None, o=FAKE,
             B=4, Hq=8, Hkv=2, pages=20, page=64, D=128, qs=(1024, 128), ks=(16384, 8192, 128), vs=(16384, 8192, 128),
             gs=(1024, 128), os=(1024, 128), gb=1, scale=0.1, fp32=1, ws=FAKE, wsb=1 << 30)
    a.update(over)
    return _lib.load().b2a_decode_paged_shared(
        a["q"], a["k"], a["v"], a["t"], a["ld"], a["w"], a["sl"], a["pre"], a["cu"], a["n"], a["least"], a["gate"],
        a["o"], a["B"], a["Hq"], a["Hkv"], a["pages"], a["page"], a["D"], LL2(*a["qs"]), LL3(*a["ks"]), LL3(*a["vs"]),
        LL2(*a["gs"]), LL2(*a["os"]), a["gb"], a["scale"], a["fp32"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(pre=None), INVALID), (dict(n=0), INVALID), (dict(cu=None), INVALID), (dict(pre=FAKE + 2), ALIGNMENT),
    (dict(cu=FAKE + 1), ALIGNMENT), (dict(t=None), INVALID), (dict(page=24), INVALID),
    (dict(D=96), _lib.B2A_ERR_HEAD_DIM), (dict(Hq=34), _lib.B2A_ERR_GQA), (dict(k=FAKE + 8), ALIGNMENT),
    (dict(ks=(16384, 8192, 130)), ALIGNMENT),
    (dict(ws=None), _lib.B2A_ERR_WORKSPACE), (dict(wsb=1000), _lib.B2A_ERR_WORKSPACE), (dict(scale=0.0), INVALID),
])
def test_refused(over, code):
    assert call(**over) == code


def test_workspace():
    lib = _lib.load()
    own = lib.b2a_decode_paged_workspace_bytes(4, 8, 2, 128)
    need = lib.b2a_decode_paged_shared_workspace_bytes(4, 8, 2, 128, 2)
    assert need > own > 0 and call(wsb=need - 1) == _lib.B2A_ERR_WORKSPACE
    assert lib.b2a_decode_paged_shared_workspace_bytes(4, 8, 2, 128, 0) == 0
    assert lib.b2a_decode_paged_shared_workspace_bytes(4, 8, 3, 128, 1) == 0
    assert api.decode_paged_shared_workspace_bytes(4, 8, 2, 128, 2) == need


def test_valid_calls_without_a_gpu_report_it():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; covered by the gpu tests")
    assert call() in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)
    assert call(cu=None, n=1) in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)


def test_host_tensors_are_refused():
    pool, lens = torch.zeros(3, 2, 16, 64).bfloat16(), torch.ones(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        api.decode_paged_shared(torch.zeros(4, 8, 64).bfloat16(), pool, pool, torch.zeros(4, 1, dtype=torch.int32),
                                lens, lens[:1])
