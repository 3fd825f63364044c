"""Refusals of the serving operators, without a GPU: nothing is launched."""
import pytest
import torch

from npu_b200 import _lib, api

FAKE = 0x10000  # aligned, never read: the checks fail first
LL2, LL3 = _lib.ll2, _lib.ll3


def varlen(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, gate=None, o=FAKE, lse=None, cq=FAKE, ck=FAKE, B=2, Nq=64, Nk=64, Hq=8, Hkv=2,
             D=128, qs=(1024, 128), ks=(256, 128), vs=(256, 128), gs=(1024, 128), os=(1024, 128), gb=1, scale=0.1,
             causal=1, fp32=1)
    a.update(over)
    return _lib.load().b2a_prefill_varlen(a["q"], a["k"], a["v"], a["gate"], a["o"], a["lse"], a["cq"], a["ck"],
                                          a["B"], a["Nq"], a["Nk"], a["Hq"], a["Hkv"], a["D"], LL2(*a["qs"]),
                                          LL2(*a["ks"]), LL2(*a["vs"]), LL2(*a["gs"]), LL2(*a["os"]), a["gb"],
                                          a["scale"], a["causal"], a["fp32"], None)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _lib.B2A_ERR_INVALID_ARG), (dict(cq=None), _lib.B2A_ERR_INVALID_ARG),
    (dict(B=0), _lib.B2A_ERR_INVALID_ARG), (dict(Nq=-1), _lib.B2A_ERR_INVALID_ARG),
    (dict(scale=0.0), _lib.B2A_ERR_INVALID_ARG), (dict(scale=float("nan")), _lib.B2A_ERR_INVALID_ARG),
    (dict(D=96), _lib.B2A_ERR_HEAD_DIM), (dict(Hkv=3), _lib.B2A_ERR_GQA),
    (dict(q=FAKE + 2), _lib.B2A_ERR_ALIGNMENT), (dict(ks=(260, 130)), _lib.B2A_ERR_ALIGNMENT),
    (dict(os=(1026, 128)), _lib.B2A_ERR_ALIGNMENT), (dict(gate=FAKE + 8), _lib.B2A_ERR_ALIGNMENT),
    (dict(vs=(-256, 128)), _lib.B2A_ERR_ALIGNMENT), (dict(Nq=0), _lib.B2A_OK),
])
def test_prefill_varlen(over, code):
    assert varlen(**over) == code


def paged(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, t=FAKE, ld=8, w=8, sl=FAKE, gate=None, o=FAKE, B=2, Hq=8, Hkv=2, pages=20,
             page=64, D=128, qs=(1024, 128), ks=(16384, 8192, 128), vs=(16384, 8192, 128), gs=(1024, 128),
             os=(1024, 128), gb=1, scale=0.1, fp32=1, ws=FAKE, wsb=1 << 30)
    a.update(over)
    return _lib.load().b2a_decode_paged(a["q"], a["k"], a["v"], a["t"], a["ld"], a["w"], a["sl"], a["gate"], a["o"],
                                        a["B"], a["Hq"], a["Hkv"], a["pages"], a["page"], a["D"], LL2(*a["qs"]),
                                        LL3(*a["ks"]), LL3(*a["vs"]), LL2(*a["gs"]), LL2(*a["os"]), a["gb"],
                                        a["scale"], a["fp32"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(t=None), _lib.B2A_ERR_INVALID_ARG), (dict(page=24), _lib.B2A_ERR_INVALID_ARG),
    (dict(page=0), _lib.B2A_ERR_INVALID_ARG), (dict(ld=7), _lib.B2A_ERR_INVALID_ARG),
    (dict(w=1 << 30, ld=1 << 30), _lib.B2A_ERR_INVALID_ARG), (dict(D=80), _lib.B2A_ERR_HEAD_DIM),
    (dict(Hq=34), _lib.B2A_ERR_GQA), (dict(Hq=9), _lib.B2A_ERR_GQA), (dict(v=FAKE + 8), _lib.B2A_ERR_ALIGNMENT),
    (dict(ks=(16384, 8192, 130)), _lib.B2A_ERR_ALIGNMENT), (dict(ws=None), _lib.B2A_ERR_WORKSPACE),
    (dict(wsb=0), _lib.B2A_ERR_WORKSPACE), (dict(scale=-1.0), _lib.B2A_ERR_INVALID_ARG),
])
def test_decode_paged(over, code):
    assert paged(**over) == code
    assert _lib.load().b2a_decode_paged_workspace_bytes(2, 8, 3, 128) == 0
    assert _lib.load().b2a_decode_paged_workspace_bytes(2, 8, 2, 128) > 0


def append(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, qs=(1024, 128), ks=(256, 128), vs=(256, 128), bf16=1, qn=None, kn=None, eps=1e-6,
             cos=FAKE, sin=FAKE, tab=0, mp=100, rope=128, qo=FAKE, ko=None, vo=None, kp=FAKE, vp=FAKE,
             kps=(16384, 8192, 128), vps=(16384, 8192, 128), t=FAKE, ld=8, w=8, pages=20, page=64, cu=FAKE, B=2, N=9,
             Hq=8, Hkv=2, D=128, sp=0, spb=None, so=None)
    a.update(over)
    return _lib.load().b2a_rope_append_paged(
        a["q"], a["k"], a["v"], LL2(*a["qs"]), LL2(*a["ks"]), LL2(*a["vs"]), a["bf16"], a["qn"], a["kn"], a["eps"],
        a["cos"], a["sin"], a["tab"], a["mp"], a["rope"], a["qo"], a["ko"], a["vo"], a["kp"], a["vp"], LL3(*a["kps"]),
        LL3(*a["vps"]), a["t"], a["ld"], a["w"], a["pages"], a["page"], a["cu"], a["B"], a["N"], a["Hq"], a["Hkv"],
        a["D"], a["sp"], a["spb"], a["so"], None)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _lib.B2A_ERR_INVALID_ARG), (dict(cu=None), _lib.B2A_ERR_INVALID_ARG),
    (dict(N=0), _lib.B2A_ERR_INVALID_ARG), (dict(rope=24), _lib.B2A_ERR_INVALID_ARG),
    (dict(rope=256), _lib.B2A_ERR_INVALID_ARG), (dict(cos=None), _lib.B2A_ERR_INVALID_ARG),
    (dict(mp=0), _lib.B2A_ERR_INVALID_ARG), (dict(sp=-1), _lib.B2A_ERR_INVALID_ARG),
    (dict(qn=FAKE, eps=float("inf")), _lib.B2A_ERR_INVALID_ARG), (dict(D=32), _lib.B2A_ERR_HEAD_DIM),
    (dict(kp=FAKE + 2), _lib.B2A_ERR_ALIGNMENT), (dict(qs=(1020, 128)), _lib.B2A_ERR_ALIGNMENT),
    (dict(page=0), _lib.B2A_ERR_INVALID_ARG), (dict(w=9), _lib.B2A_ERR_INVALID_ARG),
])
def test_rope_append_paged(over, code):
    assert append(**over) == code


def pick(**over):
    a = dict(x=FAKE, ld=100, bf16=0, e=FAKE, le=100, R=2, V=100, t=None, ta=1.0, k=None, ka=0, p=None, pa=1.0, m=None,
             ma=0.0, out=FAKE)
    a.update(over)
    return _lib.load().b2a_sample(a["x"], a["ld"], a["bf16"], a["e"], a["le"], a["R"], a["V"], a["t"], a["ta"], a["k"],
                                  a["ka"], a["p"], a["pa"], a["m"], a["ma"], a["out"], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), _lib.B2A_ERR_INVALID_ARG), (dict(out=None), _lib.B2A_ERR_INVALID_ARG),
    (dict(R=0), _lib.B2A_ERR_INVALID_ARG), (dict(V=0), _lib.B2A_ERR_INVALID_ARG),
    (dict(ld=-1), _lib.B2A_ERR_INVALID_ARG),
    (dict(le=-1), _lib.B2A_ERR_INVALID_ARG), (dict(ta=float("nan")), _lib.B2A_ERR_INVALID_ARG),
    (dict(x=FAKE + 2), _lib.B2A_ERR_ALIGNMENT), (dict(out=FAKE + 4), _lib.B2A_ERR_ALIGNMENT),
])
def test_sample(over, code):
    assert pick(**over) == code


def test_valid_calls_without_a_gpu_report_it():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; covered by the gpu tests")
    for call in (varlen, paged, append, pick):
        assert call() in (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)


def test_host_tensors_are_refused():
    q, kv = torch.zeros(4, 8, 64).bfloat16(), torch.zeros(4, 2, 64).bfloat16()
    pool, cu = torch.zeros(3, 2, 16, 64).bfloat16(), torch.tensor([0, 4], dtype=torch.int32)
    tab = torch.zeros(9, 64).bfloat16()
    with pytest.raises(ValueError):
        api.prefill_varlen(q, kv, kv, cu)
    with pytest.raises(ValueError):
        api.decode_paged(q, pool, pool, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        api.rope_append_paged(q, kv, kv, tab, tab, pool, pool, torch.zeros(1, 1, dtype=torch.int32), cu)
    with pytest.raises(ValueError):
        api.sample(torch.zeros(2, 5), torch.ones(2, 5))
