"""Refusals of the 8-bit cache's operators and of the penalties, without a GPU: nothing is launched."""
import pytest
import torch

from npu_b200 import _lib, api

FAKE = 0x10000  # aligned, never read: the checks fail first
LL2, LL3 = _lib.ll2, _lib.ll3
INVALID, ALIGNMENT = _lib.B2A_ERR_INVALID_ARG, _lib.B2A_ERR_ALIGNMENT
CPU = (_lib.B2A_ERR_CUDA, _lib.B2A_ERR_DEVICE)


def ll2(x):
    return None if x is None else LL2(*x)


def decode(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, sk=FAKE, sv=FAKE, kss=(128, 64), vss=(128, 64), t=FAKE, ld=8, w=8, sl=FAKE,
             gate=None, o=FAKE, B=2, Hq=8, Hkv=2, pages=20, page=64, D=128, qs=(1024, 128), ks=(16384, 8192, 128),
             vs=(16384, 8192, 128), gs=(1024, 128), os=(1024, 128), gb=1, scale=0.1, fp32=1, ws=FAKE, wsb=1 << 30)
    a.update(over)
    return _lib.load().b2a_decode_paged_e4m3(
        a["q"], a["k"], a["v"], a["sk"], a["sv"], ll2(a["kss"]), ll2(a["vss"]), a["t"], a["ld"], a["w"], a["sl"],
        a["gate"], a["o"], a["B"], a["Hq"], a["Hkv"], a["pages"], a["page"], a["D"], LL2(*a["qs"]), LL3(*a["ks"]),
        LL3(*a["vs"]), LL2(*a["gs"]), LL2(*a["os"]), a["gb"], a["scale"], a["fp32"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code", [
    (dict(sk=None), INVALID), (dict(sv=None), INVALID), (dict(kss=None), INVALID), (dict(vss=None), INVALID),
    (dict(sk=FAKE + 4), ALIGNMENT), (dict(vss=(128, 62)), ALIGNMENT), (dict(kss=(-128, 64)), ALIGNMENT),
    (dict(k=FAKE + 8), ALIGNMENT), (dict(ks=(16384, 8192, 136)), ALIGNMENT), (dict(vs=(16384, 8200, 128)), ALIGNMENT),
    (dict(page=24), INVALID), (dict(D=96), _lib.B2A_ERR_HEAD_DIM), (dict(Hq=34), _lib.B2A_ERR_GQA),
    (dict(ws=None), _lib.B2A_ERR_WORKSPACE), (dict(scale=0.0), INVALID),
])
def test_decode(over, code):
    assert decode(**over) == code


def append(**over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, qs=(1024, 128), ks=(256, 128), vs=(256, 128), bf16=1, qn=None, kn=None, eps=1e-6,
             cos=FAKE, sin=FAKE, tab=0, mp=100, rope=128, qo=FAKE, ko=None, vo=None, kp=FAKE, vp=FAKE,
             kps=(16384, 8192, 128), vps=(16384, 8192, 128), sk=FAKE, sv=FAKE, kss=(128, 64), vss=(128, 64), t=FAKE,
             ld=8, w=8, pages=20, page=64, cu=FAKE, B=2, N=9, Hq=8, Hkv=2, D=128, sp=0, spb=None, so=None)
    a.update(over)
    return _lib.load().b2a_rope_append_paged_e4m3(
        a["q"], a["k"], a["v"], LL2(*a["qs"]), LL2(*a["ks"]), LL2(*a["vs"]), a["bf16"], a["qn"], a["kn"], a["eps"],
        a["cos"], a["sin"], a["tab"], a["mp"], a["rope"], a["qo"], a["ko"], a["vo"], a["kp"], a["vp"], LL3(*a["kps"]),
        LL3(*a["vps"]), a["sk"], a["sv"], ll2(a["kss"]), ll2(a["vss"]), a["t"], a["ld"], a["w"], a["pages"], a["page"],
        a["cu"], a["B"], a["N"], a["Hq"], a["Hkv"], a["D"], a["sp"], a["spb"], a["so"], None)


@pytest.mark.parametrize("over,code", [
    (dict(sk=None), INVALID), (dict(sv=None), INVALID), (dict(kss=None), INVALID), (dict(sv=FAKE + 8), ALIGNMENT),
    (dict(kps=(16384, 8192, 136)), ALIGNMENT), (dict(vps=(16392, 8192, 128)), ALIGNMENT), (dict(N=0), INVALID),
    (dict(kp=None), INVALID), (dict(D=32), _lib.B2A_ERR_HEAD_DIM), (dict(spb=FAKE, so=FAKE), INVALID),
])
def test_append(over, code):
    assert append(**over) == code


def gather(**over):
    a = dict(k=FAKE, v=FAKE, ks=(16384, 8192, 128), vs=(16384, 8192, 128), sk=FAKE, sv=FAKE, kss=(128, 64),
             vss=(128, 64), t=FAKE, ld=8, w=8, pages=20, page=64, cu=FAKE, B=2, N=9, Hkv=2, D=128, sp=0, spb=None,
             ko=FAKE, vo=FAKE + 4608)
    a.update(over)
    return _lib.load().b2a_gather_paged(
        a["k"], a["v"], LL3(*a["ks"]), LL3(*a["vs"]), a["sk"], a["sv"], ll2(a["kss"]), ll2(a["vss"]), a["t"], a["ld"],
        a["w"], a["pages"], a["page"], a["cu"], a["B"], a["N"], a["Hkv"], a["D"], a["sp"], a["spb"], a["ko"], a["vo"],
        None)


@pytest.mark.parametrize("over,code", [
    (dict(k=None), INVALID), (dict(ko=None), INVALID), (dict(cu=None), INVALID), (dict(sk=None), INVALID),
    (dict(kss=None), INVALID), (dict(N=0), INVALID), (dict(B=0), INVALID), (dict(w=9), INVALID),
    (dict(sp=-1), INVALID), (dict(page=0), INVALID), (dict(D=80), _lib.B2A_ERR_HEAD_DIM),
    (dict(vo=FAKE + 4616), ALIGNMENT),
    (dict(vo=FAKE), INVALID), (dict(vo=FAKE + 4592), INVALID),
    (dict(ko=FAKE + 4608, vo=FAKE + 16), INVALID), (dict(ks=(16384, 8192, 136)), ALIGNMENT), (dict(spb=FAKE + 2), ALIGNMENT),
    (dict(sk=None, sv=None, ks=(16384, 8192, 132)), ALIGNMENT),
])
def test_gather(over, code):
    assert gather(**over) == code


def penalize(**over):
    a = dict(x=FAKE, ld=100, bf16=0, t=FAKE, wide=1, tr=8, ts=1, L=8, n=None, m=None, r=None, ra=1.1, f=None, fa=0.1,
             p=None, pa=0.2, b=None, lb=0, a=None, la=0, out=FAKE, lo=100, R=2, V=100)
    a.update(over)
    return _lib.load().b2a_penalize(
        a["x"], a["ld"], a["bf16"], a["t"], a["wide"], a["tr"], a["ts"], a["L"], a["n"], a["m"], a["r"], a["ra"],
        a["f"], a["fa"], a["p"], a["pa"], a["b"], a["lb"], a["a"], a["la"], a["out"], a["lo"], a["R"], a["V"], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), INVALID), (dict(out=None), INVALID), (dict(R=0), INVALID), (dict(V=0), INVALID),
    (dict(V=(1 << 30) + 1, lo=1 << 31), INVALID), (dict(L=-1), INVALID), (dict(t=None), INVALID),
    (dict(L=(1 << 30) + 1), INVALID), (dict(tr=-1), INVALID), (dict(lo=99), INVALID), (dict(ld=-1), INVALID),
    (dict(ra=0.0), INVALID), (dict(ra=float("inf")), INVALID), (dict(fa=float("nan")), INVALID),
    (dict(pa=float("inf")), INVALID), (dict(x=FAKE + 2), ALIGNMENT), (dict(t=FAKE + 4), ALIGNMENT),
    (dict(b=FAKE + 2), ALIGNMENT), (dict(n=FAKE + 1), ALIGNMENT),
    # Overlapping, but not in place: chunks of a row run in any order.
    (dict(out=FAKE + 4), INVALID), (dict(out=FAKE + 400), INVALID), (dict(lo=101), INVALID),
    (dict(out=FAKE - 4), INVALID),
])
def test_penalize(over, code):
    assert penalize(**over) == code


def test_valid_calls_without_a_gpu_report_it():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; covered by the gpu tests")
    assert decode() in CPU and append() in CPU and gather() in CPU and gather(sk=None, sv=None) in CPU
    assert penalize() in CPU and penalize(out=FAKE + 800) in CPU and penalize(t=None, L=0) in CPU
    assert penalize(R=1, lo=0) in CPU  # one row has no stride


def test_host_tensors_are_refused():
    q, kv = torch.zeros(4, 8, 64).bfloat16(), torch.zeros(4, 2, 64).bfloat16()
    pool, cu = torch.zeros(3, 2, 16, 64).to(torch.float8_e4m3fn), torch.tensor([0, 4], dtype=torch.int32)
    s, table = torch.ones(3, 2, 16), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        api.decode_paged(q, pool, pool, table.expand(4, 1), torch.ones(4, dtype=torch.int32), k_scales=s, v_scales=s)
    with pytest.raises(ValueError):
        api.rope_append_paged(q, kv, kv, torch.zeros(9, 64), torch.zeros(9, 64), pool, pool, table, cu, k_scales=s,
                              v_scales=s)
    with pytest.raises(ValueError):
        api.gather_paged(pool, pool, table, cu, 4, k_scales=s, v_scales=s)
    with pytest.raises(ValueError):
        api.penalize(torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.long))


@pytest.mark.parametrize("over,apart", [
    # out is FAKE .. FAKE + 800; a bias of 100 floats, one row or two, masks of 4 words, per-row arrays of two numbers.
    (dict(b=FAKE), 800), (dict(b=FAKE + 796), 800), (dict(b=FAKE - 396), -400), (dict(b=FAKE - 796, lb=100), -800),
    (dict(a=FAKE + 400), 800), (dict(a=FAKE - 12), -16), (dict(a=FAKE - 28, la=4), -32),
    (dict(r=FAKE - 4), -8), (dict(f=FAKE + 792), 800), (dict(p=FAKE), 800), (dict(n=FAKE + 8), 800),
    (dict(m=FAKE - 4), -8),
])
def test_penalize_into_its_other_inputs(over, apart):
    """Refused one element inside the output, valid right beside it."""
    assert penalize(**over) == INVALID
    if not torch.cuda.is_available():
        name = next(x for x in over if x not in ("lb", "la"))
        assert penalize(**{**over, name: FAKE + apart}) in CPU
