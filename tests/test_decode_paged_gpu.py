"""Single-token attention over a paged cache against a plain form in 64 bits.

Tolerance per element: P enters the second product as two bf16 terms (2^-16)
and scores are sums in fp32; 2^-14 of the softmax-weighted mean of |v| covers
both, and a bf16 output (8 significant bits) adds 2^-8 of its value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def paged(dev, lens, Hkv, D, page, seed=0, fill=math.nan, width=None, order="head"):
    """Random sequences scattered over a shuffled pool; every other slot holds `fill`.
    Returns k, v (lists of [len, Hkv, D]), pools [n_pages, Hkv, page, D] and the table."""
    g = torch.Generator(device=dev).manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 2
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), width or max(max(counts), 1)), -7, dtype=torch.int32, device=dev)
    pools = []
    for _ in range(2):
        shape = (pages, Hkv, page, D) if order == "head" else (pages, page, Hkv, D)
        pool = torch.full(shape, fill, dtype=torch.bfloat16, device=dev)
        pools.append(pool if order == "head" else pool.transpose(1, 2))
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        ids = perm[at:at + counts[b]]
        at += counts[b]
        table[b, :counts[b]] = ids
        for pool, keep in zip(pools, (ks, vs)):
            x = torch.randn(n, Hkv, D, generator=g, device=dev).bfloat16()
            keep.append(x)
            j = torch.arange(n, device=dev)
            pool[ids.long()[j // page], :, j % page] = x
    return ks, vs, pools[0], pools[1], table


def check(out, q, ks, vs, scale, gate=None):
    assert torch.isfinite(out).all()
    group = q.shape[1] // max(ks[0].shape[1], 1)
    for b, (k, v) in enumerate(zip(ks, vs)):
        if k.shape[0] == 0:
            assert (out[b] == 0).all()
            continue
        kk, vv = (x.double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        p = torch.softmax((kk @ q[b].double()[:, :, None]).squeeze(-1) * scale, -1)[:, None]
        o, mean = (p @ vv).squeeze(1), (p @ vv.abs()).squeeze(1)
        if gate is not None:
            o, mean = o * torch.sigmoid(gate[b].double()), mean * torch.sigmoid(gate[b].double())
        tol = 2 ** -14 * mean + 1e-7
        if out.dtype == torch.bfloat16:
            tol = tol * (1 + 2 ** -8) + 2 ** -8 * o.abs()
        d = (out[b].double() - o).abs()
        assert (d <= tol).all(), f"sequence {b}: {(d - tol).max().item()} over the tolerance"


HEADS = [(9, 3, 64), (16, 1, 64), (32, 4, 128), (5, 5, 128), (16, 2, 256), (4, 1, 256)]


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_lengths_pages_and_heads(cuda_dev, Hq, Hkv, D, page, out_dtype):
    from npu_b200 import decode_paged

    lens = [1, 15, 16, 17, 0, 63, 64, 65, 130, 1000]
    ks, vs, kp, vp, table = paged(cuda_dev, lens, Hkv, D, page, seed=page + D)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator(device=cuda_dev).manual_seed(1), device=cuda_dev)
    q = q.bfloat16()
    out = decode_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), out_dtype=out_dtype)
    check(out, q, ks, vs, 1 / math.sqrt(D))


@pytest.mark.parametrize("lens", [[20000], [3, 9000, 1, 700, 0, 12345], [500] * 40, [1] * 200,
                                  [0, 700, 33] * 45])
@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 2, 256)])
def test_long_and_many(cuda_dev, lens, Hq, Hkv, D):
    from npu_b200 import decode_paged

    ks, vs, kp, vp, table = paged(cuda_dev, lens, Hkv, D, 32, seed=len(lens))
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator(device=cuda_dev).manual_seed(2), device=cuda_dev)
    q = q.bfloat16()
    out = decode_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), scale=0.2)
    check(out, q, ks, vs, 0.2)


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("gate_dtype", [torch.float32, torch.bfloat16])
def test_token_major_pools_gate_strides_and_a_wide_table(cuda_dev, Hq, Hkv, D, gate_dtype):
    from npu_b200 import decode_paged

    lens = [100, 0, 333]
    ks, vs, kp, vp, table = paged(cuda_dev, lens, Hkv, D, 32, seed=4, width=50, order="token")
    g = torch.Generator(device=cuda_dev).manual_seed(4)
    qg = torch.randn(3, Hq, 2, D, generator=g, device=cuda_dev).bfloat16()
    q, gate = qg[:, :, 0], qg[:, :, 1].to(gate_dtype)
    hold = torch.full((3, Hq + 1, D), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    out = decode_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), out=hold[:, :Hq],
                       out_dtype=torch.bfloat16, gate=gate)
    check(out, q, ks, vs, 1 / math.sqrt(D), gate)
    assert (hold[:, Hq] == 7).all()


def test_large_scores_and_repeatable(cuda_dev):
    from npu_b200 import decode_paged

    lens = [3000, 64, 1500]
    ks, vs, kp, vp, table = paged(cuda_dev, lens, 4, 128, 64, seed=5)
    q = (30 * torch.randn(3, 32, 128, generator=torch.Generator(device=cuda_dev).manual_seed(5),
                          device=cuda_dev)).bfloat16()
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    out = decode_paged(q, kp, vp, table, sl, scale=1 / 8)
    assert torch.isfinite(out).all()
    for b in range(3):
        kk, vv = (x[b].double().transpose(0, 1).repeat_interleave(8, 0) for x in (ks, vs))
        s = (kk @ q[b].double()[:, :, None]).squeeze(-1) / 8
        o = (torch.softmax(s, -1)[:, None] @ vv).squeeze(1)
        # Scores near 1000 in fp32 are 2^-14 off, which moves weights by that much of themselves.
        assert (out[b].double() - o).abs().max().item() <= 2 ** -9 * vv.abs().max().item()
    for _ in range(3):
        assert torch.equal(decode_paged(q, kp, vp, table, sl, scale=1 / 8), out)


def test_nan_in_the_sequence_shows(cuda_dev):
    from npu_b200 import decode_paged

    lens = [200, 200]
    ks, vs, kp, vp, table = paged(cuda_dev, lens, 2, 128, 16, seed=6)
    q = torch.randn(2, 8, 128, device=cuda_dev).bfloat16()
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    clean = decode_paged(q, kp, vp, table, sl)
    kp[table[1, 3].long(), 1, 5] = math.nan
    out = decode_paged(q, kp, vp, table, sl)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :4], clean[1, :4])
    assert torch.isnan(out[1, 4:]).all()


def test_lengths_and_pages_out_of_range_report(cuda_dev):
    from npu_b200 import _lib, decode_paged, device_error

    ks, vs, kp, vp, table = paged(cuda_dev, [64, 64], 2, 128, 32, seed=7, fill=0.0)
    q = torch.randn(2, 8, 128, device=cuda_dev).bfloat16()
    assert device_error() == 0
    out = decode_paged(q, kp, vp, table, torch.tensor([65, -1], dtype=torch.int32, device=cuda_dev))
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    check(out[:1], q[:1], ks[:1], vs[:1], 128 ** -0.5)  # cut to the table's 64
    assert (out[1] == 0).all()
    table[1, 1] = 10 ** 6
    out = decode_paged(q, kp, vp, table, torch.tensor([64, 64], dtype=torch.int32, device=cuda_dev))
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    check(out[:1], q[:1], ks[:1], vs[:1], 128 ** -0.5)
    assert torch.isfinite(out).all() and device_error() == 0


def test_a_pool_past_two_to_the_31_elements(cuda_dev):
    """Pages at the far end of a pool of 2^31 + elements are found."""
    from npu_b200 import decode_paged

    n_pages = (1 << 31) // (2 * 64 * 128) + 70
    kp = torch.zeros(n_pages, 2, 64, 128, dtype=torch.bfloat16, device=cuda_dev)
    vp = torch.zeros_like(kp)
    far = torch.arange(n_pages - 5, n_pages, device=cuda_dev)
    ks = torch.randn(5 * 64, 2, 128, device=cuda_dev).bfloat16()
    vs = torch.randn(5 * 64, 2, 128, device=cuda_dev).bfloat16()
    kp[far] = ks.view(5, 64, 2, 128).transpose(1, 2)
    vp[far] = vs.view(5, 64, 2, 128).transpose(1, 2)
    q = torch.randn(1, 16, 128, device=cuda_dev).bfloat16()
    out = decode_paged(q, kp, vp, far.to(torch.int32)[None], torch.tensor([300], dtype=torch.int32, device=cuda_dev))
    check(out, q, [ks[:300]], [vs[:300]], 128 ** -0.5)
