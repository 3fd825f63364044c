"""Rotation and append into pages against the formulas in 64 bits.

Tolerance: fp32 arithmetic on values of a few units (2^-18 covers the table,
norm and two products) and one rounding to bf16 (8 significant bits: 2^-8 of
the value).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
CASES = [(9, 3, 64, 64), (8, 2, 64, 16), (32, 4, 128, 128), (4, 4, 128, 0), (16, 2, 256, 64), (2, 1, 256, 256)]


def tables(dev, max_pos, rope, dtype):
    inv = 1.0 / (10000.0 ** (torch.arange(0, rope, 2, dtype=torch.float32, device=dev) / max(rope, 1)))
    a = torch.outer(torch.arange(max_pos, dtype=torch.float32, device=dev), inv)
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype).contiguous(), a.sin().to(dtype).contiguous()


def rotated(x, w, cos, sin, pos, rope, eps=1e-6):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    c, s, h = cos.double()[pos, None], sin.double()[pos, None], rope // 2
    a, b, rest = x[..., :h], x[..., h:rope], x[..., rope:]
    return torch.cat([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], rest], -1)


def near(got, ref):
    assert ((got.double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -18 * (1 + ref.abs().amax())).all()


def setup(dev, lens, starts, Hq, Hkv, D, rope, dtype, page, tab=None, seed=0, order="head"):
    g = torch.Generator(device=dev).manual_seed(seed)
    n, most = sum(lens), max(s + t for s, t in zip(starts, lens))
    qkv = torch.randn(n, (Hq + 2 * Hkv), D, generator=g, device=dev).to(dtype)
    counts = [-(-(s + t) // page) for s, t in zip(starts, lens)]
    perm = torch.randperm(sum(counts) + 3, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    shape = (len(perm), Hkv, page, D) if order == "head" else (len(perm), page, Hkv, D)
    pools = [torch.full(shape, 3.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    if order == "token":
        pools = [x.transpose(1, 2) for x in pools]
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)
    cos, sin = tables(dev, most, rope, tab or dtype)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], cos, sin, pools[0], pools[1], table, cu


@pytest.mark.parametrize("Hq,Hkv,D,rope", CASES)
@pytest.mark.parametrize("dtype,tab", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                       (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("page,order", [(16, "head"), (48, "token")])
def test_tokens_land_rotated_in_their_pages(cuda_dev, Hq, Hkv, D, rope, dtype, tab, norm, page, order):
    from npu_b200 import rope_append_paged

    lens, starts = [5, 1, 0, 70, 33], [0, 31, 4, 100, 15]
    q, k, v, cos, sin, kp, vp, table, cu = setup(cuda_dev, lens, starts, Hq, Hkv, D, rope, dtype, page, tab, seed=D,
                                                 order=order)
    qn, kn = ((1 + 0.1 * torch.randn(2, D, device=cuda_dev)).to(dtype) if norm else (None, None))
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    ends = torch.zeros(5, dtype=torch.int32, device=cuda_dev)
    q_rot, k_rot, v_out = rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, start_pos_per_batch=start,
                                            seqlens_out=ends, q_norm=qn, k_norm=kn, rope_dim=rope, return_kv=True)
    assert ends.tolist() == [s + t for s, t in zip(starts, lens)]
    which = torch.repeat_interleave(torch.arange(5), torch.tensor(lens)).to(cuda_dev)
    pos = torch.cat([torch.arange(s, s + t) for s, t in zip(starts, lens)]).to(cuda_dev)
    near(q_rot, rotated(q, qn, cos, sin, pos, rope))
    near(k_rot, rotated(k, kn, cos, sin, pos, rope))
    assert torch.equal(v_out, v.to(torch.bfloat16))
    pages, slots = table[which, pos // page].long(), pos % page
    assert torch.equal(kp[pages, :, slots], k_rot) and torch.equal(vp[pages, :, slots], v_out)
    kp[pages, :, slots] = 3.0
    vp[pages, :, slots] = 3.0
    assert (kp == 3).all() and (vp == 3).all()  # nothing else was written


@pytest.mark.parametrize("Hq,Hkv,D,rope", CASES[:3])
def test_one_token_each_matches_the_dense_append(cuda_dev, Hq, Hkv, D, rope):
    """fp32 sources: bit for bit the dense-cache kernel's rows."""
    from npu_b200 import api

    B = 40
    starts = [(7 * b) % 50 for b in range(B)]
    q, k, v, cos, sin, kp, vp, table, cu = setup(cuda_dev, [1] * B, starts, Hq, Hkv, D, rope, torch.float32, 16)
    start = torch.tensor(starts, dtype=torch.int32, device=cuda_dev)
    got = api.rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, start_pos_per_batch=start, rope_dim=rope)
    kc, vc = (torch.zeros(B, Hkv, 64, D, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    ref = api.rope_append(q[:, None], k[:, None], v[:, None], cos, sin, kc, vc, start_pos_per_batch=start,
                          rope_dim=rope)
    assert torch.equal(got, ref[:, :, 0])
    b, s = torch.arange(B, device=cuda_dev), start.long()
    pages = table[b, s // 16].long()
    assert torch.equal(kp[pages, :, s % 16], kc[b, :, s]) and torch.equal(vp[pages, :, s % 16], vc[b, :, s])


def test_many_sequences_and_empty_ones(cuda_dev):
    from npu_b200 import rope_append_paged

    g = torch.Generator().manual_seed(3)
    lens = [t if t > 3 else 0 for t in torch.randint(0, 9, (1500,), generator=g).tolist()]
    q, k, v, cos, sin, kp, vp, table, cu = setup(cuda_dev, lens, [2] * 1500, 3, 1, 64, 64, torch.bfloat16, 16)
    out = rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, start_pos=2)
    pos = torch.cat([torch.arange(2, 2 + t) for t in lens]).to(cuda_dev)
    near(out, rotated(q, None, cos, sin, pos, 64))


def test_tokens_without_a_place_are_skipped_and_reported(cuda_dev):
    from npu_b200 import _lib, device_error, rope_append_paged

    q, k, v, cos, sin, kp, vp, table, cu = setup(cuda_dev, [20, 20], [0, 0], 4, 2, 128, 128, torch.bfloat16, 16)
    assert device_error() == 0
    table[1, 1] = -1  # tokens 16..19 of the second sequence
    rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu)
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    written = (kp != 3).any(-1).any(1).sum().item()
    assert written == 36
    start = torch.tensor([-1, 30], dtype=torch.int32, device=cuda_dev)  # before the start; past table and tables
    rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, start_pos_per_batch=start)
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN and device_error() == 0
