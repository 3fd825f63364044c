"""Attention over packed sequences against a plain form in 64 bits.

Tolerance per element: P is rounded to bf16 before the second product (8
significant bits: at most 2^-8 of the softmax-weighted mean of |v|), scores
are sums in fp32 (2^-14 of the same mean covers them), and a bf16 output adds
2^-8 of its value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


def reference(q, k, v, lens_q, lens_k, scale, causal):
    """(o, softmax-weighted mean of |v|, lse), in 64 bits; rows that see nothing: 0, 0, -inf."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mean, lse = torch.zeros_like(o), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    group, iq, ik = q.shape[1] // k.shape[1], 0, 0
    for lq, lk in zip(lens_q, lens_k):
        qs = q[iq:iq + lq].double().transpose(0, 1)
        ks, vs = (x[ik:ik + lk].double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        s = qs @ ks.transpose(1, 2) * scale
        if causal:
            at = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
            s = s.masked_fill(torch.arange(lk, device=q.device)[None] > at, -math.inf)
        if lk:
            p = torch.nan_to_num(torch.softmax(s, -1))
            o[iq:iq + lq] = (p @ vs).transpose(0, 1)
            mean[iq:iq + lq] = (p @ vs.abs()).transpose(0, 1)
            lse[iq:iq + lq] = torch.logsumexp(s, -1).T
        iq, ik = iq + lq, ik + lk
    return o, mean, lse


def check(out, o, mean, gate=None):
    if gate is not None:
        o, mean = o * torch.sigmoid(gate.double()), mean * torch.sigmoid(gate.double())
    tol = (2 ** -8 + 2 ** -14) * mean + 1e-7
    if out.dtype == torch.bfloat16:
        tol = tol * (1 + 2 ** -8) + 2 ** -8 * o.abs()
    d = (out.double() - o).abs()
    assert torch.isfinite(out).all()
    assert (d <= tol).all(), f"max {(d - tol).max().item()} over the tolerance"


def inputs(dev, lens_q, lens_k, Hq, Hkv, D, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(sum(lens_q), Hq, D, generator=g, device=dev).bfloat16()
    k = torch.randn(sum(lens_k), Hkv, D, generator=g, device=dev).bfloat16()
    v = torch.randn(sum(lens_k), Hkv, D, generator=g, device=dev).bfloat16()
    return q, k, v


HEADS = [(9, 3, 64), (8, 2, 64), (3, 1, 128), (16, 4, 128), (16, 2, 256)]
LENGTHS = [
    [1],
    [1, 1, 1],
    [5, 0, 128, 129, 1],
    [127, 128, 255, 257, 64],
    [1000, 3, 700],
    [0, 0, 40, 0],
]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_prompts_of_different_lengths(cuda_dev, lens, Hq, Hkv, D, out_dtype):
    from npu_b200 import prefill_varlen

    q, k, v = inputs(cuda_dev, lens, lens, Hq, Hkv, D, seed=sum(lens) + D)
    out, lse = prefill_varlen(q, k, v, offsets(lens).to(cuda_dev), out_dtype=out_dtype, return_lse=True)
    o, mean, ref_lse = reference(q, k, v, lens, lens, 1 / math.sqrt(D), True)
    check(out, o, mean)
    assert (lse.T.double() - ref_lse).abs().max().item() <= 2e-4


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("lens", [[2100, 40, 1300], [4500]])
def test_long_prompts_take_two_tile_items(cuda_dev, lens, Hq, Hkv, D):
    from npu_b200 import prefill_varlen

    q, k, v = inputs(cuda_dev, lens, lens, Hq, Hkv, D, seed=3)
    out = prefill_varlen(q, k, v, offsets(lens).to(cuda_dev))
    check(out, *reference(q, k, v, lens, lens, 1 / math.sqrt(D), True)[:2])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_keys_of_their_own(cuda_dev, causal, Hq, Hkv, D):
    """More keys than queries (a cached prefix), fewer (rows that see nothing), none."""
    from npu_b200 import prefill_varlen

    lens_q, lens_k = [3, 200, 50, 7, 1, 0, 130], [300, 200, 20, 0, 513, 9, 131]
    q, k, v = inputs(cuda_dev, lens_q, lens_k, Hq, Hkv, D, seed=5)
    out, lse = prefill_varlen(q, k, v, offsets(lens_q).to(cuda_dev), offsets(lens_k).to(cuda_dev), causal=causal,
                              scale=0.3, return_lse=True)
    o, mean, ref_lse = reference(q, k, v, lens_q, lens_k, 0.3, causal)
    check(out, o, mean)
    assert torch.equal(torch.isinf(lse.T), torch.isinf(ref_lse))
    assert (out[253:260] == 0).all()  # the sequence without keys


@pytest.mark.parametrize("B", [33, 70, 300, 1500])
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 1, 64), (4, 2, 128), (2, 1, 256)])
def test_many_sequences(cuda_dev, B, Hq, Hkv, D):
    from npu_b200 import prefill_varlen

    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 300, (B,), generator=g).tolist()
    q, k, v = inputs(cuda_dev, lens, lens, Hq, Hkv, D, seed=B)
    out = prefill_varlen(q, k, v, offsets(lens).to(cuda_dev), out_dtype=torch.bfloat16)
    check(out, *reference(q, k, v, lens, lens, 1 / math.sqrt(D), True)[:2])


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("gate_dtype", [torch.float32, torch.bfloat16])
def test_gate_and_strided_views(cuda_dev, Hq, Hkv, D, gate_dtype):
    """q and the gate as views of one [q | gate] projection, k and v of a fused one, a strided out."""
    from npu_b200 import prefill_varlen

    lens = [130, 1, 77]
    n = sum(lens)
    g = torch.Generator(device=cuda_dev).manual_seed(D)
    qg = torch.randn(n, Hq, 2, D, generator=g, device=cuda_dev).bfloat16()
    kv = torch.randn(n, 2 * Hkv, D, generator=g, device=cuda_dev).bfloat16()
    q, gate, k, v = qg[:, :, 0], qg[:, :, 1].to(gate_dtype), kv[:, :Hkv], kv[:, Hkv:]
    hold = torch.full((n, Hq + 1, D), 7.0, device=cuda_dev)
    out = prefill_varlen(q, k, v, offsets(lens).to(cuda_dev), out=hold[:, :Hq], gate=gate)
    check(out, *reference(q, k, v, lens, lens, 1 / math.sqrt(D), True)[:2], gate)
    assert (hold[:, Hq] == 7).all()


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_a_neighbour_of_nan_and_infinity_changes_nothing(cuda_dev, Hq, Hkv, D):
    from npu_b200 import prefill_varlen

    lens = [70, 45, 300, 60]
    q, k, v = inputs(cuda_dev, lens, lens, Hq, Hkv, D, seed=8)
    cu = offsets(lens).to(cuda_dev)
    clean = prefill_varlen(q, k, v, cu)
    q[70:115], k[70:115], v[70:115] = math.nan, math.inf, math.nan
    v[415:] = -math.inf
    out = prefill_varlen(q, k, v, cu)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[115:415], clean[115:415])
    assert torch.isnan(out[70:115]).all()


def test_rows_outside_every_sequence_are_left_alone(cuda_dev):
    from npu_b200 import prefill_varlen

    q, k, v = inputs(cuda_dev, [400], [400], 8, 2, 128, seed=9)
    cu = torch.tensor([100, 150, 300], dtype=torch.int32, device=cuda_dev)
    out = torch.full((400, 8, 128), 5.0, device=cuda_dev)
    prefill_varlen(q, k, v, cu, out=out)
    assert (out[:100] == 5).all() and (out[300:] == 5).all()
    check(out[100:300], *reference(q[100:300], k[100:300], v[100:300], [50, 150], [50, 150], 128 ** -0.5, True)[:2])


def test_same_bits_as_the_dense_kernel_at_head_dim_128(cuda_dev):
    from npu_b200 import prefill, prefill_varlen

    q, k, v = inputs(cuda_dev, [900, 900], [900, 900], 8, 4, 128, seed=10)
    out = prefill_varlen(q, k, v, offsets([900, 900]).to(cuda_dev))
    dense = prefill(*(x.view(2, 900, -1, 128).transpose(1, 2) for x in (q, k, v)))
    assert torch.equal(out.view(2, 900, 8, 128).transpose(1, 2), dense)


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_no_keys_at_all_and_no_rows(cuda_dev, Hq, Hkv, D):
    from npu_b200 import prefill_varlen

    q, k, v = inputs(cuda_dev, [30, 200], [0], Hq, Hkv, D, seed=13)
    none = torch.zeros(3, dtype=torch.int32, device=cuda_dev)
    out, lse = prefill_varlen(q, k, v, offsets([30, 200]).to(cuda_dev), none, return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all()
    assert prefill_varlen(q[:0], k, v, none, none).shape == (0, Hq, D)


def test_on_another_stream(cuda_dev):
    from npu_b200 import prefill_varlen

    lens = [300, 20]
    q, k, v = inputs(cuda_dev, lens, lens, 9, 3, 64, seed=11)
    cu = offsets(lens).to(cuda_dev)
    expected = prefill_varlen(q, k, v, cu)
    side = torch.cuda.Stream(cuda_dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = prefill_varlen(q, k, v, cu)
    side.synchronize()
    assert torch.equal(out, expected)


def test_bad_offsets_leave_their_sequence_out_and_report(cuda_dev):
    from npu_b200 import _lib, device_error, prefill_varlen

    q, k, v = inputs(cuda_dev, [200], [200], 8, 2, 128, seed=12)
    assert device_error() == 0
    out = torch.full((200, 8, 128), 5.0, device=cuda_dev)
    cu = torch.tensor([0, 50, 900], dtype=torch.int32, device=cuda_dev)  # the second one runs past the tensors
    prefill_varlen(q, k, v, cu, out=out)
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    assert (out[50:] == 5).all()
    check(out[:50], *reference(q[:50], k[:50], v[:50], [50], [50], 128 ** -0.5, True)[:2])
    assert device_error() == 0
