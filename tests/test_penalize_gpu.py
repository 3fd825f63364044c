"""Penalties, biases and masks on logits against the formula in 64 bits.

Tolerance: the steps (a product or quotient; a product and two differences; a sum) are each rounded in fp32, by 2^-24
of their result; none is larger than the sum of the magnitudes that enter, so 5 x 2^-24 of that sum covers them; a bf16
result adds 2^-8 of itself. Logits that nothing applies to come out bit by bit.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def ints(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def each(value, r):
    return float(value[r]) if isinstance(value, torch.Tensor) else float(value)


def expected(x, tokens=None, lengths=None, prompts=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None,
             allowed=None):
    """(result, sum of the magnitudes that entered) in 64 bits."""
    R, V = x.shape
    y, mass = x.double().clone(), x.double().abs()
    for r in range(R):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else min(max(int(lengths[r]), 0), tokens.shape[1])
            m = 0 if prompts is None else max(int(prompts[r]), 0)
            row = tokens[r, :n].long()
            good = (row >= 0) & (row < V)
            seen = torch.bincount(row[good], minlength=V) > 0
            c = torch.bincount(row[m:][good[m:]], minlength=V).double()
            rep, f, p = each(repetition, r), each(frequency, r), each(presence, r)
            y[r] = torch.where(seen, torch.where(y[r] > 0, y[r] / rep, y[r] * rep), y[r])
            mass[r] = torch.maximum(mass[r], y[r].abs()) + abs(f) * c + abs(p) * (c > 0)
            y[r] = y[r] - f * c - p * (c > 0)
        if bias is not None:
            b = (bias if bias.dim() == 1 else bias[r if bias.shape[0] > 1 else 0]).double()
            y[r] += b
            mass[r] += b.abs()
        if allowed is not None:
            word = (allowed if allowed.dim() == 1 else allowed[r if allowed.shape[0] > 1 else 0]).long()
            v = torch.arange(V, device=x.device)
            y[r] = torch.where((word[v // 32] >> (v % 32)) & 1 == 1, y[r], -math.inf)
    return y, mass


def compare(got, x, **kw):
    y, mass = expected(x, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape
    special = ~torch.isfinite(y)
    assert torch.equal(torch.nan_to_num(got.double()[special], nan=5, posinf=3, neginf=4),
                       torch.nan_to_num(y[special], nan=5, posinf=3, neginf=4))
    tol = 5 * 2 ** -24 * mass
    if x.dtype == torch.bfloat16:
        tol = tol + 2 ** -8 * (y.abs() + tol)
    d = (got.double() - y).abs()
    assert (d[~special] <= tol[~special]).all()


def mask_bits(dev, rows, V, seed):
    words = -(-V // 32)
    return torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen(dev, seed), device=dev).to(torch.int32)


@pytest.mark.parametrize("R,V", [(1, 1), (2, 7), (3, 31), (4, 1000), (5, 8191), (2, 49152), (7, 131071), (200, 8200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wide", [False, True])
def test_all_together(cuda_dev, R, V, dtype, wide):
    from npu_b200 import penalize

    dev, L = cuda_dev, 70
    g = gen(dev, R + V)
    x = (3 * torch.randn(R, V, generator=g, device=dev)).to(dtype)
    tokens = torch.randint(0, max(1, min(V, 40)), (R, L), generator=g, device=dev)
    tokens[:, ::2] = torch.randint(0, V, (R, L // 2), generator=g, device=dev)
    tokens = tokens if wide else tokens.to(torch.int32)
    lengths = torch.randint(0, L + 1, (R,), generator=g, device=dev, dtype=torch.int32)
    lengths[0] = L
    prompts = torch.randint(-1, L, (R,), generator=g, device=dev, dtype=torch.int32)
    kw = dict(repetition=0.5 + torch.rand(R, generator=g, device=dev), frequency=torch.randn(R, generator=g, device=dev),
              presence=torch.randn(R, generator=g, device=dev), bias=torch.randn(R, V, generator=g, device=dev),
              allowed=mask_bits(dev, R, V, 3))
    got = penalize(x, tokens, lengths, prompt_lengths=prompts, **kw)
    compare(got, x, tokens=tokens, lengths=lengths, prompts=prompts, **kw)
    # In place, the same bits.
    y = x.clone()
    assert penalize(y, tokens, lengths, prompt_lengths=prompts, out=y, **kw).data_ptr() == y.data_ptr()
    assert torch.equal(y.nan_to_num(), got.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(repetition=1.3), dict(repetition=0.7), dict(frequency=0.3), dict(presence=-0.4),
                                dict(repetition=1.2, frequency=0.1, presence=0.5), dict(frequency=1e-3)])
def test_numbers_for_all_rows(cuda_dev, dtype, kw):
    from npu_b200 import penalize

    dev = cuda_dev
    x = torch.randn(3, 5000, generator=gen(dev, 1), device=dev).to(dtype)
    tokens = torch.randint(0, 300, (3, 1000), generator=gen(dev, 2), device=dev)
    compare(penalize(x, tokens, **kw), x, tokens=tokens, **kw)
    prompts = ints(dev, [0, 1000, 400])
    compare(penalize(x, tokens, prompt_lengths=prompts, **kw), x, tokens=tokens, prompts=prompts, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_to_apply_keeps_the_bits(cuda_dev, dtype):
    from npu_b200 import penalize

    dev = cuda_dev
    x = torch.randn(4, 3001, generator=gen(dev, 1), device=dev).to(dtype)
    x[0, :4] = torch.tensor([math.inf, -math.inf, math.nan, -0.0])
    x[1, 5] = 1e-40  # subnormal in fp32
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    tokens = torch.full((4, 9), -1, device=dev)
    for got in (penalize(x), penalize(x, tokens, repetition=2.0), penalize(x, tokens[:, :0], frequency=1.0),
                penalize(x, tokens + 4, ints(dev, [0] * 4), presence=1.0),
                penalize(x, tokens + 4, repetition=1.0), penalize(x, allowed=torch.full((94,), -1, dtype=torch.int32, device=dev))):
        assert torch.equal(got.view(bits), x.view(bits))


def test_values_that_are_not_finite(cuda_dev):
    from npu_b200 import penalize

    dev = cuda_dev
    x = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, torch.finfo(torch.float32).min, 1.0]], device=dev)
    tokens = torch.arange(6, device=dev)[None]
    kw = dict(repetition=1.5, frequency=0.1, presence=0.2)
    got = penalize(x, tokens, **kw)
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and got[0, 2].isnan() and got[0, 4] == -math.inf
    assert abs(got[0, 3].item() + 0.3) < 1e-6
    bias = torch.tensor([-math.inf, math.inf, 0, -math.inf, 0, torch.finfo(torch.float32).min], device=dev)
    got = penalize(x, bias=bias)
    assert got[0, 0].isnan() and got[0, 1].isnan() and got[0, 3] == -math.inf and got[0, 5] < -3e38
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    assert (penalize(x, allowed=none) == -math.inf).all()  # a mask that leaves nothing
    from npu_b200 import sample
    assert sample(penalize(x, allowed=none), temperature=0.0).item() == -1


@pytest.mark.parametrize("ids", ["outside", "one", "long"])
def test_histories(cuda_dev, ids):
    """Ids outside the vocabulary count for nothing; the same id everywhere; tens of thousands of tokens."""
    from npu_b200 import device_error, penalize

    dev, V = cuda_dev, 20000
    device_error()
    x = torch.randn(2, V, generator=gen(dev, 1), device=dev)
    if ids == "outside":
        tokens = torch.tensor([[5, -1, V, 2 ** 40, -2 ** 40, 5 + 2 ** 32], [V - 1, 0, -100, V + 1, 2 ** 62, 7]], device=dev)
    elif ids == "one":
        tokens = torch.full((2, 5000), 19999, device=dev)
    else:
        tokens = torch.randint(0, V, (2, 60001), generator=gen(dev, 2), device=dev)
    kw = dict(repetition=1.2, frequency=0.01, presence=0.5)
    compare(penalize(x, tokens, **kw), x, tokens=tokens, **kw)
    assert device_error() == 0


def test_strides(cuda_dev):
    """Rows of a larger tensor, tokens stored step by step, one bias and one mask for all, other output strides."""
    from npu_b200 import penalize

    dev, R, V = cuda_dev, 5, 4099
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(R, V + 70, generator=gen(dev, 1), device=dev).to(dtype)
        tokens = torch.randint(0, V, (64, R), generator=gen(dev, 2), device=dev).T  # [R, 64], as generation stores them
        kw = dict(repetition=1.4, frequency=0.2)
        for at in range(0, 9):
            x = wide[:, at:at + V]
            big = torch.full((R, V + 33), 9.0, device=dev, dtype=dtype)
            out = big[:, at + 1:at + 1 + V]
            penalize(x, tokens, out=out, **kw)
            compare(out, x, tokens=tokens, **kw)
            assert (big[:, :at + 1] == 9).all() and (big[:, at + 1 + V:] == 9).all()
        x = wide[:, :V]
        bias, allowed = torch.randn(1, V, generator=gen(dev, 3), device=dev), mask_bits(dev, 1, V, 4)
        for b, a in ((bias, allowed), (bias[0], allowed[0]), (bias.expand(R, V), allowed.expand(R, -1))):
            compare(penalize(x, bias=b, allowed=a), x, bias=b, allowed=a)
        keep = wide.clone()
        compare(penalize(x, tokens, out=x, **kw), keep[:, :V], tokens=tokens, **kw)  # in place within a larger tensor
        assert torch.equal(wide[:, V:], keep[:, V:])


def test_more_rows_than_a_grid_has(cuda_dev):
    from npu_b200 import penalize

    dev, R, V = cuda_dev, 140000, 37
    g = gen(dev, 1)
    x = torch.randn(R, V, generator=g, device=dev)
    tokens = torch.randint(0, V, (R, 3), generator=g, device=dev)
    rep = 0.5 + torch.rand(R, generator=g, device=dev)
    bias = torch.randn(R, V, generator=g, device=dev)
    got = penalize(x, tokens, ints(dev, [3] * R), repetition=rep, bias=bias, prompt_lengths=ints(dev, [1] * R))
    seen = torch.zeros_like(x).scatter_(1, tokens, 1.0) > 0
    y = x.double()
    y = torch.where(seen, torch.where(y > 0, y / rep[:, None].double(), y * rep[:, None].double()), y) + bias.double()
    assert ((got.double() - y).abs() <= 3 * 2 ** -24 * (y.abs() + 2 * bias.abs().double() + 1e-30)).all()


def test_lengths_out_of_range_are_cut_and_reported(cuda_dev):
    from npu_b200 import device_error, penalize
    from npu_b200._lib import B2A_ERR_DEVICE_BAD_LEN

    dev = cuda_dev
    device_error()
    x = torch.randn(3, 100, generator=gen(dev, 1), device=dev)
    tokens = torch.randint(0, 100, (3, 8), generator=gen(dev, 2), device=dev)
    lengths = ints(dev, [-5, 9, 3])
    compare(penalize(x, tokens, lengths, repetition=1.5), x, tokens=tokens, lengths=lengths, repetition=1.5)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN


def test_empty(cuda_dev):
    from npu_b200 import penalize

    assert penalize(torch.zeros(0, 50, device=cuda_dev)).shape == (0, 50)
    assert penalize(torch.zeros(3, 0, device=cuda_dev)).shape == (3, 0)


BAD = [
    (lambda d: dict(x=torch.zeros(3, 100, device=d).half()), "logits must be"),
    (lambda d: dict(x=torch.zeros(100, device=d)), "logits must be"),
    (lambda d: dict(x=torch.zeros(3, 200, device=d)[:, ::2]), "logits must be"),
    (lambda d: dict(tokens=torch.zeros(2, 5, dtype=torch.int64, device=d)), r"tokens must be .* \[3, L\]"),
    (lambda d: dict(tokens=torch.zeros(3, 5, device=d)), "tokens must be"),
    (lambda d: dict(tokens=torch.zeros(3, 5, dtype=torch.int64)), "tokens must be"),
    (lambda d: dict(lengths=ints(d, [1, 2])), "lengths must be .* 3"),
    (lambda d: dict(tokens=None, lengths=ints(d, [1, 2, 3])), "missing"),
    (lambda d: dict(prompt_lengths=ints(d, [1, 2, 3]).long()), "prompt_lengths must be"),
    (lambda d: dict(repetition=0.0), "above 0"), (lambda d: dict(repetition=math.nan), "above 0"),
    (lambda d: dict(repetition=1e300), "above 0"), (lambda d: dict(frequency=math.inf), "frequency must be finite"),
    (lambda d: dict(presence=math.nan), "presence must be finite"), (lambda d: dict(presence="much"), "presence"),
    (lambda d: dict(frequency=torch.ones(2, device=d)), r"frequency must be .* \[3\]"),
    (lambda d: dict(bias=torch.zeros(99, device=d)), r"bias must be .* \[100\] or \[3, 100\]"),
    (lambda d: dict(bias=torch.zeros(2, 100, device=d)), "bias must be"),
    (lambda d: dict(bias=torch.zeros(100, device=d).bfloat16()), "bias must be"),
    (lambda d: dict(allowed=torch.zeros(3, dtype=torch.int32, device=d)), r"allowed must be .* \[4\] or \[3, 4\]"),
    (lambda d: dict(allowed=torch.zeros(4, dtype=torch.int64, device=d)), "allowed must be"),
    (lambda d: dict(out=torch.zeros(3, 99, device=d)), "out must match"),
    (lambda d: dict(out=torch.zeros(3, 100, device=d).bfloat16()), "out must match"),
]


@pytest.mark.parametrize("which", range(len(BAD)))
def test_refused(cuda_dev, which):
    from npu_b200 import penalize

    def call(**over):
        a = dict(x=torch.zeros(3, 100, device=cuda_dev), tokens=torch.zeros(3, 5, dtype=torch.int64, device=cuda_dev))
        a.update(over)
        return penalize(a.pop("x"), a.pop("tokens"), **a)

    over, message = BAD[which]
    call()
    with pytest.raises(ValueError, match=message):
        call(**over(cuda_dev))
    call()
    torch.cuda.synchronize()


def test_overlapping_output_is_refused(cuda_dev):
    from npu_b200 import B2AError, penalize

    buf = torch.zeros(1000, device=cuda_dev)
    with pytest.raises(B2AError):
        penalize(buf[:300].view(3, 100), out=buf[100:400].view(3, 100))
    with pytest.raises(B2AError):
        penalize(buf[:300].view(3, 100), out=buf.as_strided((3, 100), (50, 1)))
