"""Single-token attention over an 8-bit cache where V's scales span many powers of two (rows of zeros among them, whose
scale is the smallest), against 64 bits.

Tolerance, relative to the softmax-weighted mean of |v| of a column. A key's weight is 2^t, t = s + log2 sv:
- s = q k: products of f16 numbers (8 bits of q, 4 of k) are exact, each of the D / 16 steps that sum 16 of them keeps
  2^-20 of the largest at least; with A the largest sum of |q k| in base-2 units, D / 16 2^-20 A;
- t, the logarithm and t less the running maximum are fp32 numbers up to 128: 2^-18 each, 2^-17 for the logarithm and
  what the approximations of it and of 2^x add: together less than 2^-15;
- the weight as two f16 terms: 2^-22 of it, or 2^-40 of the largest weight, which multiplies codes up to 448.
With delta = ln 2 (D / 16 2^-20 A + 2^-15) for numerator and denominator: 2 delta of the mean, and n 2^-40 448 of the
largest p sv of the sequence. (fp32 sums and the quotient by sv: 2^-18 more, in the 2^-15's slack of ln 2.)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def rows(dev, n, Hkv, D, seed):
    """n rows of random codes whose largest is 448."""
    x = torch.randn(n, Hkv, D, generator=gen(dev, seed), device=dev)
    return (x / x.abs().amax(-1, keepdim=True) * 448).to(E4M3)


def paged(x, page):
    """[n, Hkv, ..] as pages [n / page, Hkv, page, ..]."""
    return x.unflatten(0, (-1, page)).transpose(1, 2).contiguous()


def check(out, q, kc, sk, vc, sv, scale, first=0):
    """out, q [B, Hq, D] against one sequence's codes [n, Hkv, D] and scales [n, Hkv], from key `first` on."""
    kc, sk, vc, sv = (x[first:].transpose(0, 1) for x in (kc, sk, vc, sv))
    n, D, group = kc.shape[1], q.shape[2], q.shape[1] // kc.shape[0]
    assert torch.isfinite(out).all()
    for g in range(kc.shape[0]):
        k, v = kc[g].double() * sk[g].double()[:, None], vc[g].double() * sv[g].double()[:, None]
        x = q[:, g * group:(g + 1) * group].double()
        A = (x.abs() @ k.abs().T).max().item() * scale * math.log2(math.e)
        p = torch.softmax(x @ k.T * scale, -1)
        o, mean = p @ v, p @ v.abs()
        delta = math.log(2) * (D / 16 * 2 ** -20 * A + 2 ** -15)
        tol = 2 * delta * mean + n * 2 ** -40 * 448 * (p * sv[g].double()).amax(-1, keepdim=True)
        d = (out[:, g * group:(g + 1) * group].double() - o).abs()
        assert (d <= tol).all(), f"KV head {g}: {(d / tol).max().item()} tolerances"


@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 1, 128), (8, 2, 256)])
@pytest.mark.parametrize("zeros", [1500, 8192, 20000, 32700])
@pytest.mark.parametrize("zero_keys", [True, False])
def test_rows_of_zeros_ahead(cuda_dev, Hq, Hkv, D, zeros, zero_keys):
    """A long stretch of zeros as a cache that was cleared holds it, then ordinary rows, in so many pairs that a CTA
    takes more than 16384 keys in a row. All sequences name the same pages."""
    from npu_b200 import decode_paged

    dev, n, page = cuda_dev, 32768, 64
    B = -(-240 // Hkv)
    kc, vc = (rows(dev, n, Hkv, D, s) for s in (1, 2))
    sk, sv = (0.002 + 0.006 * torch.rand(n, Hkv, generator=gen(dev, s), device=dev) for s in (3, 4))
    vc.view(torch.uint8)[:zeros] = 0
    sv[:zeros] = 2.0 ** -100
    if zero_keys:
        kc.view(torch.uint8)[:zeros] = 0
        sk[:zeros] = 2.0 ** -100
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(B, -1).contiguous()
    q = torch.randn(B, Hq, D, generator=gen(dev, 5), device=dev).bfloat16()
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    out = decode_paged(q, paged(kc, page), paged(vc, page), table, lens, k_scales=paged(sk, page),
                       v_scales=paged(sv, page))
    check(out, q, kc, sk, vc, sv, 1 / math.sqrt(D))


@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 1, 128), (8, 2, 256)])
@pytest.mark.parametrize("n", [48, 400, 5008])
@pytest.mark.parametrize("low,high", [(-90, 20), (-100, 10), (-20, 90), (60, 90)])
def test_scales_of_every_size(cuda_dev, Hq, Hkv, D, n, low, high):
    """V's scales of one sequence from 2^low to 2^high."""
    from npu_b200 import decode_paged

    dev, page, B = cuda_dev, 16, 3
    kc, vc = (rows(dev, n, Hkv, D, s) for s in (1, 2))
    sk = 0.002 + 0.006 * torch.rand(n, Hkv, generator=gen(dev, 3), device=dev)
    sv = 2.0 ** torch.linspace(low, high, n * Hkv, device=dev)[torch.randperm(n * Hkv, generator=gen(dev, 4),
                                                                              device=dev)].view(n, Hkv)
    sv = sv.clamp(2.0 ** low, 2.0 ** high)
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(B, -1).contiguous()
    q = torch.randn(B, Hq, D, generator=gen(dev, 5), device=dev).bfloat16()
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    out = decode_paged(q, paged(kc, page), paged(vc, page), table, lens, k_scales=paged(sk, page),
                       v_scales=paged(sv, page))
    check(out, q, kc, sk, vc, sv, 1 / math.sqrt(D))


def test_scales_past_the_range(cuda_dev):
    """Below 2^-100 a scale of V counts as that, above 2^90 as NaN, in the heads and sequences that attend it."""
    from npu_b200 import decode_paged

    dev, n, Hkv, D = cuda_dev, 48, 2, 64
    kc, vc = (rows(dev, n, Hkv, D, s) for s in (1, 2))
    sk, sv = torch.full((n, Hkv), 0.004, device=dev), torch.full((n, Hkv), 2.0 ** -110, device=dev)
    q = torch.randn(1, 4, D, generator=gen(dev, 5), device=dev).bfloat16()
    table = torch.arange(3, dtype=torch.int32, device=dev)[None]

    def call(t):
        return decode_paged(q, paged(kc, 16), paged(vc, 16), table, torch.tensor([t], dtype=torch.int32, device=dev),
                            k_scales=paged(sk, 16), v_scales=paged(sv, 16))

    check(call(n) * 2.0 ** 100, q, kc, sk, vc, torch.ones_like(sv), 1 / 8)
    for big in (2.0 ** 91, 2.0 ** 120, math.inf):
        sv.fill_(0.004)
        sv[40, 1] = big
        out = call(n)
        assert out[0, 2:].isnan().all()
        check(out[:, :2], q[:, :2], kc[:, :1], sk[:, :1], vc[:, :1], sv[:, :1], 1 / 8)
        check(call(40), q, kc[:40], sk[:40], vc[:40], sv[:40], 1 / 8)
