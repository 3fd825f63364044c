"""The 8-bit paged cache against plain forms in 64 bits: what the append stores, single-token attention over it, and
reading it back.

Tolerances. A stored value is e4m3(y / s) s: half a step of 4 significant bits (2^-4 of it) above 2^-6 s, half a step
of 2^-9 s below; s and y are fp32 results of a few operations on numbers up to the row's largest before the rotation,
which is at most sqrt(2) of that after it: 2^-20 of the largest covers them. Attention: P (times V's scale) enters the
second product as two bf16 terms (2^-16), everything else is fp32 sums: 2^-14 of the softmax-weighted mean of |v|, and
2^-8 of the value for a bf16 output.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HEADS = [(9, 3, 64), (16, 1, 64), (32, 4, 128), (5, 5, 128), (16, 2, 256), (9, 1, 256)]


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def ints(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def offsets(lens):
    at = [0]
    for t in lens:
        at.append(at[-1] + t)
    return at


def table_of(dev, caps, page, seed=0, extra=2):
    """A block table over a shuffled pool for sequences of these capacities, and the pool's pages."""
    counts = [-(-c // page) for c in caps]
    perm = torch.randperm(sum(counts) + extra, generator=gen(dev, seed), device=dev).to(torch.int32)
    table = torch.full((len(caps), max(max(counts), 1)), -7, dtype=torch.int32, device=dev)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table, sum(counts) + extra


def bytes_of(x):
    return x.view(torch.uint8)


def pool(dev, pages, Hkv, page, D, seed=0, order="head"):
    """Pools of any bytes and any scales, as freshly allocated memory holds."""
    g = gen(dev, seed)
    shape = (pages, Hkv, page, D) if order == "head" else (pages, page, Hkv, D)
    data = torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.int32).to(torch.uint8).view(E4M3)
    scales = torch.randint(-2 ** 31, 2 ** 31, (pages, Hkv, page), generator=g, device=dev).to(torch.int32)
    return data if order == "head" else data.transpose(1, 2), scales.view(torch.float32)


def rotated64(x, w, cos, sin, eps, rope):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    h = rope // 2
    a, b, rest = x[..., :h], x[..., h:rope], x[..., rope:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], rest], -1)


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("page,order", [(16, "head"), (48, "token"), (64, "head")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm,return_kv", [(False, False), (True, True)])
def test_append(cuda_dev, Hq, Hkv, D, page, order, dtype, norm, return_kv):
    from npu_b200 import rope_append_paged

    dev, lens, starts = cuda_dev, [1, 17, 0, 40, 3], [5, 0, 3, 31, 100]
    rope = D // 2 if norm else D
    N, caps = sum(lens), [s + t for s, t in zip(starts, lens)]
    table, pages = table_of(dev, caps, page)
    (kp, ks), (vp, vs) = (pool(dev, pages, Hkv, page, D, seed, order) for seed in (1, 2))
    before = [bytes_of(kp).clone(), bytes_of(vp).clone(), ks.clone(), vs.clone()]
    g = gen(dev, 3)
    q = torch.randn(N, Hq, D, generator=g, device=dev).to(dtype)
    size = 10.0 ** torch.randint(-6, 4, (N, Hkv, 1), generator=g, device=dev)
    k = (size * torch.randn(N, Hkv, D, generator=g, device=dev)).to(dtype)
    v = (size * torch.randn(N, Hkv, D, generator=g, device=dev)).to(dtype)
    k[0], v[1] = 0, 0
    w = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(dtype) if norm else None
    ang = torch.outer(torch.arange(max(caps), device=dev).float(), torch.rand(rope // 2, generator=g, device=dev))
    cos, sin = torch.cat([ang, ang], -1).cos().to(dtype), torch.cat([ang, ang], -1).sin().to(dtype)
    got_lens = torch.zeros(len(lens), dtype=torch.int32, device=dev)
    got = rope_append_paged(q, k, v, cos, sin, kp, vp, table, ints(dev, offsets(lens)),
                            start_pos_per_batch=ints(dev, starts), seqlens_out=got_lens, q_norm=w, k_norm=w,
                            rope_dim=rope, return_kv=return_kv, k_scales=ks, v_scales=vs)
    assert got_lens.tolist() == caps
    pos = torch.tensor([s + i for s, t in zip(starts, lens) for i in range(t)], device=dev)
    which = torch.tensor([b for b, t in enumerate(lens) for _ in range(t)], device=dev)
    at = table[which, pos // page].long(), pos % page
    touched = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    touched[at] = True
    k64, v64 = rotated64(k, w, cos[pos], sin[pos], 1e-6, rope), v.double()
    for x, codes, scales, old, old_scales in ((k64, kp, ks, before[0], before[2]), (v64, vp, vs, before[1], before[3])):
        s = scales[at[0], :, at[1]].double()
        top = x.abs().amax(-1)
        assert ((s - (top / 448).clamp(min=2.0 ** -100)).abs() <= 2 ** -20 * s).all()
        back = bytes_of(codes)[at[0], :, at[1]].view(E4M3).double() * s[..., None]
        tol = 2 ** -4 * x.abs() * (1 + 2 ** -18) + 2 ** -10 * s[..., None] + 2 ** -19 * top[..., None]
        assert ((back - x).abs() <= tol).all()
        rest = ~touched[:, None, :].expand(pages, Hkv, page)  # every other slot is as it was
        assert torch.equal(bytes_of(codes)[rest], old[rest])
        assert torch.equal(scales[rest].view(torch.int32), old_scales[rest].view(torch.int32))
    # v has no arithmetic before it: the very bits. (Quotients in 64 bits, rounded: torch divides by a number in fp32 as
    # a product with its reciprocal.)
    scale = (v.double().abs().amax(-1) / 448).float().clamp(min=2.0 ** -100)
    assert torch.equal(vs[at[0], :, at[1]], scale)
    codes = (v.float() * (1 / scale.double()).float()[..., None]).to(E4M3)
    assert torch.equal(bytes_of(vp)[at[0], :, at[1]], bytes_of(codes))
    # q, and the packed rows for the prompts' attention, are those of a bf16 cache.
    kp16, vp16 = (torch.zeros(pages, Hkv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    want = rope_append_paged(q, k, v, cos, sin, kp16, vp16, table, ints(dev, offsets(lens)),
                             start_pos_per_batch=ints(dev, starts), q_norm=w, k_norm=w, rope_dim=rope,
                             return_kv=return_kv)
    for a, b in zip(got if return_kv else [got], want if return_kv else [want]):
        assert torch.equal(a, b)


def test_append_what_is_not_finite(cuda_dev):
    """A row with an infinity or a NaN reads back as NaN, its neighbours as they are."""
    from npu_b200 import decode_paged, gather_paged, rope_append_paged

    dev, D = cuda_dev, 64
    v = torch.randn(5, 2, D, generator=gen(dev, 1), device=dev)
    v[0, 0, 3], v[1, 1, 63], v[2, 0, 0] = math.inf, -math.inf, math.nan
    v[3, 0] = 0
    k = torch.randn(5, 2, D, generator=gen(dev, 2), device=dev)
    (kp, ks), (vp, vs) = (pool(dev, 3, 2, 16, D, s) for s in (3, 4))
    table, cu = ints(dev, [[1]]), ints(dev, [0, 5])
    cos, sin = torch.ones(5, D, device=dev), torch.zeros(5, D, device=dev)
    q = torch.randn(5, 4, D, generator=gen(dev, 5), device=dev)
    rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, k_scales=ks, v_scales=vs)
    _, back = gather_paged(kp, vp, table, cu, 5, k_scales=ks, v_scales=vs)
    bad = torch.zeros(5, 2, dtype=torch.bool, device=dev)
    bad[0, 0] = bad[1, 1] = bad[2, 0] = True
    assert back[bad].isnan().all() and back[~bad].isfinite().all()
    assert (back[3, 0] == 0).all()
    # The largest of a row comes back exactly (448 s), rounded to bf16 once.
    top = v[4].abs().amax(-1)
    assert torch.equal(back[4].abs().amax(-1).float(), (448 * (top / 448)).bfloat16().float())
    o = decode_paged(q[:1].bfloat16(), kp, vp, table, ints(dev, [5]), k_scales=ks, v_scales=vs)
    assert o.isnan().all()
    k[4, 0, 0] = math.nan
    rope_append_paged(q, k, v.nan_to_num(1, 1, 1), cos, sin, kp, vp, table, cu, k_scales=ks, v_scales=vs)
    o = decode_paged(q[:1].bfloat16(), kp, vp, table, ints(dev, [5]), k_scales=ks, v_scales=vs)
    assert o[0, :2].isnan().all() and o[0, 2:].isfinite().all()
    o = decode_paged(q[:1].bfloat16(), kp, vp, table, ints(dev, [4]), k_scales=ks, v_scales=vs)
    assert o.isfinite().all()


def cached(dev, lens, Hkv, D, page, seed=0, order="head", width=None):
    """Random 8-bit sequences in pools whose other slots hold anything."""
    table, pages = table_of(dev, lens, page, seed)
    if width:
        table = torch.cat([table, torch.full((len(lens), width - table.shape[1]), -7, dtype=torch.int32, device=dev)], 1)
    out, seqs = [], []
    for s in (1, 2):
        data, scales = pool(dev, pages, Hkv, page, D, seed + s, order)
        g, rows = gen(dev, seed + 10 + s), []
        for b, t in enumerate(lens):
            x = torch.randn(t, Hkv, D, generator=g, device=dev)
            sc = torch.rand(t, Hkv, generator=g, device=dev) * 0.01 + 1e-3
            c = (x / x.abs().amax(-1, keepdim=True) * 448).to(E4M3)
            j = torch.arange(t, device=dev)
            at = table[b, j // page].long(), j % page
            bytes_of(data)[at[0], :, at[1]] = bytes_of(c)
            scales[at[0], :, at[1]] = sc
            rows.append(c.double() * sc.double()[..., None])
        out += [data, scales]
        seqs.append(rows)
    return (*seqs, *out, table)


def check(out, q, ks, vs, scale, gate=None):
    assert torch.isfinite(out).all()
    group = q.shape[1] // ks[0].shape[1]
    for b, (k, v) in enumerate(zip(ks, vs)):
        if k.shape[0] == 0:
            assert (out[b] == 0).all()
            continue
        kk, vv = (x.transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        p = torch.softmax((kk @ q[b].double()[:, :, None]).squeeze(-1) * scale, -1)[:, None]
        o, mean = (p @ vv).squeeze(1), (p @ vv.abs()).squeeze(1)
        if gate is not None:
            o, mean = o * torch.sigmoid(gate[b].double()), mean * torch.sigmoid(gate[b].double())
        tol = 2 ** -14 * mean + 1e-9
        if out.dtype == torch.bfloat16:
            tol = tol * (1 + 2 ** -8) + 2 ** -8 * o.abs()
        d = (out[b].double() - o).abs()
        assert (d <= tol).all(), f"sequence {b}: {(d - tol).max().item()} over the tolerance"


@pytest.mark.parametrize("page,order", [(16, "head"), (48, "token"), (64, "head"), (256, "head")])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_decode(cuda_dev, Hq, Hkv, D, page, order, out_dtype):
    from npu_b200 import decode_paged

    lens = [1, 15, 16, 17, 0, 63, 64, 65, 130, 1000]
    ks, vs, kp, sk, vp, sv, table = cached(cuda_dev, lens, Hkv, D, page, page + D, order)
    q = torch.randn(len(lens), Hq, D, generator=gen(cuda_dev, 1), device=cuda_dev).bfloat16()
    out = decode_paged(q, kp, vp, table, ints(cuda_dev, lens), out_dtype=out_dtype, k_scales=sk, v_scales=sv)
    check(out, q, ks, vs, 1 / math.sqrt(D))


@pytest.mark.parametrize("lens", [[20000], [3, 9000, 1, 700, 0, 12345], [500] * 40, [1] * 200, [0, 700, 33] * 45])
@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 2, 256), (16, 1, 128)])
def test_decode_long_and_many(cuda_dev, lens, Hq, Hkv, D):
    from npu_b200 import decode_paged

    ks, vs, kp, sk, vp, sv, table = cached(cuda_dev, lens, Hkv, D, 64, 5)
    q = torch.randn(len(lens), Hq, D, generator=gen(cuda_dev, 1), device=cuda_dev).bfloat16()
    gate = torch.randn(len(lens), Hq, D, generator=gen(cuda_dev, 2), device=cuda_dev).bfloat16()
    out = decode_paged(q, kp, vp, table, ints(cuda_dev, lens), gate=gate, scale=0.3, k_scales=sk, v_scales=sv)
    check(out, q, ks, vs, 0.3, gate)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_all_codes(cuda_dev, D):
    """Every finite e4m3 number, as a key and as a value, through scales of every size: one key at a time gives its
    value back."""
    from npu_b200 import decode_paged

    dev, n = cuda_dev, 256 // (D // 64) // 4  # D codes a row: n rows of them cover the 256 bytes
    codes = torch.arange(256, device=dev, dtype=torch.int32).repeat(D * 4 * n // 256 + 1)[:4 * n * D]
    codes = torch.where(codes % 128 == 127, codes - 1, codes).to(torch.uint8).view(4 * n, 1, 1, D)
    pages = 4 * n
    kp = codes.expand(pages, 1, 16, D).contiguous().view(E4M3)
    sv = (2.0 ** torch.linspace(-60, 60, pages, device=dev))[:, None, None].expand(pages, 1, 16).contiguous()
    sk = torch.full_like(sv, 2.0 ** -8)
    table = torch.arange(pages, dtype=torch.int32, device=dev)[:, None]
    q = torch.randn(pages, 4, D, generator=gen(dev, 1), device=dev).bfloat16()
    out = decode_paged(q, kp, kp, table, torch.ones(pages, dtype=torch.int32, device=dev), k_scales=sk, v_scales=sv)
    want = kp[:, 0, 0].double() * sv[:, 0, 0].double()[:, None]
    # p = 1 times the scale as two bf16 terms: 2^-16 of it.
    assert ((out.double() - want[:, None]).abs() <= 2 ** -15 * want[:, None].abs()).all()
    # 16 of them at a time, as keys: scores of up to some hundred.
    k64 = kp.view(pages // 4, 4, 16, D)[:, :, 0].double() * 2.0 ** -8
    kp4 = kp.view(pages // 4, 4, 16, D)[:, :, 0].repeat(1, 4, 1).view(pages // 4, 1, 16, D)
    vp4 = torch.randn(pages // 4, 1, 16, D, generator=gen(dev, 2), device=dev).to(E4M3)
    one = torch.ones(pages // 4, 1, 16, device=dev)
    out = decode_paged(q[:pages // 4], kp4.view(torch.uint8).contiguous().view(E4M3), vp4, table[:pages // 4],
                       torch.full((pages // 4,), 4, dtype=torch.int32, device=dev), k_scales=one * 2.0 ** -8,
                       v_scales=one)
    check(out, q[:pages // 4], list(k64[:, :, None]), list(vp4[:, 0, :4].double()[:, :, None]), 1 / math.sqrt(D))


@pytest.mark.parametrize("Hkv,D", [(3, 64), (1, 64), (4, 128), (9, 128), (2, 256)])
@pytest.mark.parametrize("page,order", [(16, "head"), (40, "token"), (64, "head")])
@pytest.mark.parametrize("quant", [True, False])
def test_gather(cuda_dev, Hkv, D, page, order, quant):
    from npu_b200 import gather_paged

    dev, lens, starts = cuda_dev, [1, 0, 33, 100, 7], [0, 4, 39, 1, 64]
    caps = [s + t for s, t in zip(starts, lens)]
    ks, vs, kp, sk, vp, sv, table = cached(dev, caps, Hkv, D, page, 7, order)
    if not quant:
        sk = sv = None
        kp, vp = pool16(dev, table, caps, ks, page, Hkv, D, order), pool16(dev, table, caps, vs, page, Hkv, D, order)
    cu = [3 + c for c in offsets(lens)]  # three rows ahead of the first sequence, two behind the last
    N = cu[-1] + 2
    ko, vo = (torch.full((N, Hkv, D), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    got = gather_paged(kp, vp, table, ints(dev, cu), N, start_pos_per_batch=ints(dev, starts), k_scales=sk, v_scales=sv,
                       k_out=ko, v_out=vo)
    assert got[0].data_ptr() == ko.data_ptr() and got[1].data_ptr() == vo.data_ptr()
    for rows, out in ((ks, ko), (vs, vo)):
        for b, t in enumerate(lens):
            assert torch.equal(out[cu[b]:cu[b + 1]], rows[b][starts[b]:].to(torch.bfloat16)), b
        assert (out[:3] == 7).all() and (out[-2:] == 7).all()


def pool16(dev, table, caps, rows, page, Hkv, D, order):
    """bf16 pools with these rows, NaN elsewhere."""
    pages = int(table.max()) + 1
    shape = (pages, Hkv, page, D) if order == "head" else (pages, page, Hkv, D)
    data = torch.full(shape, math.nan, dtype=torch.bfloat16, device=dev)
    data = data if order == "head" else data.transpose(1, 2)
    for b, t in enumerate(caps):
        j = torch.arange(t, device=dev)
        data[table[b, j // page].long(), :, j % page] = rows[b].to(torch.bfloat16)
    return data


def test_gather_bad_places(cuda_dev):
    """Positions without a page are zeros and reported; offsets that are no stretch leave their sequence out."""
    from npu_b200 import device_error, gather_paged
    from npu_b200._lib import B2A_ERR_DEVICE_BAD_LEN

    dev = cuda_dev
    device_error()
    ks, vs, kp, sk, vp, sv, table = cached(dev, [20, 20], 2, 64, 16, 1)
    table[1, 1] = 1 << 20
    ko, vo = gather_paged(kp, vp, table, ints(dev, [0, 40, 60]), 60, k_scales=sk, v_scales=sv)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    assert torch.equal(ko[:20], ks[0].to(torch.bfloat16)) and (ko[32:40] == 0).all() and (vo[32:40] == 0).all()
    assert torch.equal(vo[40:56], vs[1][:16].to(torch.bfloat16)) and (vo[56:] == 0).all()
    for cu in ([0, 100], [-1, 5], [9, 3]):
        ko, vo = (torch.full((10, 2, 64), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
        gather_paged(kp, vp, table[:1], ints(dev, cu), 10, k_scales=sk, v_scales=sv, k_out=ko, v_out=vo)
        assert device_error() == B2A_ERR_DEVICE_BAD_LEN
        assert (ko == 7).all() and (vo == 7).all()
    gather_paged(kp, vp, table[:1], ints(dev, [0, 5]), 5, start_pos_per_batch=ints(dev, [-3]), k_scales=sk, v_scales=sv)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    assert gather_paged(kp, vp, table[:1], ints(dev, [0, 0]), 0, k_scales=sk, v_scales=sv)[0].shape == (0, 2, 64)
    assert device_error() == 0


def test_decode_bad_pages(cuda_dev):
    from npu_b200 import decode_paged, device_error
    from npu_b200._lib import B2A_ERR_DEVICE_BAD_LEN

    dev = cuda_dev
    device_error()
    ks, vs, kp, sk, vp, sv, table = cached(dev, [20, 700], 2, 64, 16, 1)
    q = torch.randn(2, 4, 64, generator=gen(dev, 1), device=dev).bfloat16()
    bad = table.clone()
    bad[0, 1] = 1 << 20
    out = decode_paged(q, kp, vp, bad, ints(dev, [20, 700]), k_scales=sk, v_scales=sv)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    check(out[1:], q[1:], ks[1:], vs[1:], 1 / 8)
    decode_paged(q, kp, vp, table, ints(dev, [-1, 100000]), k_scales=sk, v_scales=sv)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN


BAD = [
    (dict(k_scales=None), "come together"),
    (dict(k_scales=None, v_scales=None), "need k_scales and v_scales"),
    (dict(kp="bf16"), "k_pages must be float8_e4m3fn"),
    (dict(v_scales="short"), r"v_scales must be a float32 tensor \[5, 2, 16\]"),
    (dict(k_scales="half"), "k_scales must be a float32"),
    (dict(k_scales="host"), "k_scales must be a float32"),
]


@pytest.mark.parametrize("call", ["decode", "append", "gather"])
@pytest.mark.parametrize("which", range(len(BAD)))
def test_refusals(cuda_dev, call, which):
    from npu_b200 import decode_paged, gather_paged, rope_append_paged

    dev = cuda_dev
    ones = torch.ones(5, 2, 16, device=dev)
    swaps = {"bf16": torch.zeros(5, 2, 16, 64, device=dev).bfloat16(), "short": torch.ones(5, 2, 15, device=dev),
             "half": ones.half(), "host": ones.cpu()}
    table, tab = ints(dev, [[0, 1], [2, 3]]), torch.zeros(16, 64, device=dev)

    def run(kp=None, **kw):
        a = dict(k_scales=ones, v_scales=ones)
        a.update({k: swaps.get(v, v) if isinstance(v, str) else v for k, v in kw.items()})
        zero = torch.zeros(5, 2, 16, 64, device=dev).to(E4M3)
        kp = swaps[kp] if kp else zero
        if call == "decode":
            return decode_paged(torch.zeros(2, 4, 64, device=dev).bfloat16(), kp, zero, table, ints(dev, [20, 3]), **a)
        if call == "gather":
            return gather_paged(kp, zero, table, ints(dev, [0, 2, 3]), 3, **a)
        x = torch.zeros(3, 2, 64, device=dev)
        return rope_append_paged(torch.zeros(3, 4, 64, device=dev), x, x, tab, tab, kp, zero, table, ints(dev, [0, 2, 3]),
                                 **a)

    run()
    over, message = BAD[which]
    with pytest.raises(ValueError, match=message):
        run(**over)
    run()
    torch.cuda.synchronize()
