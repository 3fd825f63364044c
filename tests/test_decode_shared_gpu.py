"""Single-token attention for sequences that share a prefix against a plain form in 64 bits.

Tolerance per element: over the shared keys P is rounded to bf16 for the tensor cores, by 2^-8 of itself at most, and
everything else is fp32 sums or two bf16 terms (2^-14 of the mean): (2^-8 + 2^-14) of the softmax-weighted mean of |v|;
a bf16 output adds 2^-8 of its value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def ints(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def build(dev, groups, Hkv, D, page, seed=0, order="head", fill=math.nan, width=None):
    """groups: [(prefix, [own keys of each sequence])]. The prefix's whole pages are shared, the rest of it is copied
    to every sequence's next page, as a cache that shares pages has it. Slots that no sequence has hold `fill`.
    Returns k and v per sequence, pools, table, seqlens, prefix_lens, cu_groups."""
    g = gen(dev, seed)
    rows, tables, n = [], [], 0
    need = sum(p // page + sum(-(-(p % page + t) // page) for t in own) for p, own in groups) + 2
    perm = torch.randperm(need, generator=g, device=dev).tolist()
    shape = (need, Hkv, page, D) if order == "head" else (need, page, Hkv, D)
    pools = [torch.full(shape, fill, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    pools = pools if order == "head" else [x.transpose(1, 2) for x in pools]
    lens = []
    for prefix, own in groups:
        shared, n = perm[n:n + prefix // page], n + prefix // page
        head = [torch.randn(prefix, Hkv, D, generator=g, device=dev).bfloat16() for _ in range(2)]
        for t in own:
            count = -(-(prefix % page + t) // page)
            tables.append(shared + perm[n:n + count])
            n += count
            kv = [torch.cat([h, torch.randn(t, Hkv, D, generator=g, device=dev).bfloat16()]) for h in head]
            rows.append(kv)
            lens.append(prefix + t)
            j = torch.arange(prefix + t, device=dev)
            at = torch.tensor(tables[-1], device=dev, dtype=torch.long)
            if len(j):
                for pool, x in zip(pools, kv):
                    pool[at[j // page], :, j % page] = x
    table = torch.full((len(tables), width or max(max(len(t) for t in tables), 1)), -5, dtype=torch.int32, device=dev)
    for b, t in enumerate(tables):
        table[b, :len(t)] = ints(dev, t)
    at = [0]
    for _, own in groups:
        at.append(at[-1] + len(own))
    return ([r[0] for r in rows], [r[1] for r in rows], *pools, table, ints(dev, lens),
            ints(dev, [p for p, _ in groups]), ints(dev, at))


def check(out, q, ks, vs, scale, gate=None, exact_p=False):
    assert torch.isfinite(out).all()
    group = q.shape[1] // ks[0].shape[1]
    for b, (k, v) in enumerate(zip(ks, vs)):
        if k.shape[0] == 0:
            assert (out[b] == 0).all()
            continue
        kk, vv = (x.double().transpose(0, 1) for x in (k, v))
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q[b].double().unflatten(0, (-1, group)), kk) * scale, -1)
        o, mean = (p @ vv).flatten(0, 1), (p @ vv.abs()).flatten(0, 1)
        if gate is not None:
            o, mean = o * torch.sigmoid(gate[b].double()), mean * torch.sigmoid(gate[b].double())
        tol = (2 ** -14 if exact_p else 2 ** -8 + 2 ** -14) * mean + 1e-7
        if out.dtype == torch.bfloat16:
            tol = tol * (1 + 2 ** -8) + 2 ** -8 * o.abs()
        d = (out[b].double() - o).abs()
        assert (d <= tol).all(), f"sequence {b}: {(d - tol).max().item()} over the tolerance"


def shared(*args, **kw):
    """The call, sharing whatever there is to share: these sizes are far below where it pays."""
    from npu_b200 import decode_paged_shared

    return decode_paged_shared(*args, **{"min_saved_bytes": 0, **kw})


HEADS = [(9, 3, 64), (16, 1, 64), (32, 4, 128), (5, 5, 128), (16, 2, 256), (7, 1, 256)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("page,order", [(16, "head"), (48, "token"), (64, "head"), (256, "head")])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_groups(cuda_dev, Hq, Hkv, D, page, order, out_dtype):
    from npu_b200 import device_error

    device_error()
    groups = [(700, [1, 30, 64, 0, 500]), (64, [10, 3]), (63, [5, 6, 900]), (1200, [7]), (0, [40, 0]),
              (129, list(range(1, 46))), (256, [0] * 3)]
    ks, vs, kp, vp, table, lens, pre, cu = build(cuda_dev, groups, Hkv, D, page, page + D, order)
    q = torch.randn(len(ks), Hq, D, generator=gen(cuda_dev, 1), device=cuda_dev).bfloat16()
    out = shared(q, kp, vp, table, lens, pre, cu, out_dtype=out_dtype)
    check(out, q, ks, vs, 1 / math.sqrt(D))
    assert device_error() == 0


@pytest.mark.parametrize("prefix,own", [(20000, [100] * 5), (5000, [1] * 200), (16384, [0, 1, 3000]),
                                        (640, [2000, 3, 70] * 30), (64, [600] * 2)])
@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 2, 256), (8, 8, 64)])
def test_one_group(cuda_dev, prefix, own, Hq, Hkv, D):
    ks, vs, kp, vp, table, lens, pre, _ = build(cuda_dev, [(prefix, own)], Hkv, D, 64, 3)
    q = torch.randn(len(ks), Hq, D, generator=gen(cuda_dev, 1), device=cuda_dev).bfloat16()
    gate = torch.randn(len(ks), Hq, D, generator=gen(cuda_dev, 2), device=cuda_dev)
    out = shared(q, kp, vp, table, lens, pre, scale=0.2, gate=gate)
    check(out, q, ks, vs, 0.2, gate)


def test_sharp_scores(cuda_dev):
    """Maxima that move from block to block, and rows that one key decides."""
    for Hq, Hkv, D in ((9, 3, 64), (32, 4, 128), (16, 2, 256)):
        ks, vs, kp, vp, table, lens, pre, _ = build(cuda_dev, [(2048, [300, 5, 64] * 5)], Hkv, D, 64, 4)
        q = torch.randn(len(ks), Hq, D, generator=gen(cuda_dev, 1), device=cuda_dev).bfloat16()
        out = shared(q, kp, vp, table, lens, pre, scale=3.0)
        check(out, q, ks, vs, 3.0)


def test_short_and_lone_sequences(cuda_dev):
    """Sequences without all of the prefix attend by themselves: the others' keys (NaN, or far larger) do not reach
    them; nor does a sequence outside every group."""
    from npu_b200 import device_error

    dev = cuda_dev
    device_error()
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(1000, [50, 60, 70, 80, 90, 20])], 2, 128, 64, 5)
    short = {1: 100, 3: 0, 4: 959}  # eff is 960
    for b, t in short.items():
        lens[b] = t
        ks[b], vs[b] = ks[b][:t], vs[b][:t]
    page = int(table[0, 14])  # keys 896 .. 959 of the prefix
    vp[page, :, 63] = math.nan
    q = torch.randn(6, 8, 128, generator=gen(dev, 1), device=dev).bfloat16()
    out = shared(q, kp, vp, table, lens, pre, ints(dev, [0, 5]))
    check(out[[1, 3, 4]], q[[1, 3, 4]], [ks[b] for b in (1, 3, 4)], [vs[b] for b in (1, 3, 4)], 128 ** -0.5,
          exact_p=True)
    assert out[[0, 2, 5]].isnan().all()
    assert device_error() == 0
    # Nobody has all of it: nothing is shared, and the entries past their pages are not read.
    lens.fill_(700)
    table[:, 11:] = -1
    out = shared(q, kp, vp, table, lens, pre)
    for b in range(6):
        src = 0 if b in short else b
        ks[b], vs[b] = ks[src][:700], vs[src][:700]
    check(out, q, ks, vs, 128 ** -0.5, exact_p=True)
    assert device_error() == 0


def test_rows_beside_a_nan(cuda_dev):
    """NaN in one sequence's query stays there."""
    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(640, [50, 60, 70]), (640, [1, 2])], 3, 64, 64, 5)
    q = torch.randn(5, 9, 64, generator=gen(dev, 1), device=dev).bfloat16()
    q[1, 4] = math.nan
    q[3] = math.inf
    out = shared(q, kp, vp, table, lens, pre, cu)
    assert out[1, 4].isnan().all() and out[3].isnan().all()
    keep = [0, 2, 4]
    check(out[keep], q[keep], [ks[b] for b in keep], [vs[b] for b in keep], 1 / 8)
    rest = torch.tensor([h for h in range(9) if h != 4], device=dev)
    one = q[1:2].clone()
    one[:, 4] = 0
    check(torch.where(out[1:2].isnan(), 0, out[1:2])[:, rest], one[:, rest].contiguous(),
          [ks[1].repeat_interleave(3, 1)[:, rest]], [vs[1].repeat_interleave(3, 1)[:, rest]], 1 / 8)


def test_bad_groups(cuda_dev):
    """Offsets that are no stretch of the sequences, groups that overlap, prefixes and pages out of range: reported, in
    bounds, and right wherever nothing wrong is said of a sequence."""
    from npu_b200 import device_error
    from npu_b200._lib import B2A_ERR_DEVICE_BAD_LEN

    dev = cuda_dev
    device_error()
    ks, vs, kp, vp, table, lens, pre, _ = build(dev, [(640, [50, 60, 70, 80])], 2, 64, 64, 5)
    q = torch.randn(4, 8, 64, generator=gen(dev, 1), device=dev).bfloat16()
    for cu in ([0, 9], [-1, 4], [3, 1]):
        out = shared(q, kp, vp, table, lens, pre, ints(dev, cu))
        assert device_error() == B2A_ERR_DEVICE_BAD_LEN
        check(out, q, ks, vs, 1 / 8, exact_p=True)
    out = shared(q, kp, vp, table, lens, ints(dev, [640] * 5), ints(dev, [0, 4, 0, 4, 0, 4]))
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    check(out, q, ks, vs, 1 / 8)
    out = shared(q, kp, vp, table, lens, ints(dev, [-64]))
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    check(out, q, ks, vs, 1 / 8, exact_p=True)
    shared(q, kp, vp, table, lens, ints(dev, [1 << 30]))
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN
    bad = table.clone()
    bad[:, 2] = 1 << 20
    shared(q, kp, vp, bad, lens, pre)
    assert device_error() == B2A_ERR_DEVICE_BAD_LEN


def test_same_as_paged(cuda_dev):
    """Short tables and single sequences go to decode_paged: the same bits."""
    from npu_b200 import decode_paged

    dev = cuda_dev
    for groups in ([(240, [1, 40, 7])], [(3000, [5])]):
        ks, vs, kp, vp, table, lens, pre, _ = build(dev, groups, 3, 64, 16, 1)
        q = torch.randn(len(ks), 9, 64, generator=gen(dev, 1), device=dev).bfloat16()
        assert torch.equal(shared(q, kp, vp, table, lens, pre), decode_paged(q, kp, vp, table, lens))


def test_streams_workspaces_and_graphs(cuda_dev):
    """Another stream, a given workspace at any 16-byte place, a captured call replayed with other lengths, outputs of
    other strides."""
    from npu_b200.api import decode_paged_shared_workspace_bytes

    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(900, [50, 60, 70]), (640, [1, 2, 400])], 4, 128, 64, 6)
    q = torch.randn(6, 32, 128, generator=gen(dev, 1), device=dev).bfloat16()
    need = decode_paged_shared_workspace_bytes(6, 32, 4, 128, 2)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=dev)
    big = torch.full((6, 40, 128), 7.0, device=dev)
    with pytest.raises(ValueError):
        shared(q, kp, vp, table, lens, pre, cu, workspace=ws[:need - 1])
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        shared(q, kp, vp, table, lens, pre, cu, workspace=ws[16:], out=big[:, 4:36])
    torch.cuda.current_stream(dev).wait_stream(side)
    check(big[:, 4:36], q, ks, vs, 128 ** -0.5)
    assert (big[:, :4] == 7).all() and (big[:, 36:] == 7).all()
    graph = torch.cuda.CUDAGraph()
    static = q.clone()
    with torch.cuda.graph(graph):
        got = shared(static, kp, vp, table, lens, pre, cu)
    for change in range(3):
        if change == 1:
            lens[1], pre[0], cu[0] = 900, 300, 1
            ks[1], vs[1] = ks[1][:900], vs[1][:900]
        if change == 2:
            static.copy_(q.flip(0))
        graph.replay()
        check(got, static, ks, vs, 128 ** -0.5)


BAD = [
    (lambda d: dict(pre=ints(d, [1, 2])), "prefix_lens must be .* 1"),
    (lambda d: dict(pre=torch.zeros(1, dtype=torch.int64, device=d)), "prefix_lens"),
    (lambda d: dict(cu=ints(d, [0])), "two offsets"),
    (lambda d: dict(cu=ints(d, [0, 1, 2])), "prefix_lens must be .* 2"),
    (lambda d: dict(cu=torch.zeros(2, dtype=torch.int64, device=d)), "cu_groups"),
    (lambda d: dict(lens=ints(d, [1, 2, 3])), "seqlens"),
    (lambda d: dict(kp=torch.zeros(60, 2, 16, 64, device=d).to(torch.float8_e4m3fn)), "k_pages must be bfloat16"),
    (lambda d: dict(workspace=torch.zeros(3, dtype=torch.uint8, device=d)), r"at least \d+ bytes"),
    (lambda d: dict(out_dtype=torch.float16), "out_dtype must be"),
    (lambda d: dict(min_saved_bytes=-1), "min_saved_bytes must not be negative, got -1"),
]


@pytest.mark.parametrize("which", range(len(BAD)))
def test_refused(cuda_dev, which):
    def call(**over):
        dev = cuda_dev
        a = dict(q=torch.zeros(2, 4, 64, device=dev).bfloat16(), kp=torch.zeros(60, 2, 16, 64, device=dev).bfloat16(),
                 vp=torch.zeros(60, 2, 16, 64, device=dev).bfloat16(),
                 table=torch.arange(60, dtype=torch.int32, device=dev).view(1, 60).expand(2, 60).contiguous(),
                 lens=ints(dev, [700, 690]), pre=ints(dev, [640]), cu=None)
        kw = {k: over.pop(k) for k in list(over) if k not in a}
        a.update(over)
        return shared(*a.values(), **kw)

    over, message = BAD[which]
    call()
    with pytest.raises(ValueError, match=message):
        call(**over(cuda_dev))
    call()
    torch.cuda.synchronize()


def test_empty(cuda_dev):
    pool = torch.zeros(3, 2, 16, 64, device=cuda_dev).bfloat16()
    out = shared(torch.zeros(0, 4, 64, device=cuda_dev).bfloat16(), pool, pool,
                              torch.zeros(0, 50, dtype=torch.int32, device=cuda_dev), ints(cuda_dev, []),
                              ints(cuda_dev, [64]))
    assert out.shape == (0, 4, 64)


def test_what_saves_too_little_is_not_shared(cuda_dev):
    """Below min_saved_bytes every sequence attends by itself (P in two bf16 terms), from it on they share."""
    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(640, [50, 60, 70]), (1280, [1, 2, 400, 9])], 4, 128, 64, 6)
    q = torch.randn(7, 32, 128, generator=gen(dev, 1), device=dev).bfloat16()
    saved = (2 * 640 + 3 * 1280) * 4 * 128 * 4
    alone = shared(q, kp, vp, table, lens, pre, cu, min_saved_bytes=saved + 4 * 128 * 4)
    check(alone, q, ks, vs, 128 ** -0.5, exact_p=True)
    together = shared(q, kp, vp, table, lens, pre, cu, min_saved_bytes=saved)
    check(together, q, ks, vs, 128 ** -0.5)
    assert torch.equal(alone, shared(q, kp, vp, table, lens, pre, cu, min_saved_bytes=None))
    assert not torch.equal(alone, together)
    assert torch.equal(together, shared(q, kp, vp, table, lens, pre, cu))
