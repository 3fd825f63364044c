"""The later serving operators where calls meet: other streams, captured steps, two calls at once, many groups, pools
whose offsets pass 32 bits. What each computes is tested in files of its own; here the same calls must give the same."""
import pytest
import torch

from test_decode_shared_gpu import build, check, shared
from test_quant_cache_gpu import E4M3, bytes_of, cached, gen, ints, offsets

pytestmark = pytest.mark.gpu


def step(st):
    """One token of every sequence: append to an 8-bit cache, attend, penalise, choose."""
    from npu_b200 import decode_paged, penalize, rope_append_paged, sample

    q = rope_append_paged(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["kp"], st["vp"], st["table"], st["cu"],
                          start_pos_per_batch=st["start"], seqlens_out=st["lens"], k_scales=st["ks"], v_scales=st["vs"])
    o = decode_paged(q, st["kp"], st["vp"], st["table"], st["lens"], k_scales=st["ks"], v_scales=st["vs"])
    logits = o.flatten(1) @ st["w"]
    penalize(logits, st["tokens"], st["count"], repetition=1.3, frequency=0.1, bias=st["bias"], out=logits)
    return o, logits, sample(logits, st["noise"], temperature=0.8, top_k=20)


def state(dev, seed, B=5, Hq=8, Hkv=2, D=64, V=1000):
    g = gen(dev, seed)
    lens = [40, 1, 100, 64, 17][:B]
    ks, vs, kp, sk, vp, sv, table = cached(dev, [t + 8 for t in lens], Hkv, D, 16, seed)
    ang = torch.outer(torch.arange(128, device=dev).float(), torch.rand(D // 2, generator=g, device=dev))
    return dict(q=torch.randn(B, Hq, D, generator=g, device=dev), k=torch.randn(B, Hkv, D, generator=g, device=dev),
                v=torch.randn(B, Hkv, D, generator=g, device=dev), cos=torch.cat([ang, ang], -1).cos(),
                sin=torch.cat([ang, ang], -1).sin(), kp=kp, vp=vp, ks=sk, vs=sv, table=table,
                cu=torch.arange(B + 1, dtype=torch.int32, device=dev), start=ints(dev, lens),
                lens=torch.zeros(B, dtype=torch.int32, device=dev),
                w=torch.randn(Hq * D, V, generator=g, device=dev), bias=torch.randn(V, generator=g, device=dev),
                tokens=torch.randint(0, V, (B, 30), generator=g, device=dev), count=ints(dev, [30, 0, 7, 30, 1][:B]),
                noise=torch.empty(B, V, device=dev).exponential_(generator=g))


def test_a_captured_step(cuda_dev):
    """The whole step in one graph, replayed with other inputs, gives what the calls give one by one."""
    st = state(cuda_dev, 1)
    want = {}
    for seed in (1, 2):  # what the calls give for either set of inputs
        own = state(cuda_dev, seed)
        want[seed] = [x.clone() for x in step(own)] + [bytes_of(own["kp"]).clone(), own["ks"].view(torch.int32).clone()]
    step(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(st)
    for seed in (2, 1, 2):
        for name, x in state(cuda_dev, seed).items():
            (bytes_of(st[name]) if x.dtype == E4M3 else st[name]).copy_(bytes_of(x) if x.dtype == E4M3 else x)
        graph.replay()
        now = list(got) + [bytes_of(st["kp"]), st["ks"].view(torch.int32)]
        assert all(torch.equal(a, b) for a, b in zip(now, want[seed])), seed


def test_steps_on_two_streams_at_once(cuda_dev):
    """Two batches with a cache each, on streams of their own, while the default stream is busy."""
    want = [[x.clone() for x in step(state(cuda_dev, seed))] for seed in (1, 2)]
    states, got = [state(cuda_dev, seed) for seed in (1, 2)], [None, None]
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    busy = torch.randn(4096, 4096, device=cuda_dev)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(cuda_dev))
    for _ in range(10):
        busy = busy @ busy * 1e-3
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(states[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_shared_prefixes_on_two_streams_at_once(cuda_dev):
    dev, calls = cuda_dev, []
    for seed, groups in ((1, [(900, [50, 60, 70]), (640, [1, 2, 400])]), (2, [(5000, [3] * 40)])):
        ks, vs, kp, vp, table, lens, pre, cu = build(dev, groups, 4, 128, 64, seed)
        q = torch.randn(len(ks), 32, 128, generator=gen(dev, seed), device=dev).bfloat16()
        calls.append((q, kp, vp, table, lens, pre, cu))
    want = [shared(*c) for c in calls]
    streams = [torch.cuda.Stream(dev) for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    got = []
    for _ in range(20):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(shared(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


def test_shared_prefixes_again_and_again(cuda_dev):
    """Calls that follow one another without a pause, each with other lengths, sharing one workspace."""
    from npu_b200.api import decode_paged_shared_workspace_bytes

    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(1500, [50, 60, 70, 9]), (640, [1, 2, 400])], 3, 64, 16, 4)
    q = torch.randn(7, 9, 64, generator=gen(dev, 1), device=dev).bfloat16()
    ws = torch.empty(decode_paged_shared_workspace_bytes(7, 9, 3, 64, 2), dtype=torch.uint8, device=dev)
    cut = [[0] * 7, [40, 0, 69, 3, 0, 1, 399], [49, 700, 70, 9, 1, 2, 20], [1549, 3, 0, 0, 600, 0, 0]]
    some = [lens - ints(dev, c) for c in cut]
    want = [shared(q, kp, vp, table, s, pre, cu, workspace=torch.empty_like(ws)) for s in some]
    torch.cuda.synchronize()
    got = [shared(q, kp, vp, table, some[i % 4], pre, cu, workspace=ws) for i in range(200)]
    assert all(torch.equal(x, want[i % 4]) for i, x in enumerate(got))
    for s, x in zip(some, want):
        n = s.tolist()
        check(x, q, [k[:t] for k, t in zip(ks, n)], [v[:t] for v, t in zip(vs, n)], 1 / 8)


@pytest.mark.parametrize("groups,size,prefix", [(40, 3, 130), (300, 2, 70), (1300, 2, 64)])
def test_many_groups(cuda_dev, groups, size, prefix):
    """More groups than a warp reads at once, than the plan has threads, than it keeps in shared memory."""
    from npu_b200 import device_error

    dev = cuda_dev
    device_error()
    own = [(prefix + g % 70, [(g + 3 * i) % 5 for i in range(size)]) for g in range(groups)]
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, own, 1, 64, 16, 3, width=33)
    q = torch.randn(len(ks), 2, 64, generator=gen(dev, 1), device=dev).bfloat16()
    out = shared(q, kp, vp, table, lens, pre, cu)
    assert device_error() == 0
    more = torch.randint(0, len(ks), (200,), generator=torch.Generator().manual_seed(1))
    pick = sorted({0, 1, len(ks) - 1, *more.tolist()})
    check(out[pick], q[pick], [ks[b] for b in pick], [vs[b] for b in pick], 1 / 8)


def test_one_large_group(cuda_dev):
    """More sequences than the plan has threads, several row blocks, most sequences without keys of their own."""
    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(700, [0, 0, 1] * 200)], 2, 64, 64, 3)
    lens[5], lens[599] = 3, 0
    ks[5], vs[5], ks[599], vs[599] = ks[5][:3], vs[5][:3], ks[599][:0], vs[599][:0]
    q = torch.randn(600, 8, 64, generator=gen(dev, 1), device=dev).bfloat16()
    out = shared(q, kp, vp, table, lens, pre)
    pick = [0, 1, 2, 5, 31, 32, 63, 64, 255, 256, 257, 511, 512, 597, 598, 599]
    check(out[pick], q[pick], [ks[b] for b in pick], [vs[b] for b in pick], 1 / 8)


@pytest.mark.parametrize("quant", [True, False])
def test_pools_past_32_bits(cuda_dev, quant):
    """Pools of over 2^32 elements: append, attend and read back in their last pages."""
    from npu_b200 import decode_paged, gather_paged, rope_append_paged

    dev, Hkv, page, D, pages = cuda_dev, 8, 64, 256, 33000
    shape = (pages, Hkv, page, D)
    dtype = E4M3 if quant else torch.bfloat16
    kp, vp = (torch.empty(shape, dtype=dtype, device=dev) for _ in range(2))
    assert kp.numel() > 2 ** 32
    scales = {}
    if quant:
        scales = dict(k_scales=torch.ones(shape[:3], device=dev), v_scales=torch.ones(shape[:3], device=dev))
    lens = [100, 70]
    table = ints(dev, [[pages - 1, 7], [pages - 2, pages - 5]])
    N, g = sum(lens), gen(dev, 1)
    q = torch.randn(N, 8, D, generator=g, device=dev)
    k, v = (torch.randn(N, Hkv, D, generator=g, device=dev) for _ in range(2))
    cos, sin, cu = torch.ones(128, D, device=dev), torch.zeros(128, D, device=dev), ints(dev, offsets(lens))
    q = rope_append_paged(q, k, v, cos, sin, kp, vp, table, cu, **scales)
    back = gather_paged(kp, vp, table, cu, N, **scales)
    for x, y in zip((k, v), back):
        tol = x.abs() * 2 ** -4 * 1.01 + 2 ** -9 * x.abs().amax(-1, keepdim=True) if quant else x.abs() * 2 ** -8
        assert ((x - y.float()).abs() <= tol).all()
    last = torch.tensor([99, 169], device=dev)
    o = decode_paged(q[last], kp, vp, table, ints(dev, lens), **scales)
    rows = []
    for pool, scale in ((kp, scales.get("k_scales")), (vp, scales.get("v_scales"))):
        rows.append([])
        for b, n in enumerate(lens):
            j = torch.arange(n, device=dev)
            at = table[b, j // page].long(), j % page
            x = bytes_of(pool)[at[0], :, at[1]].view(E4M3).double() if quant else pool[at[0], :, at[1]].double()
            rows[-1].append(x * scale[at[0], :, at[1]].double()[..., None] if quant else x)
    check(o, q[last], *rows, 1 / 16, exact_p=True)


def test_a_table_that_names_one_page_for_ever(cuda_dev):
    """A sequence of 300000 keys whose table repeats a few pages (a test of long walks, not of memory)."""
    from npu_b200 import decode_paged

    dev, Hkv, D, page, n = cuda_dev, 1, 64, 64, 300000
    ks, vs, kp, sk, vp, sv, table = cached(dev, [256], Hkv, D, page, 2)
    wide = table[:, :4].repeat(1, -(-n // 256))
    q = torch.randn(1, 4, D, generator=gen(dev, 1), device=dev).bfloat16()
    long = decode_paged(q, kp, vp, wide, ints(dev, [n // 256 * 256]), k_scales=sk, v_scales=sv)
    short = decode_paged(q, kp, vp, table, ints(dev, [256]), k_scales=sk, v_scales=sv)
    # The same keys again and again are the same average: sums of 300000 terms in fp32 parts of some thousands.
    assert ((long - short).abs() <= 2 ** -12 * vs[0].abs().amax()).all()


@pytest.mark.parametrize("captured", [False, True])
def test_shared_steps_that_grow(cuda_dev, captured):
    """Steps that follow one another without a pause, each right behind the append that writes the lengths it reads:
    what the same steps give when the device has come to rest after every call."""
    from npu_b200 import rope_append_paged

    dev, Hq, Hkv, D, page, steps = cuda_dev, 9, 3, 64, 16, 60
    own = [50, 60, 70, 9, 1, 33, 64]
    total = [640 + t + steps for t in own]

    def start_state():
        ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(640, [t + steps for t in own])], Hkv, D, page, 6, fill=0.0)
        g = gen(dev, 2)
        ang = torch.outer(torch.arange(max(total), device=dev).float(), torch.rand(D // 2, generator=g, device=dev))
        ang = torch.cat([ang, ang], -1)
        return dict(kp=kp, vp=vp, table=table, pre=pre, cos=ang.cos(), sin=ang.sin(), start=ints(dev, [640 + t for t in own]),
                    lens=torch.zeros(len(own), dtype=torch.int32, device=dev),
                    each=torch.arange(len(own) + 1, dtype=torch.int32, device=dev),
                    qkv=torch.randn(len(own), Hq + 2 * Hkv, D, generator=g, device=dev))

    def one(st, rest=lambda: None):
        q = rope_append_paged(st["qkv"][:, :Hq], st["qkv"][:, Hq:Hq + Hkv], st["qkv"][:, Hq + Hkv:], st["cos"], st["sin"],
                              st["kp"], st["vp"], st["table"], st["each"], start_pos_per_batch=st["start"],
                              seqlens_out=st["lens"])
        rest()
        o = shared(q, st["kp"], st["vp"], st["table"], st["lens"], st["pre"])
        rest()
        st["start"].add_(1)
        st["qkv"].mul_(0.99).add_(o.mean() * 1e-3)
        rest()
        return o

    st = start_state()
    want = [one(st, torch.cuda.synchronize).clone() for _ in range(steps)]
    st, got = start_state(), []
    if captured:
        first = {x: y.clone() for x, y in st.items()}
        one(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = one(st)
        for x, y in first.items():
            st[x].copy_(y)
        for _ in range(steps):
            graph.replay()
            got.append(o.clone())
    else:
        got = [one(st) for _ in range(steps)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert st["lens"].tolist() == total


@pytest.mark.parametrize("dims", [(0,), (1,), (0, 1)])
def test_shared_prefix_queries_that_are_one(cuda_dev, dims):
    """Queries expanded over the sequences or the heads, as decode_paged takes them."""
    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, cu = build(dev, [(900, [50, 60, 70]), (640, [1, 2, 400])], 2, 64, 64, 5)
    q = torch.randn(*[1 if i in dims else n for i, n in enumerate((6, 8))], 64, generator=gen(dev, 1), device=dev)
    q = q.bfloat16().expand(6, 8, 64)
    check(shared(q, kp, vp, table, lens, pre, cu), q, ks, vs, 1 / 8)


def test_penalize_into_its_bias(cuda_dev):
    from npu_b200 import penalize

    x = torch.randn(4, 1000, device=cuda_dev)
    with pytest.raises((ValueError, RuntimeError)):
        penalize(x, bias=x, out=x)
    with pytest.raises((ValueError, RuntimeError)):
        penalize(x.clone(), bias=x[1], out=x)
