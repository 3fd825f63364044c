"""The serving operators queued one behind another: lengths that the kernel just before wrote, streams other than
the default one, and CUDA graphs. Everything is compared bit for bit with the same calls made one at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cache(dev, B, Hq, Hkv, D, page, width, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).bfloat16()

    n = B * width
    table = torch.randperm(n, generator=g, device=dev).to(torch.int32).view(B, width)
    a = torch.outer(torch.arange(width * page, device=dev), 10000.0 ** -(torch.arange(D, device=dev) % (D // 2) / (D // 2)))
    return dict(k=normal(n, Hkv, page, D), v=normal(n, Hkv, page, D), table=table, cos=a.cos().bfloat16(),
                sin=a.sin().bfloat16(), one_each=torch.arange(B + 1, dtype=torch.int32, device=dev),
                q=normal(B, Hq, D), kv=normal(2, B, Hkv, D))


def step(c, start, end):
    """Append of one token per sequence at `start`, which writes the lengths `end`, and attention by these."""
    from npu_b200 import decode_paged, rope_append_paged

    q = rope_append_paged(c["q"], c["kv"][0], c["kv"][1], c["cos"], c["sin"], c["k"], c["v"], c["table"], c["one_each"],
                          start_pos_per_batch=start, seqlens_out=end)
    return decode_paged(q, c["k"], c["v"], c["table"], end)


@pytest.mark.parametrize("B,Hq,Hkv,D", [(3, 9, 3, 64), (40, 9, 3, 64), (48, 32, 4, 128), (20, 16, 2, 256), (700, 2, 2, 64)])
def test_lengths_written_by_the_kernel_before(cuda_dev, B, Hq, Hkv, D):
    """Steps with other lengths each time, queued without a pause, in one buffer of lengths."""
    from npu_b200 import device_error

    c = cache(cuda_dev, B, Hq, Hkv, D, 64, 32)
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    starts = torch.randint(0, 2048, (30, B), dtype=torch.int32, generator=g, device=cuda_dev)
    starts[::5] = 0
    starts[1::5] = 2047
    end = torch.zeros(B, dtype=torch.int32, device=cuda_dev)
    first = [step(c, s, end) for s in starts]  # also writes every slot that later steps write, with the same values
    expected = []
    for s in starts:
        expected.append(step(c, s, end))
        torch.cuda.synchronize()
    queued = [step(c, s, end) for s in starts]
    torch.cuda.synchronize()
    assert len(first) == 30 and device_error() == 0
    for a, b in zip(expected, queued):
        assert torch.equal(a, b)


def calls(dev):
    """The four operators on fixed inputs, as functions without arguments that return tensors."""
    from npu_b200 import prefill_varlen, rope_append_paged, sample

    c = cache(dev, 24, 9, 3, 64, 32, 40)
    start = torch.arange(0, 24 * 50, 50, dtype=torch.int32, device=dev)
    end = torch.zeros_like(start)
    g = torch.Generator(device=dev).manual_seed(2)
    lens = torch.tensor([0, 300, 1, 129, 700], device=dev).cumsum(0).to(torch.int32)
    out = {}
    for D, H in [(64, (9, 3)), (128, (4, 4)), (256, (4, 1))]:
        q = torch.randn(1130, H[0], D, generator=g, device=dev).bfloat16()
        kv = torch.randn(2, 1130, H[1], D, generator=g, device=dev).bfloat16()
        out[f"prefill {D}"] = lambda q=q, kv=kv: prefill_varlen(q, kv[0], kv[1], lens)
    x = torch.randn(6, 40_001, generator=g, device=dev)
    e = torch.empty_like(x).exponential_(generator=g)
    out["sample"] = lambda: sample(x, e, temperature=0.9, top_k=200, top_p=0.9)
    out["append"] = lambda: rope_append_paged(c["q"], c["kv"][0], c["kv"][1], c["cos"], c["sin"], c["k"], c["v"],
                                              c["table"], c["one_each"], start_pos_per_batch=start, seqlens_out=end)
    out["append and decode"] = lambda: step(c, start, end)
    return out


def test_on_another_stream(cuda_dev):
    for name, call in calls(cuda_dev).items():
        expected = call()
        side = torch.cuda.Stream(cuda_dev)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [call() for _ in range(3)]
        side.synchronize()
        for t in got:
            assert torch.equal(t, expected), name


def test_in_a_cuda_graph(cuda_dev):
    every = calls(cuda_dev)
    expected = {name: call() for name, call in every.items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = {name: call() for name, call in every.items()}
    for _ in range(3):
        for t in got.values():
            t.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for name, t in got.items():
        assert torch.equal(t, expected[name]), name
