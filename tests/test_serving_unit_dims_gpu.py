"""A dim of one element has any stride in torch, and none matters: the same bits as from contiguous tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def odd(x):
    """x with stride 3 in every dim of one element (but the last)."""
    strides = [3 if n == 1 and i + 1 < x.dim() else s for i, (n, s) in enumerate(zip(x.shape, x.stride()))]
    return x.as_strided(x.shape, strides)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("pages,width", [(1, 1), (40, 40)])
def test_one_kv_head_one_sequence(cuda_dev, D, quant, pages, width):
    from npu_b200 import decode_paged, decode_paged_shared, gather_paged, prefill_varlen, rope_append_paged

    dev, page, n = cuda_dev, 16, width * 16 - 5
    k, v = (torch.randn(n, 1, D, generator=gen(dev, s), device=dev) for s in (1, 2))
    cos, sin = torch.ones(n, D, device=dev), torch.zeros(n, D, device=dev)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, cu, lens = torch.arange(width, dtype=torch.int32, device=dev)[None], ints([0, n]), ints([n])
    got = []
    for f in (lambda x: x, odd):
        pools = [f(torch.zeros(pages, 1, page, D, device=dev).to(E4M3 if quant else torch.bfloat16)) for _ in range(2)]
        scales = [f(torch.zeros(pages, 1, page, device=dev)) for _ in range(2)]
        kw = dict(k_scales=scales[0], v_scales=scales[1]) if quant else {}
        q = torch.randn(n, 1, D, generator=gen(dev, 3), device=dev)
        rot, kp, vp = rope_append_paged(f(q), f(k), f(v), cos, sin, *pools, table, cu, return_kv=True, **kw)
        rows = gather_paged(*pools, table, cu, n, **kw)
        last = f(rot[-1:].contiguous())
        out = decode_paged(last, *pools, table, lens, gate=f(torch.ones_like(last)), **kw)
        got.append([rot, kp, vp, *rows, out, prefill_varlen(f(rot), f(kp), f(vp), cu)])
        if not quant:
            got[-1].append(decode_paged_shared(last, *pools, table, lens, lens // 2, min_saved_bytes=0))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("B,width", [(1, 40), (3, 1), (1, 1)])
def test_tables_of_one_row_or_column(cuda_dev, quant, B, width):
    from npu_b200 import decode_paged, decode_paged_shared, gather_paged, rope_append_paged

    dev, page, D, n = cuda_dev, 16, 64, width * 16 - 5
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width)
    # Strides (1, 1) of one row, as a column's transpose may have, and (1, 5) of one column.
    other = table.clone().as_strided((B, width), (1, 1) if width > 1 else (1, 5))
    assert other.stride() != table.stride()
    cu, lens = ints([n * b for b in range(B + 1)]), ints([n] * B)
    x = torch.randn(B * n, 2, D, generator=gen(dev, 1), device=dev)
    cos, sin = torch.ones(n, D, device=dev), torch.zeros(n, D, device=dev)
    got = []
    for t in (table, other):
        pools = [torch.zeros(B * width, 2, page, D, device=dev).to(E4M3 if quant else torch.bfloat16) for _ in range(2)]
        kw = {f"{y}_scales": torch.zeros(B * width, 2, page, device=dev) for y in "kv"} if quant else {}
        q = rope_append_paged(x, x, x, cos, sin, *pools, t, cu, **kw)[:B].contiguous()
        got.append([*gather_paged(*pools, t, cu, B * n, **kw), decode_paged(q, *pools, t, lens, **kw)])
        if not quant:
            got[-1].append(decode_paged_shared(q, *pools, t, lens, ints([n]), min_saved_bytes=0))
    for a, b in zip(*got):
        assert torch.equal(a, b)
