"""What one kernel of a stream writes, the next reads: many steps without a pause, each over the slots, logits and
tokens of the step before."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("n", [1, 5, 700])
def test_append_gather_on_the_same_slots(cuda_dev, quant, n):
    """Every step writes the same slots with other rows and reads them back."""
    from npu_b200 import gather_paged, rope_append_paged

    dev, Hkv, D, page, steps = cuda_dev, 4, 128, 64, 60
    pages = -(-n // page)
    k, v = (torch.randn(steps, n, Hkv, D, generator=gen(dev, s), device=dev).bfloat16() for s in (1, 2))
    q = torch.randn(n, 8, D, generator=gen(dev, 3), device=dev).bfloat16()
    cos, sin = torch.ones(n, D, device=dev).bfloat16(), torch.zeros(n, D, device=dev).bfloat16()
    kp, vp = (torch.zeros(pages, Hkv, page, D, device=dev).to(E4M3 if quant else torch.bfloat16) for _ in range(2))
    kw = {f"{x}_scales": torch.zeros(pages, Hkv, page, device=dev) for x in "kv"} if quant else {}
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    outs = [torch.empty(steps, n, Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(steps):
        rope_append_paged(q, k[i], v[i], cos, sin, kp, vp, table, cu, **kw)
        gather_paged(kp, vp, table, cu, n, k_out=outs[0][i], v_out=outs[1][i], **kw)
    for x, back in zip((k, v), outs):
        if quant:
            s = (x.double().abs().amax(-1, keepdim=True) / 448).float()
            codes = (x.float() * (1 / s.double()).float()).to(E4M3)
            assert torch.equal(back, (codes.float() * s).bfloat16())
        else:
            assert torch.equal(back, x)


@pytest.mark.parametrize("V,dtype", [(1000, torch.float32), (49152, torch.bfloat16), (131071, torch.bfloat16)])
def test_penalties_on_the_output_of_the_step_before(cuda_dev, V, dtype):
    """A penalised row is the next call's logits, bias and mask: sums in place, in whole numbers."""
    from npu_b200 import penalize

    dev, R, steps = cuda_dev, 8, 50
    x = torch.zeros(R, V, device=dev, dtype=dtype)
    tokens = torch.randint(0, V, (R, 64), generator=gen(dev, 1), device=dev)
    count = torch.zeros(R, V, device=dev).scatter_add_(1, tokens, torch.ones_like(tokens, dtype=torch.float32))
    first, second = (torch.empty(R, V, device=dev) for _ in range(2))
    one = torch.ones(V, device=dev)
    first.zero_()
    torch.cuda.synchronize()
    for i in range(steps):  # each adds the bias that the one before has written, and a penalty of one per token
        penalize(first, tokens, frequency=1.0, bias=one, out=second)
        first, second = second, first
        penalize(x, bias=first, out=x)
    rows = torch.arange(1, steps + 1, device=dev).double()
    want = ((1 - count.double())[..., None] * rows).sum(-1)
    if dtype == torch.float32:
        assert torch.equal(x.double(), want)
    else:  # each sum is rounded to bf16 as the kernel's are
        y = torch.zeros(R, V, device=dev)
        for i in range(1, steps + 1):
            y = (y + (1 - count) * i).bfloat16().float()
        assert torch.equal(x.float(), y)


@pytest.mark.parametrize("V", [1000, 151937])
def test_noise_of_the_kernel_before(cuda_dev, V):
    """Noise written right ahead of each choice, over that of the step before."""
    from npu_b200 import sample

    dev, R, steps = cuda_dev, 4, 40
    logits = torch.randn(R, V, generator=gen(dev, 1), device=dev)
    draws = torch.empty(steps, R, V, device=dev).exponential_(generator=gen(dev, 2))
    noise, out = torch.ones(R, V, device=dev), torch.empty(steps, R, dtype=torch.long, device=dev)
    for i in range(steps):
        noise.copy_(draws[i])
        sample(logits, noise, temperature=1.0, out=out[i])
    want = torch.stack([sample(logits, draws[i].clone(), temperature=1.0) for i in range(steps)])
    assert torch.equal(out, want)


@pytest.mark.parametrize("Hq,Hkv,D", [(9, 3, 64), (32, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("left", [0, 0xff, 0x706c616e])
def test_shared_step_whatever_the_workspace_holds(cuda_dev, Hq, Hkv, D, left):
    """Append and attend behind a prefix, step by step without a pause, in a workspace that held anything before (the
    words the kernels leave for one another among it): the bits of steps that waited for one another."""
    from npu_b200 import decode_paged_shared, rope_append_paged
    from npu_b200.api import decode_paged_shared_workspace_bytes

    dev, B, page, prefix, steps = cuda_dev, 12, 64, 1920, 30
    own = -(-(steps + 1) // page)
    pages = prefix // page + B * own
    first = [torch.randn(pages, Hkv, page, D, generator=gen(dev, s), device=dev).bfloat16() for s in (1, 2)]
    table = torch.arange(prefix // page, dtype=torch.int32, device=dev).expand(B, -1)
    table = torch.cat([table, prefix // page + torch.arange(B * own, dtype=torch.int32, device=dev).view(B, own)], 1)
    q, k, v = (torch.randn(steps, B, h, D, generator=gen(dev, 3 + i), device=dev).bfloat16()
               for i, h in enumerate((Hq, Hkv, Hkv)))
    cos, sin = torch.ones(4096, D, device=dev).bfloat16(), torch.zeros(4096, D, device=dev).bfloat16()
    one_each = torch.arange(B + 1, dtype=torch.int32, device=dev)
    pre = torch.tensor([prefix], dtype=torch.int32, device=dev)
    need = decode_paged_shared_workspace_bytes(B, Hq, Hkv, D, 1)
    got = []
    for pause in (True, False):
        kp, vp = (x.clone() for x in first)
        ws = torch.zeros(need // 4 + 1, dtype=torch.int32, device=dev)
        if not pause:
            ws.fill_(left)
        lens = torch.full((2, B), prefix, dtype=torch.int32, device=dev)
        outs = []
        torch.cuda.synchronize()
        for i in range(steps):
            a, b = lens[i % 2], lens[1 - i % 2]
            rot = rope_append_paged(q[i], k[i], v[i], cos, sin, kp, vp, table, one_each, start_pos_per_batch=a,
                                    seqlens_out=b)
            if pause:
                torch.cuda.synchronize()
            outs.append(decode_paged_shared(rot, kp, vp, table, b, pre, min_saved_bytes=0, workspace=ws))
            if pause:
                torch.cuda.synchronize()
        got.append(torch.stack(outs))
    assert torch.equal(*got)
