"""Refusals of the serving operators' arguments: ValueError with the sizes in it, nothing launched, and the next call
works."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(dev, *values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def attend(dev, **over):
    from npu_b200 import prefill_varlen

    a = dict(q=torch.zeros(20, 4, 64, device=dev).bfloat16(), k=torch.zeros(20, 2, 64, device=dev).bfloat16(),
             v=torch.zeros(20, 2, 64, device=dev).bfloat16(), cu=ints(dev, 0, 5, 20), cu_k=None)
    kw = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    return prefill_varlen(a["q"], a["k"], a["v"], a["cu"], a["cu_k"], **kw)


def decode(dev, **over):
    from npu_b200 import decode_paged

    a = dict(q=torch.zeros(2, 4, 64, device=dev).bfloat16(), kp=torch.zeros(5, 2, 16, 64, device=dev).bfloat16(),
             vp=torch.zeros(5, 2, 16, 64, device=dev).bfloat16(), table=ints(dev, 0, 1, 2, 3).view(2, 2),
             lens=ints(dev, 20, 3))
    kw = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    return decode_paged(a["q"], a["kp"], a["vp"], a["table"], a["lens"], **kw)


def append(dev, **over):
    from npu_b200 import rope_append_paged

    a = dict(q=torch.zeros(3, 4, 64, device=dev), k=torch.zeros(3, 2, 64, device=dev),
             v=torch.zeros(3, 2, 64, device=dev), cos=torch.zeros(16, 64, device=dev), sin=torch.zeros(16, 64, device=dev),
             kp=torch.zeros(5, 2, 16, 64, device=dev).bfloat16(), vp=torch.zeros(5, 2, 16, 64, device=dev).bfloat16(),
             table=ints(dev, 0, 1).view(2, 1), cu=ints(dev, 0, 1, 3))
    kw = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    return rope_append_paged(*a.values(), **kw)


def draw(dev, **over):
    from npu_b200 import sample

    a = dict(x=torch.zeros(3, 100, device=dev), e=torch.ones(3, 100, device=dev))
    kw = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    return sample(a["x"], a["e"], **kw)


BAD = [
    (attend, lambda d: dict(q=torch.zeros(20, 256, device=d).bfloat16()), r"q must have 3 dims, got shape \[20, 256\]"),
    (attend, lambda d: dict(q=torch.zeros(20, 4, 64, device=d)), "q must be bfloat16"),
    (attend, lambda d: dict(k=torch.zeros(20, 2, 128, device=d).bfloat16()), r"shape mismatch q\[20, 4, 64\]"),
    (attend, lambda d: dict(k=torch.zeros(21, 2, 64, device=d).bfloat16(),
                            v=torch.zeros(21, 2, 64, device=d).bfloat16()), "k has 21 rows and q 20"),
    (attend, lambda d: dict(cu=ints(d, 0)), "two offsets"),
    (attend, lambda d: dict(cu=ints(d, 0, 5, 20).long()), "int32 tensor of 3"),
    (attend, lambda d: dict(cu_k=ints(d, 0, 20)), "cu_seqlens_k must be a contiguous int32 tensor of 3"),
    (attend, lambda d: dict(gate=torch.zeros(20, 4, 32, device=d)), r"gate must be \[20, 4, 64\]"),
    (attend, lambda d: dict(out=torch.zeros(20, 4, 64, device=d).bfloat16()), "out must match"),
    (attend, lambda d: dict(out_dtype=torch.float16), "out_dtype must be"),
    (decode, lambda d: dict(vp=torch.zeros(5, 2, 32, 64, device=d).bfloat16()), r"k_pages\[5, 2, 16, 64\]"),
    (decode, lambda d: dict(table=ints(d, 0, 1)), r"int32 tensor \[2, pages\]"),
    (decode, lambda d: dict(lens=ints(d, 1, 2, 3)), "int32 tensor of 2"),
    (decode, lambda d: dict(workspace=torch.zeros(3, dtype=torch.uint8, device=d)), r"at least \d+ bytes"),
    (append, lambda d: dict(v=torch.zeros(3, 1, 64, device=d)), r"k\[3, 2, 64\] v\[3, 1, 64\]"),
    (append, lambda d: dict(kp=torch.zeros(5, 3, 16, 64, device=d).bfloat16()), r"cache shape \[5, 3, 16, 64\]"),
    (append, lambda d: dict(start_pos_per_batch=ints(d, 1)), "int32 tensor of 2"),
    (append, lambda d: dict(start_pos=1 << 40), "start_pos is too large: 1099511627776"),
    (append, lambda d: dict(q_norm=torch.ones(32, device=d)), "q_norm"),
    (append, lambda d: dict(rope_dim=32), "cos/sin"),
    (draw, lambda d: dict(e=torch.ones(3, 50, device=d)), r"noise must be a float32 tensor \[3, 100\]"),
    (draw, lambda d: dict(e=None), "needs noise"),
    (draw, lambda d: dict(temperature=torch.ones(4, device=d)), r"temperature must be .* tensor \[3\]"),
    (draw, lambda d: dict(top_k=torch.ones(3, device=d)), "top_k must be"),
    (draw, lambda d: dict(out=torch.zeros(3, dtype=torch.int32, device=d)), "out must be"),
]


@pytest.mark.parametrize("which", range(len(BAD)))
def test_refused(cuda_dev, which):
    call, over, message = BAD[which]
    call(cuda_dev)
    with pytest.raises(ValueError, match=message):
        call(cuda_dev, **over(cuda_dev))
    call(cuda_dev)
    torch.cuda.synchronize()
