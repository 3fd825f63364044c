"""When single-token attention over shared prefixes shares by itself: the default of min_saved_bytes. What is shared is
seen in the bits (P is rounded to bf16 there)."""
import pytest
import torch

from test_decode_shared_gpu import build, check, gen, ints

pytestmark = pytest.mark.gpu


def call(dev, groups, width=None, **kw):
    from npu_b200 import decode_paged, decode_paged_shared

    ks, vs, kp, vp, table, lens, pre, cu = build(dev, groups, 4, 128, 64, 3, width=width)
    q = torch.randn(len(ks), 32, 128, generator=gen(dev, 1), device=dev).bfloat16()
    out = decode_paged_shared(q, kp, vp, table, lens, pre, cu, **kw)
    check(out[::7], q[::7], ks[::7], vs[::7], 128 ** -0.5)
    return not torch.equal(out, decode_paged(q, kp, vp, table, lens))


@pytest.mark.parametrize("groups,width,shares", [
    ([(2048, [10] * 64)], None, True),        # 63 x 2112 keys x 2 KB = 272 MB
    ([(2048, [10] * 32)] * 2, None, True),    # 268 MB
    ([(2048, [10] * 2)] * 32, None, False),   # 32 groups: 138 MB
    ([(2048, [10] * 30)], None, False),       # 125 MB
    ([(2048, [10] * 30)], 48, True),          # a wider table: 182 MB, and the device finds 122
    ([(256, [10] * 30)], 48, False),          # the same, and it finds 15
    ([(0, [500] * 70)], None, False),
    ([(4096, [10] * 8)] * 1, 64 * 8, True),   # 59 MB of what a wide table could name
])
def test_default(cuda_dev, groups, width, shares):
    assert call(cuda_dev, groups, width) == shares


def test_empty_groups_do_not_count_where_the_caller_decides(cuda_dev):
    """With min_saved_bytes only what there is to save counts, however many groups there are."""
    from npu_b200 import decode_paged, decode_paged_shared

    dev = cuda_dev
    ks, vs, kp, vp, table, lens, pre, _ = build(dev, [(1000, [10, 20, 30])], 4, 128, 64, 3)
    q = torch.randn(3, 32, 128, generator=gen(dev, 1), device=dev).bfloat16()
    cu = ints(dev, [0, 3, 3, 3, 3, 3])
    out = decode_paged_shared(q, kp, vp, table, lens, pre.expand(5).contiguous(), cu, min_saved_bytes=0)
    check(out, q, ks, vs, 128 ** -0.5)
    assert not torch.equal(out, decode_paged(q, kp, vp, table, lens))
