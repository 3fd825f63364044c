"""How single-token attention over a paged cache numbers its work, up to lengths whose numbers pass 32 bits: found on
the device, compared with the same in Python."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def on_device(dev, lens, ahead, Hkv, cap, tile, units):
    from npu_b200 import _lib

    lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    four = torch.zeros(len(lens), 4, dtype=torch.int32, device=dev)
    if ahead:
        four[:, 0] = torch.tensor(ahead, dtype=torch.int32, device=dev)
    units = torch.tensor(units, dtype=torch.int64, device=dev)
    out = torch.empty(len(units), 4, dtype=torch.int64, device=dev)
    rc = _lib.load().b2a_diag_paged_units(lens.data_ptr(), four.data_ptr() if ahead else None, len(lens), Hkv,
                                          cap // 16, 16, tile, units.data_ptr(), len(units), out.data_ptr(),
                                          torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0
    return [tuple(x) for x in out.tolist()]


def in_python(lens, ahead, Hkv, tile, units):
    tiles = [max(-(-t // tile) - a // tile, 0) for t, a in zip(lens, ahead or [0] * len(lens))]
    total = Hkv * sum(n + 1 for n in tiles if n)
    out = []
    for u in units:
        at, found = u, (-1, -1, -1)
        for b, n in enumerate(tiles):
            if n and at < Hkv * (n + 1):
                g, x = divmod(at, n + 1)
                found = (b, g, x) if x < n else found
                break
            at -= Hkv * (n + 1) if n else 0
        out.append((total, *found))
    return out


@pytest.mark.parametrize("tile,shared", [(64, False), (128, False), (64, True)])
@pytest.mark.parametrize("B", [1, 31, 33, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("longest", [3000, 2 ** 31 - 160])
def test_units(cuda_dev, B, longest, tile, shared):
    g = torch.Generator().manual_seed(B + tile)
    Hkv, cap = 3, longest // 16 * 16
    lens = torch.randint(longest * 3 // 4, longest, (B,), generator=g).tolist()
    for b in range(0, B, 5):
        lens[b] = (0, 1, cap, 64)[b // 5 % 4]
    ahead = [t // 2 // 64 * 64 * (b % 3 == 0) for b, t in enumerate(lens)] if shared else None
    total = in_python(lens, ahead, Hkv, tile, [0])[0][0]
    units = [0, 1, total - 2, total - 1, total]
    units += [int(x) for x in (torch.rand(40, generator=g, dtype=torch.float64) * total).tolist()]
    assert on_device(cuda_dev, lens, ahead, Hkv, cap, tile, units) == in_python(lens, ahead, Hkv, tile, units)
