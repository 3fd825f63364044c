"""The numbering of packed prompts' query blocks (which block of which sequence number i is), against the same
numbering on the host, for numbers asked for in any order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ROWS, BY_POSITION = 128, 256


def numbered(lens_q, lens_k, causal):
    """Blocks (first row, rows, first key, keys, block), heaviest level first and by sequence within a level."""
    out, iq, ik = [], 0, 0
    for b, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        ahead = max(lk - lq if causal else lk, 0) // ROWS
        out += [((-(ahead + i), b), (iq, lq, ik, lk, i)) for i in range(-(-lq // ROWS))]
        iq, ik = iq + lq, ik + lk
    return [block for _, block in sorted(out)]


def offsets(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


def ask(cu_q, cu_k, Nq, Nk, causal, ids):
    from npu_b200 import _lib

    out = torch.full((len(ids), 5), -9, dtype=torch.int32, device=cu_q.device)
    rc = _lib.load().b2a_diag_packed_blocks(cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, Nq, Nk, causal,
                                            ids.data_ptr(), len(ids), out.data_ptr(),
                                            torch.cuda.current_stream(cu_q.device).cuda_stream)
    assert rc == 0
    return [tuple(t) for t in out.tolist()]


def lengths(B, most, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most, (B,), generator=g).tolist()


@pytest.mark.parametrize("order", ["growing", "falling", "shuffled"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("B,most", [(1, 2000), (5, 1500), (32, 900), (33, 900), (200, 600)])
def test_blocks_in_any_order(cuda_dev, B, most, causal, order):
    from npu_b200 import device_error

    lens_q, lens_k = lengths(B, most, B), lengths(B, 2 * most, B + 1)
    expected = numbered(lens_q, lens_k, causal)
    n = len(expected)
    ids = {"growing": torch.arange(n), "falling": torch.arange(n - 1, -1, -1),
           "shuffled": torch.randperm(n, generator=torch.Generator().manual_seed(B))}[order]
    got = ask(offsets(lens_q, cuda_dev), offsets(lens_k, cuda_dev), sum(lens_q), sum(lens_k), causal,
              ids.to(torch.int32).to(cuda_dev))
    assert got == [expected[i] for i in ids.tolist()]
    assert device_error() == 0


@pytest.mark.parametrize("order", ["growing", "shuffled"])
def test_blocks_by_position_in_any_order(cuda_dev, order):
    """More sequences than are sorted: every block has one number, spare numbers have no rows."""
    lens = lengths(BY_POSITION + 90, 400, 3)
    n = sum(lens) // ROWS + len(lens)
    ids = torch.arange(n) if order == "growing" else torch.randperm(n, generator=torch.Generator().manual_seed(4))
    cu = offsets(lens, cuda_dev)
    got = ask(cu, cu, sum(lens), sum(lens), 1, ids.to(torch.int32).to(cuda_dev))
    assert sorted(b for b in got if b[1] > 0) == sorted(numbered(lens, lens, 1))


@pytest.mark.parametrize("B", [40, BY_POSITION + 90])
@pytest.mark.parametrize("which,value", [("q", -5), ("q", 10 ** 9), ("q", 200), ("k", -5), ("k", 10 ** 9), ("k", 200)])
@pytest.mark.parametrize("at", [20, -1])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 64), (2, 1, 128), (1, 1, 256)])
def test_a_bad_offset_is_reported_wherever_it_is(cuda_dev, B, which, value, at, Hq, Hkv, D):
    """One offset below 0, past the tensors or below the one before it: the call reports it, and what it writes lies
    in the output."""
    from npu_b200 import _lib, device_error, prefill_varlen

    n = 40 * B
    cu = {x: torch.arange(0, n + 1, 40, dtype=torch.int32, device=cuda_dev) for x in "qk"}
    cu[which][at] = value
    g = torch.Generator(device=cuda_dev).manual_seed(B)
    q = torch.randn(n, Hq, D, generator=g, device=cuda_dev).bfloat16()
    kv = torch.randn(n, Hkv, D, generator=g, device=cuda_dev).bfloat16()
    hold = torch.full((n + 256, Hq, D), 5.0, device=cuda_dev)
    clean = prefill_varlen(q, kv, kv, torch.arange(0, n + 1, 40, dtype=torch.int32, device=cuda_dev))
    assert device_error() == 0
    prefill_varlen(q, kv, kv, cu["q"], cu["k"], out=hold[128:-128])
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    assert (hold[:128] == 5).all() and (hold[-128:] == 5).all()
    inner = hold[128:-128]
    assert torch.isfinite(inner).all()
    if B <= BY_POSITION and (which, value) != ("q", 200):  # (there the next pair's queries overlap others')
        kept = torch.ones(n, dtype=torch.bool)  # only the pairs with that offset are left out
        b = at % (B + 1)
        kept[40 * (b - 1):40 * (b + 1)] = False
        assert torch.equal(inner[kept.to(cuda_dev)], clean[kept.to(cuda_dev)])
