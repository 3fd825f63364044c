"""What the serving operators do when a wait runs out or their device-side
arguments are out of range: they end, report it and leave the context usable."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mute_pass,temperature,top_p", [(0, 0.0, 1.0), (0, 1.0, 1.0), (1, 1.0, 1.0), (2, 1.0, 0.3)])
@pytest.mark.parametrize("R,V", [(1, 49152), (5, 40_001), (200, 3000)])
def test_sampling_ends_when_a_part_of_a_row_stops_answering(cuda_dev, R, V, mute_pass, temperature, top_p):
    """The last block of every row stops sending at one of the joins: with waits of 1 ms (the kernels' are 2 s) the
    row's blocks give up together, the rows give -1 and the error word says why."""
    from npu_b200 import _lib, api

    g = torch.Generator(device=cuda_dev).manual_seed(V)
    x = 2 * torch.randn(R, V, generator=g, device=cuda_dev)
    e = torch.empty(R, V, device=cuda_dev).exponential_(generator=g)
    expected = api.sample(x, e, temperature=temperature, top_p=top_p)
    assert api.device_error() == 0
    out = torch.full((R,), -7, dtype=torch.long, device=cuda_dev)
    rc = _lib.load().b2a_diag_sample_timeout(x.data_ptr(), e.data_ptr(), R, V, temperature, top_p, mute_pass,
                                             2_000_000, out.data_ptr(),
                                             torch.cuda.current_stream(cuda_dev).cuda_stream)
    assert rc == 0
    assert api.device_error() == _lib.B2A_ERR_DEVICE_TIMEOUT
    if mute_pass < 2:
        assert (out == -1).all()
    else:  # rows whose first race decides never get to the third join
        assert ((out == -1) | (out == expected)).all() and (out == -1).any()
    assert torch.equal(api.sample(x, e, temperature=temperature, top_p=top_p), expected)
    assert api.device_error() == 0


def test_lengths_written_over_the_positions_are_refused(cuda_dev):
    from npu_b200 import rope_append_paged

    B = 3
    q = torch.zeros(B, 4, 64, dtype=torch.bfloat16, device=cuda_dev)
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=cuda_dev)
    tab = torch.zeros(16, 64, dtype=torch.bfloat16, device=cuda_dev)
    pos = torch.zeros(2, B, dtype=torch.int32, device=cuda_dev)
    table = torch.arange(B, dtype=torch.int32, device=cuda_dev)[:, None]
    cu = torch.arange(B + 1, dtype=torch.int32, device=cuda_dev)

    def call(start, end):
        return rope_append_paged(q, q[:, :2], q[:, :2], tab, tab, pool, pool.clone(), table, cu,
                                 start_pos_per_batch=start, seqlens_out=end)

    for start, end in [(pos[0], pos[0]), (pos[0], pos.view(-1)[1:4]), (pos.view(-1)[2:5], pos[0])]:
        with pytest.raises(ValueError, match="overlap"):
            call(start, end)
    call(pos[0], pos[1])
    assert pos.tolist() == [[0] * B, [1] * B]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 40])
def test_tokens_past_the_rotary_tables_are_skipped_whole(cuda_dev, dtype, tokens):
    """Positions that the block table has pages for but the rotary tables no row: q, k and v stay unwritten."""
    from npu_b200 import _lib, device_error, rope_append_paged

    g = torch.Generator(device=cuda_dev).manual_seed(1)
    q = torch.randn(tokens, 4, 64, generator=g, device=cuda_dev).to(dtype)
    kv = torch.randn(2, tokens, 2, 64, generator=g, device=cuda_dev).to(dtype)
    kp, vp = (torch.full((8, 2, 16, 64), 3.0, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device=cuda_dev)[None]
    tab = torch.randn(2, 20, 64, generator=g, device=cuda_dev).to(dtype)
    q_out = torch.full((tokens, 4, 64), 3.0, dtype=torch.bfloat16, device=cuda_dev)
    first = 20 - tokens // 2  # the second half of the tokens is past the tables' 20 rows
    cu = torch.tensor([0, tokens], dtype=torch.int32, device=cuda_dev)
    assert device_error() == 0
    rope_append_paged(q, kv[0], kv[1], tab[0], tab[1], kp, vp, table, cu, start_pos=first, q_out=q_out)
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    n = tokens // 2
    for pool in (kp, vp):
        rows = pool.transpose(1, 2).reshape(128, 2, 64)
        assert (rows[20:] == 3).all() and (rows[:first] == 3).all()
        assert (rows[first:20] != 3).any(-1).all()
    assert (q_out[n:] == 3).all() and (q_out[:n] != 3).any(-1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cu,good", [([0, 5, 900], 0), ([-3, 5, 10], 1), ([0, 5, -7], 0), ([5, 0, 5], 1),
                                     ([0, 11, 10], None)])
@pytest.mark.parametrize("lengths", [True, False])
def test_append_reports_offsets_that_are_no_stretch(cuda_dev, cu, good, lengths, dtype):
    """Two sequences over ten tokens, at most one of them good: its tokens are written, the other's are not and its
    length stays."""
    from npu_b200 import _lib, device_error, rope_append_paged

    g = torch.Generator(device=cuda_dev).manual_seed(2)
    q = torch.randn(10, 4, 64, generator=g, device=cuda_dev).to(dtype)
    kv = torch.randn(2, 10, 2, 64, generator=g, device=cuda_dev).to(dtype)
    tab = torch.randn(2, 32, 64, generator=g, device=cuda_dev).to(dtype)
    kp, vp = (torch.full((4, 2, 16, 64), 3.0, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=cuda_dev).view(2, 2)
    end = torch.full((2,), -1, dtype=torch.int32, device=cuda_dev) if lengths else None
    assert device_error() == 0
    rope_append_paged(q, kv[0], kv[1], tab[0], tab[1], kp, vp, table, torch.tensor(cu, dtype=torch.int32, device=cuda_dev),
                      start_pos=4, seqlens_out=end)
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    n = [0, 0]
    if good is not None:
        n[good] = cu[good + 1] - cu[good]
    if lengths:
        assert end.tolist() == [4 + t for t in n]
    for b in range(2):
        rows = kp[2 * b:2 * b + 2].transpose(1, 2).reshape(32, 2, 64)
        assert (rows[4:4 + n[b]] != 3).any(-1).all() and (rows[:4] == 3).all() and (rows[4 + n[b]:] == 3).all()
