"""Empty batches of the serving operators: empty results, and lengths that stay."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_to_sample(cuda_dev, dtype):
    from npu_b200 import sample

    x = torch.zeros(0, 100, dtype=dtype, device=cuda_dev)
    e = torch.ones(0, 100, device=cuda_dev)
    rows = torch.zeros(0, device=cuda_dev)
    for got in (sample(x, temperature=0.0), sample(x, e), sample(x, e, temperature=rows, top_p=rows, min_p=rows,
                                                                top_k=rows.int())):
        assert got.shape == (0,) and got.dtype == torch.long
    out = torch.zeros(0, dtype=torch.long, device=cuda_dev)
    assert sample(x, e, out=out).shape == (0,)
    with pytest.raises(ValueError):
        sample(x, e[:, :50])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_tokens_to_append(cuda_dev, dtype):
    from npu_b200 import device_error, rope_append_paged

    q, kv = torch.zeros(0, 4, 64, dtype=dtype, device=cuda_dev), torch.zeros(0, 2, 64, dtype=dtype, device=cuda_dev)
    pool = torch.full((5, 2, 16, 64), 3.0, dtype=torch.bfloat16, device=cuda_dev)
    tab = torch.zeros(16, 64, dtype=dtype, device=cuda_dev)
    table = torch.arange(3, dtype=torch.int32, device=cuda_dev)[:, None]
    cu = torch.zeros(4, dtype=torch.int32, device=cuda_dev)
    start = torch.tensor([3, 0, 9], dtype=torch.int32, device=cuda_dev)
    end = torch.full((3,), -1, dtype=torch.int32, device=cuda_dev)
    got = rope_append_paged(q, kv, kv, tab, tab, pool, pool.clone(), table, cu, start_pos_per_batch=start,
                            seqlens_out=end, return_kv=True)
    assert [tuple(t.shape) for t in got] == [(0, 4, 64), (0, 2, 64), (0, 2, 64)]
    assert all(t.dtype == torch.bfloat16 for t in got)
    assert torch.equal(end, start) and (pool == 3).all()
    rope_append_paged(q, kv, kv, tab, tab, pool, pool.clone(), table, cu, start_pos=7, seqlens_out=end)
    assert end.tolist() == [7, 7, 7] and device_error() == 0


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_no_sequences_to_decode(cuda_dev, out_dtype):
    from npu_b200 import decode_paged

    pool = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16, device=cuda_dev)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=cuda_dev)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_dev)
    got = decode_paged(q, pool, pool, none.view(0, 3), none, out_dtype=out_dtype, gate=q)
    assert got.shape == (0, 4, 64) and got.dtype == out_dtype
