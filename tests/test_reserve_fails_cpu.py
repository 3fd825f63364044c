"""Sequences that cannot be set up leave the pages free and the prefix without them."""
import pytest
import torch


@pytest.mark.parametrize("behind", [False, True])
def test_pages_come_back(monkeypatch, behind):
    from npu_b200 import kvcache

    cache = kvcache.PagedKVCache(1, 9, 1, 16, 64, torch.device("cpu"))
    prefix = cache.reserve([32]) if behind else None
    free = list(cache._free)

    def no_memory(*args, **kw):
        raise torch.OutOfMemoryError("no memory for the offsets")

    with monkeypatch.context() as m:
        m.setattr(kvcache.torch, "arange", no_memory)
        with pytest.raises(torch.OutOfMemoryError):
            cache.reserve([40, 16], prefix=prefix)
    assert cache._free == free
    seqs = cache.reserve([40, 16], prefix=prefix)
    if behind:
        assert prefix.followers == 1
        with pytest.raises(ValueError, match="1 batches of sequences"):
            prefix.release()
    seqs.release()
    if behind:
        prefix.release()
    assert cache.free_pages == 9
