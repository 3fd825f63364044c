"""Pages of a PagedKVCache belong to one sequence at a time: what a sequence without room or one that gave its pages
back does to the others (nothing)."""
import pytest
import torch


def reserved(*capacities, page=16, n_pages=12):
    from npu_b200.kvcache import PagedKVCache

    cache = PagedKVCache(1, n_pages, 2, page, 64, torch.device("cpu"))
    return cache, cache.reserve(list(capacities))


def test_unused_table_entries_name_no_page():
    _, seqs = reserved(16, 48, 1, 33)
    used = []
    for row, pages in zip(seqs.block_table.tolist(), (1, 3, 1, 3)):
        assert all(0 <= p < 12 for p in row[:pages]) and row[pages:] == [-1] * (3 - pages)
        used += row[:pages]
    assert len(set(used)) == len(used)


def tiny(dev):
    from npu_b200.smollm_b200 import SmolLMB200, SmolLMConfig

    cfg = SmolLMConfig(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, head_dim=64, ffn_dim=64, vocab=50, max_pos=64)
    g = torch.Generator().manual_seed(0)

    def w(*shape):
        return 0.2 * torch.randn(*shape, generator=g)

    p = "model.layers.0."
    sd = {"model.embed_tokens.weight": w(50, 64), "model.norm.weight": torch.ones(64),
          p + "self_attn.q_proj.weight": w(128, 64), p + "self_attn.k_proj.weight": w(64, 64),
          p + "self_attn.v_proj.weight": w(64, 64), p + "self_attn.o_proj.weight": w(64, 128),
          p + "mlp.gate_proj.weight": w(64, 64), p + "mlp.up_proj.weight": w(64, 64),
          p + "mlp.down_proj.weight": w(64, 64), p + "input_layernorm.weight": torch.ones(64),
          p + "post_attention_layernorm.weight": torch.ones(64)}
    return SmolLMB200(sd, cfg, dev)


def test_steps_on_released_sequences_are_refused():
    model = tiny(torch.device("cpu"))  # nothing runs: the check comes first
    cache = model.new_paged_cache(4, 16)
    seqs = cache.reserve([16])
    seqs.release()
    with pytest.raises(ValueError, match="released"):
        model.prefill_packed(torch.tensor([1, 2]), torch.tensor([0, 2], dtype=torch.int32), seqs)
    with pytest.raises(ValueError, match="released"):
        model.decode_packed(torch.tensor([1]), seqs)


@pytest.mark.gpu
def test_a_step_past_the_pages_leaves_the_others_alone(cuda_dev):
    """Two sequences with a full first page; only the first has another. The second's next token has no place: it is
    left out and reported, and the first sequence goes on as without it."""
    from npu_b200 import _lib, device_error

    model = tiny(cuda_dev)
    ids = torch.arange(32, device=cuda_dev) % 50
    cu = torch.tensor([0, 16, 32], dtype=torch.int32, device=cuda_dev)

    def steps(capacities):
        cache = model.new_paged_cache(8, 16)
        cache.k.zero_()
        cache.v.zero_()
        seqs = cache.reserve(capacities)
        model.prefill_packed(ids, cu, seqs)
        assert device_error() == 0
        before = cache.k.clone()
        logits = model.decode_packed(torch.tensor([7, 8], device=cuda_dev), seqs)
        return cache, seqs, before, logits

    cache, seqs, before, logits = steps([48, 16])
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    written = (cache.k != before).any(-1).any(2).nonzero()  # (layer, page, slot)
    assert written.tolist() == [[0, seqs.block_table[0, 1].item(), 0]]
    _, _, _, room_for_both = steps([48, 48])
    assert device_error() == 0 and torch.equal(logits[0], room_for_both[0])


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 5, 900], [0, -3, 10], [0, 5, -7]])
def test_prompt_offsets_past_the_tokens_are_reported(cuda_dev, cu):
    """Not a fault: the bad prompt is left out, a good one keeps its logits."""
    from npu_b200 import _lib, device_error

    model = tiny(cuda_dev)
    ids = torch.arange(10, device=cuda_dev)

    def logits(cu):
        cache = model.new_paged_cache(8, 16)
        return model.prefill_packed(ids, torch.tensor(cu, dtype=torch.int32, device=cuda_dev), cache.reserve([16, 16]))

    good = logits([0, 5, 10])
    assert device_error() == 0
    got = logits(cu)
    torch.cuda.synchronize()
    assert device_error() == _lib.B2A_ERR_DEVICE_BAD_LEN
    if cu[1] == 5:
        assert torch.equal(got[0], good[0])
