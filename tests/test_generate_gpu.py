"""The SmolLM forward on packed prompts and a paged cache (prefill_packed,
decode_packed, generate) against the reference's CPU path, prompt by prompt,
and the page bookkeeping."""
import pytest
import torch

from oracle.smollm_ref import Config, SmolLM, make_state_dict

LENS = [5, 1, 130, 64, 33]


def small():
    return Config(n_layers=4)


def test_pages_are_taken_and_given_back():
    from npu_b200.kvcache import PagedKVCache

    cache = PagedKVCache(2, 10, 3, 16, 64, torch.device("cpu"))
    a = cache.reserve([16, 17, 1])
    assert cache.free_pages == 6 and a.batch == 3 and tuple(a.block_table.shape) == (3, 2)
    used = [a.block_table[0, 0].item(), *a.block_table[1].tolist(), a.block_table[2, 0].item()]
    assert len(set(used)) == 4 and all(0 <= u < 10 for u in used)
    with pytest.raises(ValueError):
        cache.reserve([16 * 7])
    with pytest.raises(ValueError):
        cache.reserve([4, 0])
    b = cache.reserve([96])
    assert cache.free_pages == 0 and not set(b.block_table[0].tolist()) & set(used)
    a.release()
    a.release()
    assert cache.free_pages == 4
    with pytest.raises(ValueError):
        PagedKVCache(2, 10, 3, 24, 64, torch.device("cpu"))


@pytest.fixture(scope="module")
def weights():
    return make_state_dict(small(), seed=0)


def model_on(dev, sd, dtype=None):
    from npu_b200.smollm_b200 import SmolLMB200, SmolLMConfig

    return SmolLMB200(sd, SmolLMConfig(n_layers=4), dev, dtype=dtype)


def prompts():
    g = torch.Generator().manual_seed(7)
    return [torch.randint(0, 49152, (n,), generator=g).tolist() for n in LENS]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 48, 64])
def test_packed_steps_match_the_reference(cuda_dev, weights, page):
    """Prefill of five prompts at once, then three steps fed the reference's
    greedy tokens: logits and top-1 of every sequence."""
    from npu_b200 import api

    ref, model, ids = SmolLM(weights, small()), model_on(cuda_dev, weights), prompts()
    cache = model.new_paged_cache(40, page)
    seqs = cache.reserve([n + 8 for n in LENS])
    cu = torch.tensor([0] + LENS).cumsum(0).to(torch.int32).to(cuda_dev)
    logits = model.prefill_packed(torch.tensor([t for p in ids for t in p], device=cuda_dev), cu, seqs)
    refs = [ref.forward(torch.tensor([p])) for p in ids]
    for step in range(4):
        nxt = []
        for b, (want, _) in enumerate(refs):
            assert (logits[b].float().cpu() - want[0, -1]).abs().max().item() < 0.25, (step, b)
            assert logits[b].argmax().item() == want[0, -1].argmax().item(), (step, b)
            nxt.append(want[0, -1].argmax().item())
        assert seqs.lengths() == [n + step for n in LENS]
        if step == 3:
            break
        logits = model.decode_packed(torch.tensor(nxt, device=cuda_dev), seqs)
        refs = [ref.forward(torch.tensor([[t]]), cache=r[1], start_pos=n + step)
                for t, r, n in zip(nxt, refs, LENS)]
    assert api.device_error() == 0


@pytest.mark.gpu
def test_generate_greedy_is_the_references_loop(cuda_dev, weights):
    ref, model, ids = SmolLM(weights, small()), model_on(cuda_dev, weights), prompts()
    out = model.generate(ids, 6).tolist()
    for p, got in zip(ids, out):
        logits, past = ref.forward(torch.tensor([p]))
        for step, token in enumerate(got):
            assert token == logits[0, -1].argmax().item(), step
            logits, past = ref.forward(torch.tensor([[token]]), cache=past, start_pos=len(p) + step)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_generate_samples_and_returns_its_pages(cuda_dev, weights, dtype):
    """The same generator state gives the same tokens, another one others; top-k 1 is greedy; pages come back."""
    from npu_b200 import api

    model, ids = model_on(cuda_dev, weights, dtype), prompts()
    cache = model.new_paged_cache(64, 16)
    free = cache.free_pages

    def run(seed, **kw):
        g = torch.Generator(device=cuda_dev).manual_seed(seed)
        return model.generate(ids, 8, cache=cache, generator=g, **kw)

    a = run(1, temperature=0.9, top_k=50, top_p=0.95, min_p=0.001)
    assert a.shape == (5, 8) and ((a >= 0) & (a < 49152)).all()
    assert torch.equal(a, run(1, temperature=0.9, top_k=50, top_p=0.95, min_p=0.001))
    assert not torch.equal(a, run(2, temperature=0.9, top_k=50, top_p=0.95, min_p=0.001))
    assert torch.equal(run(3, temperature=1.0, top_k=1), model.generate(ids, 8, cache=cache))
    rows = torch.tensor([0.0, 0.5, 1.0, 2.0, 0.0], device=cuda_dev)
    mixed = run(4, temperature=rows)
    greedy = model.generate(ids, 8, cache=cache)
    assert torch.equal(mixed[[0, 4]], greedy[[0, 4]])
    assert cache.free_pages == free and api.device_error() == 0


@pytest.mark.gpu
def test_generate_refusals(cuda_dev, weights):
    model = model_on(cuda_dev, weights)
    cache = model.new_paged_cache(2, 16)
    for bad in ([], [[1], []]):
        with pytest.raises(ValueError):
            model.generate(bad, 4)
    with pytest.raises(ValueError):
        model.generate([[1]], 0)
    with pytest.raises(ValueError):
        model.generate([[1] * 8000], 1000)
    with pytest.raises(ValueError):
        model.generate([[1] * 30, [2]], 4, cache=cache)
    assert cache.free_pages == 2
