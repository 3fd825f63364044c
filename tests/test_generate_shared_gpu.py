"""SmolLMB200.generate with an 8-bit cache, a shared prefix and penalties: the serving operators together."""
import functools
import math

import pytest
import torch

from oracle.smollm_ref import Config, SmolLM, make_state_dict

LENS = [5, 1, 130, 64, 33]


@pytest.fixture(scope="module")
def weights():
    return make_state_dict(Config(n_layers=4), seed=0)


def model_on(dev, sd, dtype=None):
    from npu_b200.smollm_b200 import SmolLMB200, SmolLMConfig

    return SmolLMB200(sd, SmolLMConfig(n_layers=4), dev, dtype=dtype)


def some(seed, *lens):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 49152, (n,), generator=g).tolist() for n in lens]


def test_prefix_pages():
    """Followers name the prefix's pages first, start after its tokens and keep it from being released."""
    from npu_b200.kvcache import PagedKVCache

    cache = PagedKVCache(2, 12, 3, 16, 64, torch.device("cpu"), torch.float8_e4m3fn)
    assert cache.k.dtype == torch.float8_e4m3fn and tuple(cache.scales(1)["v_scales"].shape) == (12, 3, 16)
    assert PagedKVCache(1, 2, 3, 16, 64, torch.device("cpu")).scales(0) == {}
    head = cache.reserve([48])
    seqs = cache.reserve([16, 17], prefix=head)
    assert cache.free_pages == 6 and tuple(seqs.block_table.shape) == (2, 5)
    assert (seqs.block_table[:, :3] == head.block_table[0]).all() and seqs.block_table[0, 4] == -1
    own = set(seqs.block_table[:, 3:].flatten().tolist()) - {-1}
    assert len(own) == 3 and not own & set(head.block_table[0].tolist())
    assert seqs.lengths() == [48, 48] and seqs.prefix_lens.tolist() == [48] and seqs.prefix_tokens == 48
    with pytest.raises(ValueError, match="go on from"):
        head.release()
    seqs.release()
    seqs.release()
    head.release()
    assert cache.free_pages == 12 and head.released
    for bad in (head, cache.reserve([17]), cache.reserve([16, 16]),
                PagedKVCache(1, 2, 3, 16, 64, torch.device("cpu")).reserve([16])):
        free = cache.free_pages
        with pytest.raises(ValueError, match="prefix must be"):
            cache.reserve([4], prefix=bad)
        assert cache.free_pages == free
    with pytest.raises(ValueError):
        PagedKVCache(2, 10, 3, 16, 64, torch.device("cpu"), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("least", [0, None])
@pytest.mark.parametrize("page,length", [(16, 700), (64, 640), (48, 1000), (64, 40)])
def test_steps_behind_a_prefix_match_the_reference(cuda_dev, weights, page, length, least, monkeypatch):
    """The prefix once, five prompts behind it, then three steps fed the reference's greedy tokens: logits and top-1 of
    every sequence, as prompts without a shared prefix are tested."""
    from npu_b200 import api

    # These sizes are below where sharing pays: 0 shares all the same.
    monkeypatch.setattr(api, "decode_paged_shared", functools.partial(api.decode_paged_shared, min_saved_bytes=least))
    ref, model = SmolLM(weights, Config(n_layers=4)), model_on(cuda_dev, weights)
    (prefix,), ids = some(3, length), some(7, *LENS)
    shared = length // page * page
    cache = model.new_paged_cache(100, page)
    own = [prefix[shared:] + p for p in ids]
    if shared:
        head = cache.reserve([shared])
        model.prefill_packed(torch.tensor(prefix[:shared], device=cuda_dev),
                             torch.tensor([0, shared], dtype=torch.int32, device=cuda_dev), head)
        seqs = cache.reserve([len(p) + 8 for p in own], prefix=head)
    else:
        seqs = cache.reserve([len(p) + 8 for p in own])
    cu = torch.tensor([0] + [len(p) for p in own]).cumsum(0).to(torch.int32).to(cuda_dev)
    logits = model.prefill_packed(torch.tensor([t for p in own for t in p], device=cuda_dev), cu, seqs)
    refs = [ref.forward(torch.tensor([prefix + p])) for p in ids]
    for step in range(4):
        nxt = []
        for b, (want, _) in enumerate(refs):
            assert (logits[b].float().cpu() - want[0, -1]).abs().max().item() < 0.25, (step, b)
            assert logits[b].argmax().item() == want[0, -1].argmax().item(), (step, b)
            nxt.append(want[0, -1].argmax().item())
        assert seqs.lengths() == [length + n + step for n in LENS]
        if step == 3:
            break
        logits = model.decode_packed(torch.tensor(nxt, device=cuda_dev), seqs)
        refs = [ref.forward(torch.tensor([[t]]), cache=r[1], start_pos=length + n + step)
                for t, r, n in zip(nxt, refs, LENS)]
    assert api.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_generate_with_everything(cuda_dev, weights, dtype):
    """Reproducible, pages come back, and an 8-bit cache runs the same calls."""
    from npu_b200 import api

    model, ids, (prefix,) = model_on(cuda_dev, weights, torch.bfloat16), some(7, *LENS), some(3, 700)
    cache = model.new_paged_cache(200, 16, dtype)
    free = cache.free_pages

    def run(seed, **kw):
        g = torch.Generator(device=cuda_dev).manual_seed(seed)
        a = dict(temperature=0.9, top_k=50, prefix=prefix, repetition_penalty=1.2, frequency_penalty=0.1,
                 presence_penalty=torch.full((5,), 0.3, device=cuda_dev))
        return model.generate(ids, 8, cache=cache, generator=g, **{**a, **kw})

    a = run(1)
    assert a.shape == (5, 8) and ((a >= 0) & (a < 49152)).all()
    assert torch.equal(a, run(1)) and not torch.equal(a, run(2))
    assert cache.free_pages == free and api.device_error() == 0
    # A bias that favours one token beyond everything; a mask that leaves two.
    bias = torch.zeros(49152, device=cuda_dev)
    bias[777] = 1e4
    assert (run(1, logit_bias=bias, repetition_penalty=1.0, frequency_penalty=0.0, presence_penalty=0.0) == 777).all()
    allowed = torch.zeros(49152 // 32, dtype=torch.int32, device=cuda_dev)
    allowed[40000 // 32] = 3 << (40000 % 32)
    two = run(1, allowed=allowed, logit_bias=None)
    assert ((two == 40000) | (two == 40001)).all()
    with pytest.raises(ValueError):
        run(1, repetition_penalty=0.0)
    assert cache.free_pages == free  # and after a refusal in the middle too


@pytest.mark.gpu
def test_penalties_see_what_was_generated(cuda_dev, weights):
    """A frequency penalty above every difference of logits makes all tokens of a row differ; a repetition penalty
    above it keeps prompt and prefix tokens out as well."""
    model, ids, (prefix,) = model_on(cuda_dev, weights), some(7, *LENS), some(3, 100)
    out = model.generate(ids, 12, frequency_penalty=1e6, prefix=prefix).tolist()
    assert all(len(set(row)) == 12 for row in out)
    plain = model.generate(ids, 12, prefix=prefix).tolist()
    assert [r[0] for r in out] == [r[0] for r in plain]  # nothing generated yet: the prompt does not count
    out = model.generate(ids, 12, repetition_penalty=1e6, prefix=prefix).tolist()
    for row, p in zip(out, ids):
        assert len(set(row)) == 12 and not set(row) & (set(p) | set(prefix))


@pytest.mark.gpu
def test_8_bit_cache_keeps_close(cuda_dev, weights):
    """One decode step over an 8-bit cache: each cached value is off by at most 2^-4 of itself and the rest of the
    arithmetic is the same, so logits stay far nearer to the bf16 cache's than to another prompt's."""
    model, ids = model_on(cuda_dev, weights), some(7, *LENS)
    cu = torch.tensor([0] + LENS).cumsum(0).to(torch.int32).to(cuda_dev)
    flat, got = torch.tensor([t for p in ids for t in p], device=cuda_dev), []
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        seqs = model.new_paged_cache(40, 16, dtype).reserve([n + 8 for n in LENS])
        first = model.prefill_packed(flat, cu, seqs)
        got.append((first, model.decode_packed(torch.tensor([9, 8, 7, 6, 5], device=cuda_dev), seqs)))
    assert torch.equal(got[0][0], got[1][0])  # prompts attend the values before they are cached
    far = (got[0][1] - got[1][1]).norm(dim=-1)
    apart = (got[0][1] - got[0][1].roll(1, 0)).norm(dim=-1)
    assert torch.isfinite(got[1][1]).all() and (far < 0.25 * apart).all() and far.max() > 0


@pytest.mark.gpu
def test_refusals(cuda_dev, weights):
    model = model_on(cuda_dev, weights)
    for bad in (dict(prefix=[49152]), dict(prefix=[-1]), dict(prefix=[1] * 8190), dict(frequency_penalty=math.inf),
                dict(logit_bias=torch.zeros(5, device=cuda_dev))):
        with pytest.raises(ValueError):
            model.generate([[1, 2]], 4, **bad)
    cache = model.new_paged_cache(5, 16)
    with pytest.raises(ValueError):
        model.generate([[1], [2]], 4, cache=cache, prefix=[3] * 70)  # pages for the prefix and one prompt only
    assert cache.free_pages == 5
