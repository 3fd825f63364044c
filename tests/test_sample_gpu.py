"""Sampling against its definition in 64 bits. fp32 weights and their sums are
within 1e-5 of themselves: a token that close to a threshold may be in or out,
and a row is compared unless such a token, or a race that close, decides it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def defined(x, e, T, k, p, m):
    """(token, clear): one row, lists in 64 bits."""
    x = [-math.inf if math.isnan(t) else t for t in x]
    top = max(x)
    if top == -math.inf:
        return -1, True
    if not T > 0:
        return x.index(top), True
    w = [1.0 if t == top else (math.exp((t - top) / T) if top < math.inf else 0.0) for t in x]
    order = sorted((i for i in range(len(x)) if x[i] > -math.inf), key=lambda i: -x[i])
    total, ahead = math.fsum(w), 0.0
    kept, maybe = [], [0.0]
    for rank, i in enumerate(order):
        close = False
        if rank:
            if (k > 0 and rank >= k) or (p < 1 and ahead >= (p + 1e-5) * total) or w[i] < m * (1 - 1e-5):
                break
            close = (p < 1 and ahead > (p - 1e-5) * total) or w[i] < m * (1 + 1e-5)
        ahead += w[i]
        if close:
            maybe.append(w[i] / e[i])
        else:
            kept.append((w[i] / e[i], -i))
    kept.sort(reverse=True)
    best = kept[0][0]
    second = next((r for r, _ in kept[1:] if r != best), 0.0)
    return -kept[0][1], best == 0 or max(second, *maybe) < best * (1 - 1e-5)


def compare(logits, noise, T, k, p, m, rows=None):
    from npu_b200 import sample

    got = sample(logits, noise, temperature=T, top_k=k, top_p=p, min_p=m)
    if rows is not None:  # of these only
        logits, noise, got = logits[rows], noise[rows], got[rows]
    got = got.tolist()
    R = logits.shape[0]
    rows = [t.tolist() if isinstance(t, torch.Tensor) else [t] * R for t in (T, k, p, m)]
    x, e = logits.double().tolist(), noise.double().tolist()
    unclear = 0
    for r in range(R):
        token, clear = defined(x[r], e[r], *(t[r] for t in rows))
        if clear:
            assert got[r] == token, f"row {r}"
        else:
            unclear += 1
    assert unclear <= max(1, R // 50)


def draw(dev, R, V, dtype=torch.float32, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (spread * torch.randn(R, V, generator=g, device=dev)).to(dtype)
    return x, torch.empty(R, V, device=dev).exponential_(generator=g).clamp_(min=1e-20)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.9, 200, 0.95, 0.01),
            (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 2.0), (5.0, 10 ** 9, 0.999, 0.0), (0.0, 5, 0.5, 0.5),
            (0.01, 3, 0.5, 0.0), (40.0, 0, 0.3, 0.0)]


@pytest.mark.parametrize("T,k,p,m", SETTINGS)
@pytest.mark.parametrize("R,V,dtype", [(7, 1, torch.float32), (5, 2, torch.bfloat16), (9, 33, torch.float32),
                                       (12, 1000, torch.bfloat16), (6, 4097, torch.float32),
                                       (4, 49152, torch.float32), (3, 131071, torch.bfloat16)])
def test_settings_and_sizes(cuda_dev, T, k, p, m, R, V, dtype):
    compare(*draw(cuda_dev, R, V, dtype, seed=V + R), T, k, p, m)


@pytest.mark.parametrize("T,k,p,m", [SETTINGS[0], SETTINGS[1], SETTINGS[4], SETTINGS[9]])
@pytest.mark.parametrize("V,dtype", [(300_001, torch.bfloat16), (450_000, torch.float32)])
def test_vocabularies_past_a_slice_of_shared_memory(cuda_dev, T, k, p, m, V, dtype):
    compare(*draw(cuda_dev, 1, V, dtype, seed=V), T, k, p, m)


@pytest.mark.parametrize("R,V,dtype", [(300, 700, torch.float32), (64, 5001, torch.bfloat16)])
def test_each_row_its_own_settings(cuda_dev, R, V, dtype):
    x, e = draw(cuda_dev, R, V, dtype, seed=R)
    pick = [SETTINGS[r % len(SETTINGS)] for r in range(R)]
    T, p, m = (torch.tensor([s[i] for s in pick], dtype=torch.float32, device=cuda_dev) for i in (0, 2, 3))
    compare(x, e, T, torch.tensor([s[1] for s in pick], dtype=torch.int32, device=cuda_dev), p, m)


def test_ties_go_by_index(cuda_dev):
    from npu_b200 import sample

    x = torch.zeros(4, 3000, device=cuda_dev)
    x[1, 100:200] = 1.0
    x[2, ::7] = 2.0
    x[3] = -0.0
    x[3, 5:] = 0.0
    e = draw(cuda_dev, 4, 3000, seed=1)[1]
    assert sample(x, e, temperature=0.0).tolist() == [0, 100, 0, 0]
    for k in (1, 2, 10, 150):
        compare(x, e, 1.0, k, 1.0, 0.0)
    compare(x, e, 1.0, 0, 0.3, 0.0)
    e[:] = 1.0  # the race itself ties
    assert sample(x, e).tolist() == [0, 100, 0, 0]


def test_infinities_nan_and_rows_without_a_token(cuda_dev):
    from npu_b200 import sample

    x, e = draw(cuda_dev, 7, 500, seed=2)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :] = -math.inf
    x[2, 77] = -3.0
    x[3, 100:400] = -math.inf
    x[4, 9] = x[4, 300] = math.inf
    x[5, ::2] = math.nan
    x[6] = torch.finfo(torch.float32).min
    x[6, 450:] = 1.0
    for T, k, p, m in SETTINGS:
        compare(x, e, T, k, p, m)
    assert sample(x, e)[:3].tolist() == [-1, -1, 77]
    assert sample(x, e)[4].item() in (9, 300)
    low = torch.full((1, 500), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device=cuda_dev)
    compare(low, e[:1], 1.0, 7, 0.5, 0.0)


def test_greedy_needs_no_noise_and_strided_rows(cuda_dev):
    from npu_b200 import sample

    x, e = draw(cuda_dev, 6, 1003, seed=3)
    assert torch.equal(sample(x, temperature=0.0), x.argmax(-1))
    wide, noise = draw(cuda_dev, 6, 1200, seed=4)
    compare(wide[:, 3:1001], noise[:, 5:1003], 1.0, 40, 0.9, 0.0)
    assert torch.equal(sample(wide[::2, 1:], temperature=0.0), wide[::2, 1:].argmax(-1))


def test_tokens_come_up_as_often_as_their_weight(cuda_dev):
    """20000 rows of the same 50 logits, top-p 0.8: counts within 5 standard deviations of the kept weights."""
    from npu_b200 import sample

    n, V = 20000, 50
    x = draw(cuda_dev, 1, V, seed=5)[0].expand(n, V)
    e = draw(cuda_dev, n, V, seed=6)[1]
    got = torch.bincount(sample(x, e, temperature=1.5, top_p=0.8), minlength=V).double().cpu()
    w = torch.softmax(x[0].double().cpu() / 1.5, 0)
    ranked, order = torch.sort(w, descending=True, stable=True)
    kept = torch.zeros(V, dtype=torch.bool)
    kept[order[(ranked.cumsum(0) - ranked) < 0.8]] = True
    w = torch.where(kept, w, 0) / w[kept].sum()
    assert (got[~kept] == 0).all()
    assert ((got - n * w).abs() <= 5 * (n * w * (1 - w)).sqrt() + 1).all()


def test_noise_against_the_ranking_still_ends(cuda_dev):
    """Noise that makes every race's winner the last in rank, the worst order for a search by rejection."""
    x = torch.linspace(0, -5, 3000, device=cuda_dev)[None].repeat(2, 1)
    e = torch.exp(2 * x) + 1e-6
    compare(x, e, 1.0, 5, 1.0, 0.0)


@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.4, 0.0), (0, 1.0, 0.5)])
def test_an_infinite_temperature_weighs_all_logits_alike(cuda_dev, k, p, m):
    x, e = draw(cuda_dev, 6, 9001, seed=8)
    x[1, ::3] = torch.finfo(torch.float32).min
    T = torch.tensor([math.inf, math.inf, 1.0, math.inf, 1e30, math.inf], device=cuda_dev)
    compare(x, e, T, k, p, m)


@pytest.mark.parametrize("T,k,p,m", SETTINGS)
@pytest.mark.parametrize("R,V,dtype", [(6, 40_001, torch.float32), (160, 20_000, torch.bfloat16)])
def test_a_row_whose_parts_differ(cuda_dev, T, k, p, m, R, V, dtype):
    """Long rows are shared by several blocks: parts without a usable logit, far below the row's maximum, or with
    its only infinities."""
    x, e = draw(cuda_dev, R, V, dtype, seed=9)
    x[0, : V // 2] = -math.inf
    x[1, V // 8 :] = math.nan
    x[2, : V - V // 8] -= 60
    x[3, V // 3] = x[3, V - 2] = math.inf
    x[4, V // 4 : V // 2] = torch.finfo(dtype).min
    x[5] = -math.inf
    near = torch.cat([torch.arange(6), torch.arange(R - 2, R)]).to(cuda_dev) if R > 8 else slice(None)
    compare(x, e, T, k, p, m, near)
