"""Vocabularies whose slices stay in global memory: rows that start anywhere within 16 bytes, settings of their own,
parts without a usable logit. Compared with the definition in 64 bits; at least half of the rows of a call must be clear
of thresholds (test_sample_gpu.py's measure)."""
import math

import pytest
import torch

from test_sample_gpu import defined, draw

pytestmark = pytest.mark.gpu
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.9, 50, 0.95, 0.0), (1.0, 0, 1.0, 0.02), (0.0, 0, 1.0, 0.0), (0.8, 500, 1.0, 0.0)]


@pytest.mark.parametrize("V,dtype", [(850_003, torch.bfloat16), (420_001, torch.float32)])
@pytest.mark.parametrize("first", [0, 1, 5])
def test_rows_that_start_anywhere(cuda_dev, V, dtype, first):
    """Eight blocks a row: slices of more than 100 thousand bf16 or 50 thousand fp32 logits do not fit shared memory."""
    from npu_b200 import sample

    R = len(SETTINGS)
    wide, noise = draw(cuda_dev, R, V + 7, dtype, seed=V + first)  # rows V + 7 apart: each starts elsewhere
    x, e = wide[:, first:first + V], noise[:, 2:2 + V]
    x[1, :V // 3] = -math.inf
    x[2, V // 2:] = math.nan
    x[4, V - 1] = x[4].float().nan_to_num(-9).amax() + 1  # the last token leads
    x[0, V // 8:V // 4] = torch.finfo(dtype).min
    T, p, m = (torch.tensor([s[i] for s in SETTINGS], device=cuda_dev) for i in (0, 2, 3))
    k = torch.tensor([s[1] for s in SETTINGS], dtype=torch.int32, device=cuda_dev)
    got = sample(x, e, temperature=T, top_k=k, top_p=p, min_p=m).tolist()
    clear = 0
    for r, s in enumerate(SETTINGS):
        token, sure = defined(x[r].double().tolist(), e[r].double().tolist(), T[r].item(), s[1], p[r].item(),
                              m[r].item())
        if sure:
            clear += 1
            assert got[r] == token, f"row {r}"
    assert 2 * clear >= R
