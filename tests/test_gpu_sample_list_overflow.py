"""Top-k of a few whose border lies among more equal tokens than the sorted list holds, so that the row goes on to the bins:
all threads have to leave the list together. Many calls of many rows, each with the same answer: the u-th of the first k."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 148, 300])
@pytest.mark.parametrize("top_p", [False, True])
def test_more_equal_tokens_than_the_list_holds(dtype, rows, top_p):
    v, k = 8700, 200
    x = torch.full((rows, v), -1.0)
    x[:, 40:] = 1.5  # 8660 equal ones
    x[::2, 8000] = 4.0
    x = x.to(dtype).to(DEV)
    u = (torch.arange(rows) + 0.37) / rows
    # by hand: k tokens of weight 1 from token 40 on; or the large one, of weight e^2.5, and k - 1 of weight 1
    share = 0.5 if top_p else 1.0
    want = []
    for r in range(rows):
        if r % 2:
            kept, large = int(k * share), 0.0
        else:
            large = torch.tensor(2.5).double().exp().item()
            kept = -int(-(share * (k - 1 + large) - large) // 1) if top_p else k - 1
        at = u[r].item() * (kept + large)
        assert abs(at - round(at)) > 1e-4
        want.append(40 + int(at) if at < kept else 8000)
    ids, logp = torch.empty(rows, dtype=torch.int64, device=DEV), torch.empty(rows, device=DEV)
    u, t = u.to(DEV), torch.ones(rows, device=DEV)
    args = torch.full((rows,), k, dtype=torch.int32, device=DEV), torch.full((rows,), 0.5, device=DEV) if top_p else None, None
    wrong, bits = torch.zeros((), dtype=torch.int64, device=DEV), None
    expected = torch.tensor(want, device=DEV)
    for _ in range(200):
        torch.ops.cdb.sample_tokens(x, u, t, *args, ids, logp)
        bits = logp.clone() if bits is None else bits
        wrong += (ids != expected).sum() + (logp != bits).sum()
    assert int(wrong) == 0, (ids.tolist(), want)
