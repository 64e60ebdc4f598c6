"""A store that is filled as it grows: slots that no row was written to score 0,
and a bias of minus infinity keeps them out of the best rows."""
import pytest
import torch

import insitu_b200 as ib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 20, 300])
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
def test_best_rows_of_a_half_empty_store(cuda_ok, m, t):
    g = torch.Generator(device="cuda").manual_seed(m)
    cap, d, n = 3000, 96, 700
    rows = -torch.rand(n, d, generator=g, device="cuda")         # every score is negative
    q = torch.rand(m, d, generator=g, device="cuda")
    slots = torch.randperm(cap, generator=g, device="cuda")[:n]
    store = ib.SQRows(cap, d).write(rows, slots)
    empty = torch.ones(cap, dtype=torch.bool, device="cuda")
    empty[slots] = False
    plain = store.scores(q, dtype=t)
    assert (plain[:, empty] == 0).all() and (plain[:, ~empty] < 0).all()
    bias = torch.full((cap,), float("-inf"), device="cuda")
    bias[slots] = 0
    masked = store.scores(q, bias=bias, dtype=t)
    assert (masked[:, empty] == float("-inf")).all() and torch.equal(masked[:, ~empty], plain[:, ~empty])
    assert not empty[masked.topk(100, dim=1).indices].any()
