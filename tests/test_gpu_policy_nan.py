"""Rows with a legal NaN or +inf and no teacher entry that is kept."""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_policy import DEV, _mask_arg, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["none", "bits", "bool"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("a", [50, 600, 3001, 20000])
def test_spoiled_row_without_a_kept_entry(a, bad, kind, tail):
    """Loss and gradient of such a row are NaN together, those of its neighbours 0."""
    from ataraxos_b200.policy import distill_loss

    x, ok, _ = _rows(5, a, torch.float32, 0.3)
    ok[3, 7] = True
    x[3, 7] = bad
    ta = torch.full((5, 40), -1, dtype=torch.int64)
    ta[:, 35] = a                                         # past the last action
    lx = x.to(DEV).requires_grad_()
    loss = distill_loss(lx, ta.to(DEV), torch.zeros(5, 40, device=DEV), _mask_arg(ok, kind), tail=tail)
    grad = torch.autograd.grad(loss.sum(), lx)[0].cpu()
    legal = torch.ones(a, dtype=torch.bool) if kind == "none" else ok[3]
    assert loss[3].isnan() and grad[3][legal].isnan().all() and not grad[3][~legal].any()
    rest = [0, 1, 2, 4]
    assert not loss[rest].any()
    # tail: p (1 - q_r / p_r) with q_r = p_r = 1 up to rounding (33 terms in a lane's sum and its joins, 64 u)
    assert grad[rest].abs().max().item() <= 64 * 2.0 ** -24


@pytest.mark.parametrize("kind", ["none", "bits", "bool"])
@pytest.mark.parametrize("a", [50, 3001])
def test_spoiled_row_and_actions_without_a_probability(a, kind):
    """-1 keeps its 0 and an action that is not legal its -inf beside a legal NaN; the rest of the row is NaN."""
    from ataraxos_b200.policy import action_logprobs

    x, ok, _ = _rows(5, a, torch.float32, 0.3)
    ok[3:, 7] = True
    x[3:, 7] = math.nan
    out = action_logprobs(x.to(DEV), torch.tensor([-1, -1, -1, -1, a], device=DEV), _mask_arg(ok, kind), top=2)
    assert out.logprob.tolist() == [0.0, 0.0, 0.0, 0.0, -math.inf]
    assert out.entropy[3:].isnan().all() and out.top_logprob[3:].isnan().all()
    assert not out.entropy[:3].isnan().any()
