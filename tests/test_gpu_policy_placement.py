"""What a policy row's results owe to where the row lies in memory."""

from __future__ import annotations

import pytest
import torch
from test_gpu_policy import DEV, INF, Policy, _actions, _close, _mask_arg, _rows

pytestmark = pytest.mark.gpu


def _run(x, act, mask):
    from ataraxos_b200.policy import action_logprobs

    x = x.detach().requires_grad_()
    o = action_logprobs(x, act, mask, top=4)
    return o.logprob, o.entropy, o.top_action, o.top_logprob, torch.autograd.grad(o.logprob.sum(), x)[0]


def _inputs(a, density, dtype, kind):
    x, ok, g = _rows(40, a, dtype, density, seed=a)
    act = _actions(torch.ones_like(ok) if kind == "none" else ok, g)
    return x, ok, act, x.to(DEV), act.to(DEV), _mask_arg(ok, kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["bits", "bool"])
@pytest.mark.parametrize("a, density", [(9999, 0.004), (2501, 0.03), (20001, 0.3), (100, 0.5), (61, 1.0)])
def test_listed_and_small_rows_keep_their_bits_anywhere(a, density, kind, dtype):
    """Masked rows whose legal actions are listed, and rows of up to 128 actions: a copy of a row on its own, at
    another alignment, has the same bits."""
    _, _, _, x, act, mask = _inputs(a, density, dtype, kind)
    whole = _run(x, act, mask)
    for i in (0, 1, 7, 39):
        for p, q in zip(whole, _run(x[i:i + 1].clone(), act[i:i + 1], mask[i:i + 1].clone())):
            assert torch.equal(p[i:i + 1], q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind, a, density", [("none", 9999, 1.0), ("none", 601, 1.0), ("bits", 9999, 0.6),
                                              ("bool", 2501, 0.5)])
def test_rows_read_whole_agree_within_rounding_anywhere(kind, a, density, dtype):
    """Rows that are read whole are dealt to the lanes by sectors of memory: their sums' order, and so their last bits,
    go with the alignment.  Both placements lie within the bounds of the definition, so within twice those of each
    other; the alternatives are the same."""
    x, ok, act, dx, dact, mask = _inputs(a, density, dtype, kind)
    okk = torch.ones_like(ok) if kind == "none" else ok
    P = Policy(x, okk, 1.0)
    at = act.clamp(min=0)[:, None]
    lp_tol = P.lp_tol.gather(1, at)[:, 0]
    whole = _run(dx, dact, mask)
    for i in (0, 1, 7, 39):
        one = _run(dx[i:i + 1].clone(), dact[i:i + 1], None if mask is None else mask[i:i + 1].clone())
        _close(one[0], whole[0][i:i + 1], 2 * lp_tol[i:i + 1])
        _close(one[1], whole[1][i:i + 1], 2 * P.h_tol[i:i + 1])
        assert torch.equal(one[2], whole[2][i:i + 1])
        best = one[2].cpu().clamp(min=0)
        top_tol = torch.where(one[3].cpu() > -INF, P.lp_tol[i:i + 1].gather(1, best), 0.0)
        _close(one[3], whole[3][i:i + 1], 2 * top_tol)
        # -p (and 1 - p at the action): p to its relative bound, two roundings of the result each
        p = P.p[i:i + 1]
        _close(one[4], whole[4][i:i + 1], 2 * p * (P.p_rel[i:i + 1] + 2.0 ** -22) + 2.0 ** -22 * whole[4][i:i + 1].cpu().abs()
               .double() + (0 if dtype is torch.float32 else torch.finfo(dtype).eps / 2 * p), dtype)
