"""Operands of the policy operators' gradients that point outside their rows: left out, never followed."""

from __future__ import annotations

import pytest
import torch
from test_gpu_policy import DEV, _actions, _mask_arg, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind, code", [("none", 0), ("u8", 1), ("bits", 2)])
@pytest.mark.parametrize("r, a", [(5, 50), (5, 128), (5, 3001), (5, 20000), (1300, 2600)])
def test_alternatives_outside_the_row_are_left_out(r, a, kind, code):
    """The alternatives are the caller's to keep between the passes: overwritten ones give what -1 gives."""
    from ataraxos_b200.policy import action_logprobs

    x, ok, g = _rows(r, a, torch.float32, 0.3)
    mask = _mask_arg(ok, kind)
    x, act = x.to(DEV), _actions(torch.ones_like(ok) if kind == "none" else ok, g).to(DEV)
    out = action_logprobs(x, act, mask, top=8)
    ops = torch.ops.stratego_b200
    stats = ops._action_logprobs(x, act, mask, code, 8, 1.0, True)[-1]
    gt = torch.randn((r, 8), generator=g).to(DEV)
    none, outside = out.top_action.clone(), out.top_action.clone()
    none[3, :4] = none[r - 1, 7] = -1
    outside[3, :4] = torch.tensor([a, -2, 1 << 40, (1 << 32) + 1], device=DEV)
    outside[r - 1, 7] = a + 15
    got, want = (ops._action_logprobs_backward(x, act, mask, code, t, out.entropy, stats, None, None, gt, 1.0)
                 for t in (outside, none))
    assert torch.equal(got, want)
