"""Distillation with the rest of the legal actions as one entry (``tail=True``), where
the student puts next to nothing, or nothing at all, on that rest.

Oracle and rounding bounds are those of ``test_gpu_policy``: float64, in which a
mass of e**-700 is still a number and one below e**-745 is 0.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_policy import _check_distill, _teacher

pytestmark = pytest.mark.gpu

# rows of eight lanes, of a warp and of four warps, unmasked and masked
WIDTHS = [50, 128, 600, 2000, 10000, 20000]


@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("a", WIDTHS)
@pytest.mark.parametrize("dtype, density", [(torch.float32, 0.05), (torch.bfloat16, 0.7)])
@pytest.mark.parametrize("t", [1.0, 0.1])
def test_rest_far_below_the_listed_actions(t, dtype, density, a, kind):
    """Gaps of 80 to 300 nats: p_r leaves float32's range and q_r / p_r does too; the gradient stays within q_r.
    The second row's upstream weight is 0."""
    g = torch.Generator().manual_seed(a)
    gaps = torch.tensor([80.0, 90.0, 110.0, 300.0])
    ok = torch.rand((4, a), generator=g) < density
    ok[:, :5] = True
    x = torch.randn((4, a), generator=g) - gaps[:, None]
    x[:, :3] = torch.tensor([0.0, -1.0, 0.5])
    x = (x * t).to(dtype)
    ta = torch.tensor([[0, 1, 2]]).expand(4, 3).contiguous()
    tl = torch.log(torch.tensor([[0.5, 0.3, 0.1]])).expand(4, 3).contiguous()
    loss, grad = _check_distill(x, ok, ta, tl, kind, t, True)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and not grad[1].any()


@pytest.mark.parametrize("kind", ["none", "bits"])
@pytest.mark.parametrize("a", WIDTHS)
def test_rest_far_below_many_listed_actions(a, kind):
    """40 listed actions (entries in two groups of 32), one of them twice, beside a rest 200 nats below."""
    g = torch.Generator().manual_seed(a + 1)
    ok = torch.rand((3, a), generator=g) < 0.5
    ok[:, :40] = True
    x = torch.randn((3, a), generator=g)
    x[:, 40:] -= 200.0
    ta, tl = _teacher(x, ok, 40, g, True, 1.0)
    tl -= 0.25                                            # a fifth of the teacher's mass is left over
    ta[1, 35] = ta[1, 2]
    tl[1, 35] = -7.0
    loss, grad = _check_distill(x, ok, ta, tl, kind, 1.0, True)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("a", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spare", [0.0, 0.3])
def test_rest_without_mass(spare, dtype, a, kind):
    """Moves masked inside the logits (-1e9, the type's lowest value, -inf on places that the mask allows) and a teacher
    that lists all real ones: what rounding (or ``spare``) leaves of its mass is not set against nothing."""
    g = torch.Generator().manual_seed(a)
    ok = torch.rand((4, a), generator=g) < 0.4
    ok[:, :12] = True
    low = torch.finfo(dtype).min
    x = torch.randn((4, a), generator=g)
    x[:, 12:] = torch.tensor([max(-1e9, low), low, -float("inf"), -2000.0])[:, None]
    x = x.to(dtype)
    real = torch.zeros_like(ok)
    real[:, :12] = True
    ta, tl = _teacher(x, real, 12, g, True, 1.0)
    tl += torch.log1p(torch.tensor(-spare))
    loss, grad = _check_distill(x, ok, ta, tl, kind, 1.0, True)
    assert loss.abs().max().item() < 20 and torch.isfinite(grad).all()
    assert not grad[:, 12:].any()
