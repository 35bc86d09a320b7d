"""The policy operators under torch's other ways to run a function (CPU; no kernel is launched)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

from ataraxos_b200.policy import action_logprobs, distill_loss

X = torch.zeros(3, 20)
A = torch.zeros(3, dtype=torch.int64)
TA, TL = torch.zeros((3, 4), dtype=torch.int64), torch.zeros(3, 4)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", [
    lambda d: action_logprobs(d(X), A),
    lambda d: action_logprobs(d(X), top=2),
    lambda d: distill_loss(d(X), TA, TL),
    lambda d: distill_loss(d(X), TA, TL, tail=True),
    lambda d: distill_loss(X, TA, d(TL)),
])
def test_forward_mode_derivatives_are_refused(call, grad):
    """A tangent is refused, not dropped: torch takes an output without one for a constant."""
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(lambda t: fwad.make_dual(t, torch.ones_like(t)))
        # the tangent is not looked at where forward mode is off, nor in the primal
        with fwad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA device"):
            call(lambda t: fwad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="CUDA device"):
            call(lambda t: fwad.unpack_dual(fwad.make_dual(t, torch.ones_like(t))).primal)


def test_functional_forward_mode_is_refused():
    one = torch.ones_like(X)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: action_logprobs(x, A).logprob, (X,), (one,))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: distill_loss(x, TA, TL), (X,), (one,))
