"""Distilling another network as the integration notes show it."""

from __future__ import annotations

import pytest
import torch
from test_gpu_policy import DEV

pytestmark = pytest.mark.gpu


def test_a_teacher_network_with_weights_of_its_own():
    from ataraxos_b200 import StrategoRolloutBuffer
    from ataraxos_b200.policy import action_logprobs, distill_loss

    n = 8
    roots = StrategoRolloutBuffer(n, 0, seed=4, pool_size=64)
    roots.reset_all_from_pool()
    mask = roots.compute_legal_action_mask_bits()
    move_net, teacher_net = (torch.nn.Linear(6, 10000, device=DEV) for _ in range(2))
    info = torch.randn(n, 6, device=DEV)
    with torch.no_grad():
        best = action_logprobs(teacher_net(info), mask=mask, top=32, temperature=2.0)
    loss = distill_loss(move_net(info), best.top_action, best.top_logprob, mask, temperature=2.0, tail=True)
    loss.mean().backward()
    assert torch.isfinite(loss).all() and torch.isfinite(move_net.weight.grad).all() and move_net.weight.grad.any()
    assert teacher_net.weight.grad is None
    best = action_logprobs(teacher_net(info), mask=mask, top=32, temperature=2.0)
    with pytest.raises(RuntimeError, match="no gradient for teacher_logits"):
        distill_loss(move_net(info), best.top_action, best.top_logprob, mask, temperature=2.0, tail=True)
