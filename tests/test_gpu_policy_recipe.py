"""The policy operators as the integration notes show them."""

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


@pytest.mark.parametrize("mask_format", ["bits", "u8"])
def test_equal_logits_give_the_rings_own_log_probabilities(mask_format):
    """A ring played by uniform moves, scored under equal logits: what it recorded, -log of the number of legal moves,
    and 0 where no move was made; the same bits slot by slot, as flat rows and for any equal logits."""
    from ataraxos_b200 import StrategoRolloutBuffer
    from ataraxos_b200.policy import action_logprobs
    from ataraxos_b200.trajectory import TrajectoryBuffer

    n, t = 24, 6
    b = StrategoRolloutBuffer(n, 0, seed=5, pool_size=64, max_game_length=4)
    b.reset_all_from_pool()
    ring = TrajectoryBuffer(b, t, obs_dtype=None, mask_format=mask_format, policy="uniform")
    ring.prime()
    ring.rollout(t - 1, auto_reset=False)
    moved = ring.action >= 0
    assert moved.any() and not moved.all()
    r = ring.action_logprobs(torch.zeros((t, n, 10000), device=DEV))
    assert torch.isfinite(r.logprob).all() and not r.logprob[~moved].any()
    # log1p of a count and its negative against the ring's own logarithm: 2 u each of values below 9.3
    assert ((r.logprob - ring.logprob)[moved].abs() <= 4 * 2.0 ** -24 * 9.3).all()
    assert torch.equal(r.entropy[moved], -r.logprob[moved])
    flat = action_logprobs(torch.full((t * n, 10000), 3.5, device=DEV), ring.action.view(-1), ring.mask.flatten(0, 1))
    assert torch.equal(flat.logprob.view(t, n), r.logprob) and torch.equal(flat.entropy.view(t, n), r.entropy)
    for s in range(t):
        one = ring.action_logprobs(torch.zeros((1, n, 10000), device=DEV), slice(s, s + 1))
        assert torch.equal(one.logprob[0], r.logprob[s])
