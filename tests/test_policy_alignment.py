"""The policy operators' C entry points refuse pointers that are not aligned to their type (CPU; no launch)."""

from __future__ import annotations

import pytest

from ataraxos_b200 import _capi as C

PTR = 1 << 20  # never read: every call below is refused before a launch


def _x():
    return C.SbLogits(logits=PTR, mask=None, n_rows=3, row_stride=20, mask_stride=0, n_actions=20, dtype=0, mask_kind=0,
                      temperature=1.0)


def _refused(rc):
    return rc == C.SB_E_ARG and b"aligned" in C.lib().sb_last_error()


FORWARD = dict(actions=PTR, action_bytes=4, top=3, logprob=PTR, entropy=PTR, row_stats=PTR, top_action=PTR, top_logprob=PTR)
TEACHER = dict(teacher_actions=PTR, teacher_logits=PTR, action_bytes=8, teacher_dtype=0, listed=4, tail=0, loss=PTR,
               row_stats=PTR)


@pytest.mark.parametrize("name, by", [("logprob", 2), ("entropy", 1), ("row_stats", 4), ("top_action", 4),
                                      ("top_logprob", 2)])
def test_logprobs_outputs(name, by):
    assert _refused(C.lib().sb_action_logprobs(_x(), C.SbLogprobs(**{**FORWARD, name: PTR + by}), None))


@pytest.mark.parametrize("name, by", [("row_stats", 4), ("entropy", 2), ("top_action", 4), ("actions", 2)])
def test_logprobs_backward_operands(name, by):
    g = C.SbLogprobsGrad(g_top=PTR, grad=PTR)
    assert _refused(C.lib().sb_action_logprobs_backward(_x(), C.SbLogprobs(**{**FORWARD, name: PTR + by}), g, None))


@pytest.mark.parametrize("name, by", [("g_logprob", 2), ("g_entropy", 1), ("g_top", 2), ("grad", 2)])
def test_logprobs_backward_gradients(name, by):
    g = C.SbLogprobsGrad(**{**dict(g_logprob=PTR, g_entropy=PTR, g_top=PTR, grad=PTR), name: PTR + by})
    assert _refused(C.lib().sb_action_logprobs_backward(_x(), C.SbLogprobs(**FORWARD), g, None))


@pytest.mark.parametrize("name, by", [("loss", 2), ("row_stats", 4), ("teacher_logits", 2)])
def test_distill_operands(name, by):
    assert _refused(C.lib().sb_distill_loss(_x(), C.SbDistill(**{**TEACHER, name: PTR + by}), None))


@pytest.mark.parametrize("g_loss, grad", [(PTR + 2, PTR), (PTR, PTR + 2)])
def test_distill_backward_gradients(g_loss, grad):
    assert _refused(C.lib().sb_distill_loss_backward(_x(), C.SbDistill(**TEACHER), g_loss, 1, grad, None))
