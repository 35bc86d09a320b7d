"""Operators on rows of policy logits under the simulator's legal masks.

``action_logprobs(logits, actions, mask, top=k)`` evaluates recorded actions
under a network's policy: the log-probability of each row's action under the
softmax of its legal logits, the entropy of that softmax and its ``k``
likeliest actions, with gradients to the logits.  It is the training-side
counterpart of the simulator's own sampling (``step(policy="gumbel",
logits=...)`` and ``sample_actions``): the reference's ``softmax`` +
``_map_policy_to_actions`` (stratego/training/selfplay.py:221-228, 301-317).

``distill_loss(logits, teacher_actions, teacher_logits, mask)`` pulls such a
policy towards a teacher that is known by its likeliest actions: another
network's ``action_logprobs(..., top=k)``, or a search policy
(``SearchResult.teacher``).

Both take the masks as the simulator writes them, uint8 / bool per action
(``[..., 10000]`` or ``[..., 100, 100]``) or bit-packed (``[..., 1250]``), and
any other number of actions A up to 65,536 (bit-packed: ``ceil(A / 8)`` bytes; a
mask of one byte for one action is that action's).  A masked-out logit is never looked
at, so it may be anything, NaN included.  Sums and statistics are float32 for
float32, bfloat16 and float16 logits alike; gradients are rounded once, to the
logits' type.  A legal NaN or +inf makes its row's results NaN (the
log-probability of an action that has none, -1 or not legal, aside).

Both launch on the current torch stream of the logits' device and can be
captured into a CUDA graph, gradients included (as with any torch operator, no
eager autograd graph of the same leaf tensor may be alive then).  The gradient
is computed from the logits, the mask and the listed actions again: leave them
unchanged until the backward pass has run (the masks and observations of
``step`` are overwritten by the next step; ``TrajectoryBuffer`` keeps them).
The gradients have no derivatives of their own, and there are none in forward
mode: a dual tensor is refused, and so is ``vmap``.  Fake tensors, traced graphs
(``make_fx``) and ``torch.compile`` take a call as one opaque operator for each
kernel; call an operator once before a compilation with ``fullgraph=True``, since
the first call binds the library.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _capi as C

MAX_ACTIONS = C.SB_POLICY_MAX_ACTIONS
MAX_TOP = C.SB_POLICY_MAX_TOP
MAX_TEACHER = C.SB_POLICY_MAX_TEACHER


@dataclass
class ActionLogProbs:
    """What :func:`action_logprobs` returns, shaped like the logits' leading dimensions ``[...]``."""

    logprob: torch.Tensor | None      # [...] float32 (None: no actions given)
    entropy: torch.Tensor             # [...] float32, nats
    top_action: torch.Tensor | None   # [...,k] int64, likeliest first (-1: no further action); None for top=0
    top_logprob: torch.Tensor | None  # [...,k] float32 (-inf there); None for top=0


_ops = None


def _load():
    """The torch operators over libstratego_b200 (``csrc/sb_torch.cpp``), bound to the library in use."""
    global _ops
    if _ops is None:
        lib = C.lib()
        if not C.TORCH_LIB_PATH.exists():
            raise ImportError(f"{C.TORCH_LIB_PATH} is missing: build it with `python -m ataraxos_b200.build`")
        torch.ops.load_library(str(C.TORCH_LIB_PATH))
        names = ("sb_action_logprobs", "sb_action_logprobs_backward", "sb_distill_loss", "sb_distill_loss_backward",
                 "sb_last_error")
        torch.ops.stratego_b200.bind([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names])
        ops = torch.ops.stratego_b200
        _ops = (ops.action_logprobs.default, ops.distill_loss.default)
    return _ops


def action_logprobs(
    logits: torch.Tensor,
    actions: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    *,
    top: int = 0,
    temperature: float = 1.0,
) -> ActionLogProbs:
    """Log-probabilities of given actions under ``softmax(logits / temperature)``
    over the legal actions, with entropy and the ``top`` likeliest actions.

    ``logits`` ``[..., A]`` float32 / bfloat16 / float16 on a CUDA device;
    ``actions`` ``[...]`` int16 / int32 / int64: -1 stands for "no action" (a
    finished game, padding) and gives log-probability 0 and no gradient; any
    other action that is not legal gives -inf and no gradient.  ``mask``: see
    the module; None makes every action legal; ``[A]`` (or size-1 dimensions)
    serves all rows.  A row without a legal action has entropy 0.

    The ``top`` (0..32) likeliest actions come in descending order, ties to
    the lower action; where a row has fewer of non-zero probability the rest
    are action -1 with log-probability -inf.  Gradients flow to ``logits``
    from ``logprob``, ``entropy`` and ``top_logprob``.
    """
    if not isinstance(logits, torch.Tensor):
        raise RuntimeError("logits must be a float32, bfloat16 or float16 tensor")
    out = (_ops or _load())[0](logits, actions, mask, top, temperature)
    lp = None if actions is None else out[1]
    return ActionLogProbs(lp, out[0], out[-1], out[-2]) if top else ActionLogProbs(lp, out[0], None, None)


def distill_loss(
    logits: torch.Tensor,
    teacher_actions: torch.Tensor,
    teacher_logits: torch.Tensor,
    mask: torch.Tensor | None = None,
    *,
    temperature: float = 1.0,
    tail: bool = False,
) -> torch.Tensor:
    """Divergence ``sum q (log q - log p)`` of the policy ``p`` (softmax of
    ``logits / temperature`` over the legal actions) from a teacher ``q`` given
    by up to 512 of its actions; float32 ``[...]``, one value per row.

    ``teacher_actions`` ``[..., K]`` int16 / int32 / int64 and
    ``teacher_logits`` ``[..., K]`` float32 / bfloat16 / float16.  Entries whose
    action is negative (padding) or not legal, or whose logit is -inf, are
    left out; an action listed twice counts twice.

    ``tail=False``: ``q`` is the softmax of ``teacher_logits / temperature`` over
    the entries that are left (log-probabilities serve as logits).
    ``tail=True``: ``teacher_logits`` are the teacher's log-probabilities at
    this temperature, as ``action_logprobs(..., top=K, temperature=...)`` gives
    them, and all legal actions that are not listed count as one entry: the
    teacher's mass left over against the policy's own mass on them.  Where the
    policy has no mass there (no such action, or less than ``e**-745``, as for
    actions masked inside the logits by -inf, -1e9 or the type's lowest value)
    what is left over is dropped.

    The gradient flows to ``logits`` only.  Multiply by ``temperature ** 2`` to
    keep its scale when mixing it with a loss at temperature 1.
    """
    if not (isinstance(logits, torch.Tensor) and isinstance(teacher_actions, torch.Tensor)
            and isinstance(teacher_logits, torch.Tensor)):
        raise RuntimeError("logits, teacher_actions and teacher_logits must be tensors")
    return (_ops or _load())[1](logits, teacher_actions, teacher_logits, mask, temperature, tail)


__all__ = ["ActionLogProbs", "action_logprobs", "distill_loss", "MAX_ACTIONS", "MAX_TOP", "MAX_TEACHER"]
