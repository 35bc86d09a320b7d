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
any other number of actions up to 65,536.  A masked-out logit is never looked
at, so it may be anything, NaN included.  Sums and statistics are float32 for
float32, bfloat16 and float16 logits alike; gradients are rounded once, to the
logits' type.  A legal NaN or +inf makes its row's results NaN.

Both launch on the current torch stream of the logits' device and can be
captured into a CUDA graph, gradients included (as with any torch operator, no
eager autograd graph of the same leaf tensor may be alive then).  The gradient is computed from the logits, the
mask and the listed actions again: leave them unchanged until the backward
pass has run (the masks and observations of ``step`` are overwritten by the
next step; ``TrajectoryBuffer`` keeps them).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _capi as C
from .buffer import NUM_ACTIONS, NUM_SQUARES, _raw_stream, _vp

MAX_ACTIONS = C.SB_POLICY_MAX_ACTIONS
MAX_TOP = C.SB_POLICY_MAX_TOP
MAX_TEACHER = C.SB_POLICY_MAX_TEACHER

_DTYPES = {torch.float32: C.SB_DTYPE_F32, torch.bfloat16: C.SB_DTYPE_BF16, torch.float16: C.SB_DTYPE_F16}
_INDEX_BYTES = {torch.int16: 2, torch.int32: 4, torch.int64: 8}


@dataclass
class ActionLogProbs:
    """What :func:`action_logprobs` returns, shaped like the logits' leading dimensions ``[...]``."""

    logprob: torch.Tensor | None      # [...] float32 (None: no actions given)
    entropy: torch.Tensor             # [...] float32, nats
    top_action: torch.Tensor | None   # [...,k] int64, likeliest first (-1: no further action); None for top=0
    top_logprob: torch.Tensor | None  # [...,k] float32 (-inf there); None for top=0


def _call(name: str, dev: torch.device, *args) -> None:
    """The library's entry point ``name`` on the current stream of ``dev``."""
    index = dev.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(dev):
            rc = getattr(C.lib(), name)(*args, _raw_stream(index))
    else:
        rc = getattr(C.lib(), name)(*args, _raw_stream(index))
    if rc:
        C.check(rc)


def _check_logits(logits: torch.Tensor, temperature: float) -> None:
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        raise RuntimeError("logits must be a float32, bfloat16 or float16 tensor")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_ACTIONS:
        raise RuntimeError(f"logits must be [..., A] with 1 <= A <= {MAX_ACTIONS}, got {tuple(logits.shape)}")
    if not (math.isfinite(temperature) and temperature >= 1e-30):
        raise RuntimeError(f"temperature must be finite and at least 1e-30, got {temperature}")


def _check_cuda(logits: torch.Tensor) -> None:
    if not logits.is_cuda:
        raise RuntimeError("logits must be on a CUDA device (there is no CPU fallback)")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t [..., W]`` as ``[R, W]`` with adjacent elements of a row adjacent in
    memory: a view where its strides allow one, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _mask_rows(mask: torch.Tensor | None, logits: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    """The mask as ``[R, W]`` bytes (W = A, or ceil(A / 8) for bits) and its kind."""
    if mask is None:
        return None, C.SB_MASK_NONE
    if not isinstance(mask, torch.Tensor) or mask.dtype not in (torch.bool, torch.uint8):
        raise RuntimeError("mask must be a bool or uint8 tensor")
    if mask.device != logits.device:
        raise RuntimeError(f"mask is on {mask.device}, the logits are on {logits.device}")
    a, lead = logits.shape[-1], logits.shape[:-1]
    if a == NUM_ACTIONS and mask.dim() >= 2 and tuple(mask.shape[-2:]) == (NUM_SQUARES, NUM_SQUARES):
        mask = mask.flatten(-2)
    width = mask.shape[-1] if mask.dim() else 0
    if width == a:
        kind = C.SB_MASK_U8
    elif width == (a + 7) // 8 and mask.dtype is torch.uint8:
        kind = C.SB_MASK_BITS
    else:
        raise RuntimeError(f"mask must be [..., {a}] bool / uint8 or [..., {(a + 7) // 8}] bit-packed uint8 for "
                           f"{a} actions, got {tuple(mask.shape)} {mask.dtype}")
    if mask.shape[:-1] != lead:
        try:
            mask = mask.expand(*lead, width)
        except RuntimeError:
            raise RuntimeError(f"mask {tuple(mask.shape)} does not match logits {tuple(logits.shape)}") from None
    if mask.dim() == 1:
        mask = mask.unsqueeze(0)
    if mask.dim() > 2 and all(s == 0 for s, n in zip(mask.stride()[:-1], lead) if n > 1):
        mask = mask.as_strided((math.prod(lead), width), (0, mask.stride(-1)))  # one row for all
    return _rows(mask), kind


def _index_rows(t: torch.Tensor, shape, what: str, dev: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype not in _INDEX_BYTES:
        raise RuntimeError(f"{what} must be an int16, int32 or int64 tensor")
    if t.shape != shape:
        raise RuntimeError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise RuntimeError(f"{what} are on {t.device}, the logits are on {dev}")
    return t.contiguous()


def _logits_arg(x: torch.Tensor, mask: torch.Tensor | None, kind: int, temperature: float) -> C.SbLogits:
    return C.SbLogits(x.data_ptr(), _vp(mask), x.shape[0], x.stride(0),
                      0 if mask is None else mask.stride(0), x.shape[1], _DTYPES[x.dtype], kind, temperature)


def _row_grad(g: torch.Tensor | None) -> tuple[torch.Tensor | None, int]:
    """A per-row gradient and its stride; autograd's expanded scalars (of a sum or mean) stay one element."""
    if g is None:
        return None, 0
    if g.dtype is not torch.float32:
        g = g.float()
    if g.stride(0) not in (0, 1):
        g = g.contiguous()
    return g, g.stride(0)


def _logprobs_forward(x, x_arg, actions, top, keep):
    """Launch the forward kernel; returns the outputs and its C description (``keep``: with the backward's rows)."""
    r, dev = x.shape[0], x.device
    entropy = torch.empty(r, dtype=torch.float32, device=dev)
    logprob = None if actions is None else torch.empty_like(entropy)
    stats = torch.empty((r, 2), dtype=torch.float32, device=dev) if keep else None
    top_lp = top_action = None
    if top:
        top_lp = torch.empty((r, top), dtype=torch.float32, device=dev)
        top_action = torch.empty((r, top), dtype=torch.int64, device=dev)
    arg = C.SbLogprobs(_vp(actions), 0 if actions is None else actions.element_size(), top, _vp(logprob),
                       entropy.data_ptr(), _vp(stats), _vp(top_action), _vp(top_lp))
    if r:
        _call("sb_action_logprobs", dev, x_arg, arg)
    return logprob, entropy, top_lp, top_action, stats, arg


def _first_order(backward):
    """A backward pass without a derivative of its own: autograd's guard against
    differentiating it again costs microseconds, so it is put up only where a
    second derivative could be asked for (``create_graph=True``)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _repoint(x_arg: C.SbLogits, x: torch.Tensor, mask: torch.Tensor | None) -> C.SbLogits:
    """The description of the forward call for the saved tensors (saved-tensor hooks may have moved them)."""
    x_arg.logits, x_arg.row_stride = x.data_ptr(), x.stride(0)
    if mask is not None:
        x_arg.mask, x_arg.mask_stride = mask.data_ptr(), mask.stride(0)
    return x_arg


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mask, x_arg, actions, top):
        lp, ent, top_lp, top_action, stats, arg = _logprobs_forward(x, x_arg, actions, top, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, mask, actions, ent, top_action, stats)
        ctx.args = (x_arg, arg)
        if not top:
            return lp, ent
        ctx.mark_non_differentiable(top_action)
        return lp, ent, top_lp, top_action

    @staticmethod
    @_first_order
    def backward(ctx, g_lp, g_ent, g_top=None, _=None):
        x, mask, actions, ent, top_action, stats = ctx.saved_tensors
        x_arg, arg = ctx.args
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:
            g_lp, s_lp = _row_grad(g_lp)
            g_ent, s_ent = _row_grad(g_ent)
            g_top = None if g_top is None else g_top.float().contiguous()
            arg.actions, arg.entropy, arg.row_stats = _vp(actions), ent.data_ptr(), stats.data_ptr()
            arg.top_action = _vp(top_action)
            g = C.SbLogprobsGrad(_vp(g_lp), _vp(g_ent), _vp(g_top), s_lp, s_ent, grad.data_ptr())
            _call("sb_action_logprobs_backward", x.device, _repoint(x_arg, x, mask), arg, g)
        return grad, None, None, None, None


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
    _check_logits(logits, temperature)
    top = int(top)
    if not 0 <= top <= MAX_TOP:
        raise RuntimeError(f"top must be 0..{MAX_TOP}, got {top}")
    lead = logits.shape[:-1]
    m, kind = _mask_rows(mask, logits)
    if actions is not None:
        actions = _index_rows(actions, lead, "actions", logits.device)
    _check_cuda(logits)
    x = _rows(logits if logits.dim() > 1 else logits.unsqueeze(0))
    x_arg = _logits_arg(x, m, kind, temperature)
    top_lp = top_action = None
    if not (torch.is_grad_enabled() and x.requires_grad):
        lp, ent, top_lp, top_action, _, _ = _logprobs_forward(x, x_arg, actions, top, False)
    elif top:
        lp, ent, top_lp, top_action = _ActionLogProbs.apply(x, m, x_arg, actions, top)
    else:
        lp, ent = _ActionLogProbs.apply(x, m, x_arg, actions, 0)
    if len(lead) != 1:
        lp, ent = (None if t is None else t.view(lead) for t in (lp, ent))
        top_lp, top_action = (None if t is None else t.view(*lead, top) for t in (top_lp, top_action))
    return ActionLogProbs(lp, ent, top_action, top_lp)


def _distill_forward(x, x_arg, t_act, t_log, tail, keep):
    r, dev = x.shape[0], x.device
    loss = torch.empty(r, dtype=torch.float32, device=dev)
    stats = torch.empty((r, 6), dtype=torch.float32, device=dev) if keep else None
    arg = C.SbDistill(t_act.data_ptr(), t_log.data_ptr(), t_act.element_size(), _DTYPES[t_log.dtype], t_act.shape[1],
                      tail, loss.data_ptr(), _vp(stats))
    if r:
        _call("sb_distill_loss", dev, x_arg, arg)
    return loss, stats, arg


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mask, x_arg, t_act, t_log, tail):
        loss, stats, arg = _distill_forward(x, x_arg, t_act, t_log, tail, True)
        ctx.save_for_backward(x, mask, t_act, t_log, stats)
        ctx.args = (x_arg, arg)
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, g_loss):
        x, mask, t_act, t_log, stats = ctx.saved_tensors
        x_arg, arg = ctx.args
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:
            g_loss, stride = _row_grad(g_loss)
            arg.teacher_actions, arg.teacher_logits, arg.row_stats = t_act.data_ptr(), t_log.data_ptr(), stats.data_ptr()
            _call("sb_distill_loss_backward", x.device, _repoint(x_arg, x, mask), arg, g_loss.data_ptr(), stride,
                  grad.data_ptr())
        return grad, None, None, None, None, None


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
    teacher's mass left over against the policy's own mass on them.

    The gradient flows to ``logits`` only.  Multiply by ``temperature ** 2`` to
    keep its scale when mixing it with a loss at temperature 1.
    """
    _check_logits(logits, temperature)
    lead, dev = logits.shape[:-1], logits.device
    if not isinstance(teacher_actions, torch.Tensor) or teacher_actions.dim() != logits.dim():
        raise RuntimeError(f"teacher_actions must be [..., K] over the logits' leading dimensions {tuple(lead)}")
    k = teacher_actions.shape[-1]
    if not 1 <= k <= MAX_TEACHER:
        raise RuntimeError(f"teacher_actions must list 1..{MAX_TEACHER} actions per row, got {k}")
    t_act = _index_rows(teacher_actions, torch.Size((*lead, k)), "teacher_actions", dev)
    if not isinstance(teacher_logits, torch.Tensor) or teacher_logits.dtype not in _DTYPES:
        raise RuntimeError("teacher_logits must be a float32, bfloat16 or float16 tensor")
    if teacher_logits.shape != teacher_actions.shape or teacher_logits.device != dev:
        raise RuntimeError(f"teacher_logits must be {tuple(teacher_actions.shape)} on {dev}, got "
                           f"{tuple(teacher_logits.shape)} on {teacher_logits.device}")
    grad = torch.is_grad_enabled()
    if grad and teacher_logits.requires_grad:
        raise RuntimeError("distill_loss has no gradient for teacher_logits: detach them")
    m, kind = _mask_rows(mask, logits)
    _check_cuda(logits)
    x = _rows(logits if logits.dim() > 1 else logits.unsqueeze(0))
    x_arg = _logits_arg(x, m, kind, temperature)
    t_log = teacher_logits.contiguous()
    if len(lead) != 1:
        t_act, t_log = t_act.view(-1, k), t_log.view(-1, k)
    if grad and x.requires_grad:
        loss = _DistillLoss.apply(x, m, x_arg, t_act, t_log, 1 if tail else 0)
    else:
        loss, _, _ = _distill_forward(x, x_arg, t_act, t_log, 1 if tail else 0, False)
    return loss if len(lead) == 1 else loss.view(lead)


__all__ = ["ActionLogProbs", "action_logprobs", "distill_loss", "MAX_ACTIONS", "MAX_TOP", "MAX_TEACHER"]
