"""The policy operators' argument checks and C structs (CPU; no kernel is launched).

Every refusal of ``action_logprobs`` / ``distill_loss`` that does not depend on
a device is raised before the device check, so it is tested here with CPU
tensors; the C entry points refuse on their own before they launch.
"""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from ataraxos_b200 import _capi as C
from ataraxos_b200.policy import action_logprobs, distill_loss

ROOT = Path(__file__).resolve().parent.parent

X = torch.zeros(3, 20)
A = torch.zeros(3, dtype=torch.int64)
TA, TL = torch.zeros((3, 4), dtype=torch.int64), torch.zeros(3, 4)


@pytest.mark.parametrize("match, args, kw", [
    ("float32, bfloat16 or float16", (X.double(),), {}),
    ("float32, bfloat16 or float16", ([1.0],), {}),
    ("float32, bfloat16 or float16", (X.long(),), {}),
    ("1 <= A", (torch.zeros(3, 0),), {}),
    ("1 <= A", (torch.zeros(1, 65537),), {}),
    ("1 <= A", (torch.zeros(()),), {}),
    ("temperature", (X,), {"temperature": 0.0}),
    ("temperature", (X,), {"temperature": -1.0}),
    ("temperature", (X,), {"temperature": math.inf}),
    ("temperature", (X,), {"temperature": math.nan}),
    ("temperature", (X,), {"temperature": 1e-40}),
    ("top must be", (X,), {"top": 33}),
    ("top must be", (X,), {"top": -1}),
    ("bool or uint8", (X, A, torch.zeros(3, 20)), {}),
    ("mask must be", (X, A, torch.zeros(3, 19, dtype=torch.uint8)), {}),
    ("mask must be", (X, A, torch.zeros(3, 3, dtype=torch.bool)), {}),
    ("mask must be", (X, A, torch.zeros((), dtype=torch.bool)), {}),
    ("does not match", (X, A, torch.zeros(4, 20, dtype=torch.bool)), {}),
    ("does not match", (X, A, torch.zeros(2, 3, 20, dtype=torch.bool)), {}),
    ("actions must be an int", (X, A.float()), {}),
    ("actions must have shape", (X, A[:2]), {}),
    ("actions must have shape", (X, A[:, None]), {}),
    ("CUDA device", (X, A, torch.zeros(3, 3, dtype=torch.uint8)), {"top": 4}),
])
def test_action_logprobs_refuses(match, args, kw):
    with pytest.raises(RuntimeError, match=match):
        action_logprobs(*args, **kw)


@pytest.mark.parametrize("match, args, kw", [
    ("float32, bfloat16 or float16", (X.double(), TA, TL), {}),
    ("temperature", (X, TA, TL), {"temperature": 0.0}),
    ("teacher_actions must be", (X, TA[0], TL), {}),
    ("must list 1..512", (X, TA[:, :0], TL[:, :0]), {}),
    ("must list 1..512", (X, torch.zeros((3, 513), dtype=torch.int64), torch.zeros(3, 513)), {}),
    ("teacher_actions must be an int", (X, TL, TL), {}),
    ("teacher_actions must have shape", (X, TA[:2], TL[:2]), {}),
    ("teacher_logits must be a float", (X, TA, TL.double()), {}),
    ("teacher_logits must be", (X, TA, TL[:, :3]), {}),
    ("no gradient for teacher_logits", (X, TA, TL.clone().requires_grad_()), {}),
    ("bool or uint8", (X, TA, TL, torch.zeros(3, 20)), {}),
    ("CUDA device", (X, TA, TL), {"tail": True}),
])
def test_distill_loss_refuses(match, args, kw):
    with pytest.raises(RuntimeError, match=match):
        distill_loss(*args, **kw)


def test_ring_without_masks_refuses():
    from ataraxos_b200.trajectory import TrajectoryBuffer

    ring = TrajectoryBuffer.__new__(TrajectoryBuffer)
    ring.mask = None
    with pytest.raises(RuntimeError, match="keeps no legal masks"):
        ring.action_logprobs(torch.zeros(1, 1, 10000))


PTR = 1 << 20  # never read: every call below is refused before a launch


def _x(**kw):
    base = dict(logits=PTR, mask=None, n_rows=3, row_stride=20, mask_stride=0, n_actions=20, dtype=0, mask_kind=0,
                temperature=1.0)
    return C.SbLogits(**{**base, **kw})


@pytest.mark.parametrize("message, kw", [
    (b"n_rows < 0", dict(n_rows=-1)),
    (b"n_actions", dict(n_actions=0)),
    (b"n_actions", dict(n_actions=65537)),
    (b"dtype", dict(dtype=3)),
    (b"mask kind", dict(mask_kind=3)),
    (b"temperature", dict(temperature=0.0)),
    (b"temperature", dict(temperature=math.nan)),
    (b"temperature", dict(temperature=math.inf)),
    (b"temperature", dict(temperature=1e-40)),
    (b"negative row stride", dict(row_stride=-1)),
    (b"negative row stride", dict(mask_stride=-1)),
    (b"logits NULL", dict(logits=None)),
    (b"logits NULL or not aligned", dict(logits=PTR + 2)),
    (b"disagree", dict(mask_kind=1)),
    (b"disagree", dict(mask=PTR)),
])
def test_c_entry_points_refuse_bad_rows(message, kw):
    lib, x = C.lib(), _x(**kw)
    out = C.SbLogprobs(entropy=PTR)
    d = C.SbDistill(teacher_actions=PTR, teacher_logits=PTR, action_bytes=8, teacher_dtype=0, listed=4, tail=0,
                    loss=PTR, row_stats=PTR)
    for rc in (lib.sb_action_logprobs(x, out, None),
               lib.sb_action_logprobs_backward(x, out, C.SbLogprobsGrad(grad=PTR), None),
               lib.sb_distill_loss(x, d, None),
               lib.sb_distill_loss_backward(x, d, PTR, 1, PTR, None)):
        assert rc == C.SB_E_ARG
        assert message in lib.sb_last_error()


@pytest.mark.parametrize("message, kw", [
    (b"top must", dict(top=33)),
    (b"top must", dict(top=-1)),
    (b"wide", dict(actions=PTR, action_bytes=3, logprob=PTR)),
    (b"not aligned", dict(actions=PTR + 4, action_bytes=8, logprob=PTR)),
    (b"entropy is NULL", dict(entropy=None)),
    (b"disagree", dict(actions=PTR, action_bytes=8)),
    (b"disagree", dict(logprob=PTR)),
    (b"top outputs", dict(top=4, top_action=PTR)),
])
def test_c_logprobs_refuses(message, kw):
    assert C.lib().sb_action_logprobs(_x(), C.SbLogprobs(**{**dict(entropy=PTR), **kw}), None) == C.SB_E_ARG
    assert message in C.lib().sb_last_error()


@pytest.mark.parametrize("message, fwd, g", [
    (b"grad, row_stats", dict(), dict()),
    (b"grad, row_stats", dict(row_stats=None), dict(grad=PTR)),
    (b"did not have", dict(), dict(grad=PTR, g_logprob=PTR)),
    (b"did not have", dict(), dict(grad=PTR, g_top=PTR)),
    (b"not aligned", dict(), dict(grad=PTR + 2)),
])
def test_c_logprobs_backward_refuses(message, fwd, g):
    f = C.SbLogprobs(**{**dict(entropy=PTR, row_stats=PTR), **fwd})
    assert C.lib().sb_action_logprobs_backward(_x(), f, C.SbLogprobsGrad(**g), None) == C.SB_E_ARG
    assert message in C.lib().sb_last_error()


@pytest.mark.parametrize("message, kw", [
    (b"listed must", dict(listed=0)),
    (b"listed must", dict(listed=513)),
    (b"wide", dict(action_bytes=1)),
    (b"teacher dtype", dict(teacher_dtype=7)),
    (b"tail must", dict(tail=2)),
    (b"are NULL", dict(teacher_logits=None)),
    (b"not aligned", dict(teacher_actions=PTR + 2)),
    (b"loss is NULL", dict(loss=None)),
])
def test_c_distill_refuses(message, kw):
    base = dict(teacher_actions=PTR, teacher_logits=PTR, action_bytes=8, teacher_dtype=0, listed=4, tail=0, loss=PTR)
    d = C.SbDistill(**{**base, **kw})
    assert C.lib().sb_distill_loss(_x(), d, None) == C.SB_E_ARG
    assert message in C.lib().sb_last_error()


def test_null_descriptions_are_refused():
    lib = C.lib()
    assert lib.sb_action_logprobs(None, None, None) == C.SB_E_ARG
    assert lib.sb_action_logprobs(_x(), None, None) == C.SB_E_ARG
    assert lib.sb_action_logprobs_backward(_x(), C.SbLogprobs(entropy=PTR), None, None) == C.SB_E_ARG
    assert lib.sb_distill_loss(_x(), None, None) == C.SB_E_ARG
    assert lib.sb_distill_loss_backward(_x(), None, None, 1, None, None) == C.SB_E_ARG


def test_no_rows_is_no_launch():
    lib, x = C.lib(), _x(n_rows=0, logits=None)
    d = C.SbDistill(action_bytes=8, listed=1)
    assert lib.sb_action_logprobs(x, C.SbLogprobs(), None) == C.SB_OK
    assert lib.sb_action_logprobs_backward(x, C.SbLogprobs(), C.SbLogprobsGrad(), None) == C.SB_OK
    assert lib.sb_distill_loss(x, d, None) == C.SB_OK
    assert lib.sb_distill_loss_backward(x, d, None, 1, None, None) == C.SB_OK


_LAYOUT = r"""
#include <stdio.h>
#include <stddef.h>
#include "stratego_b200.h"
int main(void) {
  printf("%zu %zu %zu %zu\n", sizeof(sb_logits), sizeof(sb_logprobs), sizeof(sb_logprobs_grad), sizeof(sb_distill));
  printf("%zu %zu %zu %zu\n", offsetof(sb_logits, temperature), offsetof(sb_logprobs, top_logprob),
         offsetof(sb_logprobs_grad, grad), offsetof(sb_distill, row_stats));
  printf("%d %d %d\n", SB_POLICY_MAX_ACTIONS, SB_POLICY_MAX_TOP, SB_POLICY_MAX_TEACHER);
  return 0;
}
"""


def test_struct_layouts_match_the_header(tmp_path):
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(_LAYOUT)
    subprocess.run(["gcc", "-I", str(ROOT / "include"), "-o", str(exe), str(src)], check=True)
    got = [[int(v) for v in line.split()]
           for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    assert got == [
        [ctypes.sizeof(t) for t in (C.SbLogits, C.SbLogprobs, C.SbLogprobsGrad, C.SbDistill)],
        [C.SbLogits.temperature.offset, C.SbLogprobs.top_logprob.offset, C.SbLogprobsGrad.grad.offset,
         C.SbDistill.row_stats.offset],
        [C.SB_POLICY_MAX_ACTIONS, C.SB_POLICY_MAX_TOP, C.SB_POLICY_MAX_TEACHER]]
