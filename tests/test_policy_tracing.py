"""The policy operators on fake tensors and in traced graphs (CPU; no kernel is launched).

Fake tensors have a device, types and shapes and no memory, so what a tracer
records of a call can be looked at without a GPU.
"""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.fx.experimental.symbolic_shapes import ShapeEnv

from ataraxos_b200.policy import action_logprobs, distill_loss

OPS = torch.ops.stratego_b200


def _operands(lead=(6,), a=20, dtype=torch.float32, grad=False):
    x = torch.empty((*lead, a), dtype=dtype, device="cuda", requires_grad=grad)
    act = torch.empty(lead, dtype=torch.int16, device="cuda")
    ta = torch.empty((*lead, 4), dtype=torch.int64, device="cuda")
    return x, act, ta, torch.empty((*lead, 4), device="cuda")


def _mask(kind, lead, a):
    if kind == "none":
        return None
    if kind == "bits":
        return torch.empty((*lead, (a + 7) // 8), dtype=torch.uint8, device="cuda")
    return torch.empty((a,) if kind == "one" else (*lead, a), dtype=torch.bool, device="cuda")


def _launches(g):
    return [n.target for n in g.graph.nodes if n.op == "call_function" and str(n.target).startswith("stratego_b200.")]


@pytest.mark.parametrize("kind", ["none", "bits", "bool", "one"])
@pytest.mark.parametrize("lead", [(), (6,), (3, 2), (0,)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fake_tensors_give_shapes_and_types(lead, dtype, kind):
    with FakeTensorMode():
        x, act, ta, tl = _operands(lead, dtype=dtype, grad=True)
        mask = _mask(kind, lead, 20)
        r = action_logprobs(x, act, mask, top=3)
        loss = distill_loss(x, ta, tl, mask, tail=True)
        for v, shape, t in ((r.logprob, lead, torch.float32), (r.entropy, lead, torch.float32), (loss, lead, torch.float32),
                            (r.top_logprob, (*lead, 3), torch.float32), (r.top_action, (*lead, 3), torch.int64)):
            assert tuple(v.shape) == tuple(shape) and v.dtype == t and v.device.type == "cuda"
        assert r.logprob.requires_grad and r.top_logprob.requires_grad and not r.top_action.requires_grad
        assert action_logprobs(x.detach()).logprob is None


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_a_trace_records_each_launch(mode, grad):
    """One operator on rows for each kernel, none of their results left as fresh memory."""
    def both(x, act, ta, tl, mask):
        x = x.detach().requires_grad_(grad)
        r = action_logprobs(x, act, mask, top=3)
        return r.logprob, r.top_action, distill_loss(x, ta, tl, mask)

    with FakeTensorMode(shape_env=ShapeEnv()):
        args = (*_operands((3, 2)), _mask("bits", (3, 2), 20))
        g = make_fx(both, tracing_mode=mode)(*args)
    assert list(map(str, _launches(g))) == ["stratego_b200._action_logprobs.default", "stratego_b200._distill_loss.default"]
    assert not [n for n in g.graph.nodes if "empty" in str(n.target)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gradients_of_rows_have_the_logits_shape_and_type(dtype):
    with FakeTensorMode():
        x, act, ta, tl = _operands(dtype=dtype)
        action_logprobs(x, act)  # loads the library
        ent, _, _, best, stats = OPS._action_logprobs(x, act, None, 0, 3, 1.0, True)
        g = OPS._action_logprobs_backward(x, act, None, 0, best, ent, stats, ent, None, None, 1.0)
        loss, stats = OPS._distill_loss(x, ta, tl, None, 0, 1.0, True, True)
        h = OPS._distill_loss_backward(x, ta, tl, None, 0, stats, loss, 1.0, True)
        for v in (g, h):
            assert v.shape == x.shape and v.dtype == dtype and v.is_contiguous()


def test_symbolic_sizes_stay_symbolic():
    def score(x, act, mask):
        return action_logprobs(x, act, mask, top=2).top_logprob

    with FakeTensorMode(shape_env=ShapeEnv()) as fake:
        g = make_fx(score, tracing_mode="symbolic")(_operands((6,))[0], _operands((6,))[1], _mask("bits", (6,), 20))
        with fake:
            x, act, _, _ = _operands((9,))
            assert g(x, act, _mask("bits", (9,), 20)).shape == (9, 2)


def test_rows_on_the_cpu_are_refused():
    with FakeTensorMode():
        action_logprobs(_operands()[0])  # loads the library
    cpu = torch.zeros(6, 20)
    for call in (lambda: OPS._action_logprobs(cpu, None, None, 0, 0, 1.0, False),
                 lambda: OPS._distill_loss(cpu, torch.zeros(6, 4).long(), torch.zeros(6, 4), None, 0, 1.0, False, False)):
        with pytest.raises(NotImplementedError, match="CPU"):
            call()


def test_vmap_is_refused():
    with FakeTensorMode(), pytest.raises(RuntimeError):
        x, act, _, _ = _operands((3, 2))
        torch.func.vmap(lambda x, a: action_logprobs(x, a).logprob)(x, act)
