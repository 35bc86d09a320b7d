"""The policy operators in traced and compiled functions: the same bits as eager calls (no code is generated)."""

from __future__ import annotations

import pytest
import torch
from test_gpu_policy import DEV, _actions, _pack, _rows, _teacher
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def _operands(r=6, a=3000, seed=1, dtype=torch.float32):
    x, ok, g = _rows(r, a, dtype, 0.02, seed=seed)
    ta, tl = _teacher(x, ok, 8, g, True, 1.0)
    return tuple(v.to(DEV) for v in (x, _actions(ok, g), ta, tl, _pack(ok)))


def _values(x, act, ta, tl, bits):
    from ataraxos_b200.policy import action_logprobs, distill_loss

    r = action_logprobs(x, act, bits, top=3)
    return r.logprob, r.entropy, r.top_logprob, r.top_action, distill_loss(x, ta, tl, bits, tail=True)


def _both(x, *rest):
    x = x.detach().requires_grad_()
    v = _values(x, *rest)
    some = v[3] >= 0
    pull = v[0].sum() + 0.5 * v[1].sum() + torch.where(some, v[2], 0.0).sum() + v[4].sum()
    return (*(t.detach() for t in v), torch.autograd.grad(pull, x)[0])


def _same(got, want):
    for p, q in zip(got, want, strict=True):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_traced_graph_launches_the_kernels(dtype):
    """Forward and gradient recorded on one set of operands and run on others, laid out otherwise too."""
    g = make_fx(_both)(*_operands(dtype=dtype))
    names = [str(n.target) for n in g.graph.nodes if str(n.target).startswith("stratego_b200.")]
    assert sorted(names) == sorted(f"stratego_b200.{n}.default" for n in (
        "_action_logprobs", "_distill_loss", "_action_logprobs_backward", "_distill_loss_backward"))
    other = _operands(seed=2, dtype=dtype)
    want = _both(*other)
    _same(g(*other), want)
    spread = tuple(v.t().contiguous().t() if v.dim() == 2 else v.repeat_interleave(2)[::2] for v in other)
    assert spread[0].stride(1) != 1 and spread[1].stride(0) == 2
    _same(g(*spread), want)


def test_a_graph_traced_without_gradients_has_none():
    """Run on logits that require grad, its values are right and its backward pass raises."""
    args = _operands()
    g = make_fx(_values)(*args)
    x = args[0].clone().requires_grad_()
    got = g(x, *args[1:])
    _same(got, _values(*args))
    assert not got[3].requires_grad
    for v in (got[0], got[4]):
        with pytest.raises(RuntimeError, match="not implemented"):
            v.sum().backward()


@pytest.mark.parametrize("public", ["action_logprobs", "distill_loss"])
def test_torch_s_own_checks_of_an_operator(public):
    """Schema, autograd registration, fake tensors and compilation with dynamic sizes, public and on rows."""
    x, act, ta, tl, bits = _operands()
    _values(x, act, ta, tl, bits)
    ops = torch.ops.stratego_b200
    lx = x.clone().requires_grad_()
    if public == "action_logprobs":
        out = ops._action_logprobs(x, act, bits, 2, 3, 1.0, True)
        torch.library.opcheck(ops.action_logprobs.default, (lx, act, bits, 3, 1.0))
        torch.library.opcheck(ops._action_logprobs.default, (x, act, bits, 2, 3, 1.0, True))
        torch.library.opcheck(ops._action_logprobs_backward.default,
                              (x, act, bits, 2, out[3], out[0], out[4], out[0], out[1], out[2], 1.0))
    else:
        loss, stats = ops._distill_loss(x, ta, tl, bits, 2, 1.0, True, True)
        torch.library.opcheck(ops.distill_loss.default, (lx, ta, tl, bits, 1.0, True))
        torch.library.opcheck(ops._distill_loss.default, (x, ta, tl, bits, 2, 1.0, True, True))
        torch.library.opcheck(ops._distill_loss_backward.default, (x, ta, tl, bits, 2, stats, loss, 1.0, True))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_functions_keep_their_results(backend):
    """torch.compile with static and then changing numbers of rows, forward and gradient."""
    torch._dynamo.reset()

    def loss(x, act, ta, tl, bits):
        v = _values(x, act, ta, tl, bits)
        return v[0].sum() + 0.5 * v[1].sum() + v[4].sum(), v[3]

    fast = torch.compile(loss, backend=backend)
    for r in (6, 6, 11, 4):
        x, *rest = _operands(r, seed=r)
        lx, ly = x.clone().requires_grad_(), x.clone().requires_grad_()
        got, top = fast(lx, *rest)
        want, ref = loss(ly, *rest)
        got.backward()
        want.backward()
        _same((got, top, lx.grad), (want, ref, ly.grad))
        with torch.no_grad():
            _same(fast(x, *rest), loss(x, *rest))
    torch._dynamo.reset()


def test_one_graph_once_the_library_is_loaded():
    torch._dynamo.reset()
    args = _operands()
    want = _values(*args)  # an eager call has bound the library
    _same(torch.compile(_values, backend="aot_eager", fullgraph=True)(*args), want)
    torch._dynamo.reset()


@pytest.mark.parametrize("what", ["actions", "alternatives", "statistics", "teacher"])
def test_rows_of_another_type_are_refused(what):
    ops = torch.ops.stratego_b200
    x, act, ta, tl, bits = _operands()
    _values(x, act, ta, tl, bits)
    ent, _, _, best, stats = ops._action_logprobs(x, act, bits, 2, 3, 1.0, True)

    def back(best=best, stats=stats):
        return ops._action_logprobs_backward(x, act, bits, 2, best, ent, stats, ent, None, None, 1.0)

    back()
    calls = {
        "actions": lambda: ops._action_logprobs(x, act.double(), bits, 2, 0, 1.0, False),
        "alternatives": lambda: back(best=best.int()),
        "statistics": lambda: back(stats=stats.half()),
        "teacher": lambda: ops._distill_loss(x, ta.double(), tl, bits, 2, 1.0, True, False),
    }
    with pytest.raises(RuntimeError, match="must be"):
        calls[what]()


@pytest.mark.parametrize("what", ["mask", "actions", "teacher", "gradient"])
def test_rows_that_do_not_belong_together_are_refused(what):
    """What a traced graph calls checks its operands before it launches."""
    ops = torch.ops.stratego_b200
    x, act, ta, tl, bits = _operands()
    _values(x, act, ta, tl, bits)
    loss, stats = ops._distill_loss(x, ta, tl, bits, 2, 1.0, True, True)
    calls = {
        "mask": lambda: ops._action_logprobs(x, act, bits[:5], 2, 0, 1.0, False),
        "actions": lambda: ops._action_logprobs(x, act[:5], bits, 2, 0, 1.0, False),
        "teacher": lambda: ops._distill_loss(x, ta, tl[:, :7], bits, 2, 1.0, True, False),
        "gradient": lambda: ops._distill_loss_backward(x, ta, tl, bits, 2, stats, loss[:5], 1.0, True),
    }
    with pytest.raises(RuntimeError, match="do not match"):
        calls[what]()
