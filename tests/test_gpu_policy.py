"""The policy operators on a B200 against their definitions in 64 bits.

The oracle is the definition written with torch's float64 log-softmax on the
CPU; gradients are float64 autograd of it.  Tolerances are worst-case rounding
bounds, accumulated beside the oracle's values with u = 2**-24 (half a step of
float32), for a row of n legal actions:
  * d = (x - M) / T: its error is at most 5u|d| (subtraction, product, and the
    constant log2(e) / T of a base-2 exponential);
  * exp(d): relative 4u (2**-22) + 5u|d|;
  * sums of positive terms: relative (n / 32 + 12) u, a lane of 32 adding every
    32nd term and a tree joining the lanes;
  * results in 16 bits: half a step more (finfo.eps / 2 relative, 2**-25
    absolute below float16's normal range).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
INF = float("inf")


def _pack(ok: torch.Tensor) -> torch.Tensor:
    """Bit-packed rows with the bits past the last action set (they must be ignored)."""
    r, a = ok.shape
    full = torch.ones((r, (a + 7) // 8 * 8), dtype=torch.bool)
    full[:, :a] = ok
    return torch.from_numpy(np.packbits(full.numpy(), axis=1, bitorder="little").copy())


def _mask_arg(ok: torch.Tensor, kind: str):
    if kind == "none":
        return None
    if kind == "bits":
        return _pack(ok).to(DEV)
    return ok.to(DEV) if kind == "bool" else (ok.to(torch.uint8) * 7).to(DEV)  # any non-zero byte is legal


def _rows(r, a, dtype, density=0.3, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn((r, a), generator=g)).to(dtype)
    ok = torch.rand((r, a), generator=g) < density
    if r >= 3:
        ok[1] = False                                   # a row without a legal action
        ok[2] = False
        ok[2, int(torch.randint(0, a, (1,), generator=g))] = True  # and one with a single action
    return x, ok, g


class Policy:
    """Softmax of the legal logits in float64 with the bounds above."""

    def __init__(self, x, ok, t):
        x = x.double()
        self.x, self.ok, self.t = x, ok, t
        self.some = (ok & (x > -INF)).any(-1)
        z = torch.where(ok, x / t, torch.full_like(x, -INF))
        self.m = torch.where(self.some, z.masked_fill(~ok, -INF).amax(-1), torch.zeros(()).double())
        self.d = torch.where(ok, z - self.m[:, None], torch.zeros_like(x))
        e = torch.where(ok & self.some[:, None], self.d.exp(), torch.zeros_like(x))
        self.z = torch.where(self.some, e.sum(-1), torch.ones_like(self.m))
        self.logz = self.z.log()
        self.p = e / self.z[:, None]
        self.lp = torch.where(ok & self.some[:, None], self.d - self.logz[:, None], torch.full_like(x, -INF))
        dd = torch.where(self.p > 0, self.d, torch.zeros_like(self.d))
        self.h = torch.where(self.some, self.logz - (self.p * dd).sum(-1), torch.zeros_like(self.m))
        n = ok.sum(-1).double()
        self.sum_rel = U * (n / 32 + 12)
        d1, d2 = (self.p * dd.abs()).sum(-1), (self.p * dd * dd).sum(-1)
        self.z_rel = self.sum_rel + U * (4 + 5 * d1)
        dabs = torch.where(self.p > 0, self.d.abs(), torch.zeros_like(self.d))
        lpabs = torch.where(self.p > 0, self.lp.abs(), torch.zeros_like(self.d))
        self.lp_tol = (self.z_rel + 3 * U * self.logz)[:, None] + U * (5 * dabs + 2 * lpabs) + 1e-30
        self.h_tol = (self.z_rel * (1 + d1) + d1 * self.sum_rel + U * (4 * d1 + 5 * d2) + 3 * U * (self.logz + d1)
                      + 1e-30)
        self.p_rel = self.lp_tol + 4 * U


def _close(got, want, tol, dtype=torch.float32):
    got, want, tol = (v.detach().double().cpu() for v in (got, want, tol))
    if dtype is not torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    tol = tol + 1e-37  # float32's normal range
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}, tolerance {tol[bad][0].item()}")


def _top_of(x, ok, k):
    """Likeliest legal actions by value and then by lower index, zero-probability ones left out."""
    r, a = x.shape
    out = torch.full((r, k), -1, dtype=torch.int64)
    for i in range(r):
        c = [(-float(x[i, j]), j) for j in ok[i].nonzero()[:, 0].tolist() if float(x[i, j]) > -INF]
        for n, (_, j) in enumerate(sorted(c)[:k]):
            out[i, n] = j
    return out


def _check_logprobs(x, ok, act, kind, top, t, logits=None, mask=None, seed=1):
    """Forward and gradient of one call against the oracle; ``logits``: the device tensor to pass for x."""
    from ataraxos_b200.policy import action_logprobs

    r, a = x.shape
    okk = torch.ones_like(ok) if kind == "none" else ok
    P = Policy(x, okk, t)
    lx = (x.to(DEV) if logits is None else logits).detach().requires_grad_()
    out = action_logprobs(lx, act.to(DEV), _mask_arg(ok, kind) if mask is None else mask, top=top, temperature=t)
    inside = (act >= 0) & (act < a)
    at = act.clamp(0, a - 1).long()[:, None]
    legal = inside & okk.gather(1, at)[:, 0]
    want = torch.where(act == -1, torch.zeros_like(P.h), torch.where(legal, P.lp.gather(1, at)[:, 0],
                                                                     torch.full_like(P.h, -INF)))
    _close(out.logprob, want, P.lp_tol.gather(1, at)[:, 0])
    _close(out.entropy, P.h, P.h_tol)
    g = torch.Generator().manual_seed(seed)
    gl, gh, gt = (torch.randn(s, generator=g).double() for s in ((r,), (r,), (r, max(top, 1))))
    grads, outs = [gl, gh], [out.logprob, out.entropy]
    add = torch.zeros_like(P.p)
    add.scatter_add_(1, at, torch.where(legal, gl, torch.zeros_like(gl))[:, None])
    weight = torch.where(legal, gl.abs(), torch.zeros_like(gl))
    if top:
        ref = _top_of(x.double(), okk, top)
        assert torch.equal(out.top_action.cpu(), ref)
        live = ref >= 0
        tl = torch.where(live, P.lp.gather(1, ref.clamp(min=0)), torch.full_like(gt, -INF))
        _close(out.top_logprob, tl, P.lp_tol.gather(1, ref.clamp(min=0)))
        g2 = torch.where(live, gt, torch.zeros_like(gt))
        add.scatter_add_(1, ref.clamp(min=0), g2)
        weight = weight + g2.abs().sum(-1)
        grads.append(gt)
        outs.append(out.top_logprob)
    total = add.sum(-1)
    lp0 = torch.where(P.p > 0, P.lp, torch.zeros_like(P.lp))
    base = -(total + gh * P.h)[:, None] - gh[:, None] * lp0
    base_tol = ((33 * U) * weight + gh.abs() * (P.h_tol + 3 * U * P.h))[:, None] + gh.abs()[:, None] * (
        P.lp_tol + 3 * U * lp0.abs()) + 4 * U * base.abs()
    want_g = (P.p * base + add) / t
    tol_g = (P.p * (base.abs() * P.p_rel + base_tol) * 1.01 + 4 * U * ((P.p * base).abs() + add.abs())
             + 33 * U * weight[:, None] * (add != 0)) / t
    grad = torch.autograd.grad(outs, [lx], [v.float().to(DEV) for v in grads])[0]
    assert grad.dtype == lx.dtype and grad.shape == lx.shape
    want_g = torch.where(okk, want_g, torch.zeros_like(want_g))
    _close(grad, want_g, tol_g, lx.dtype)
    return out, grad


def _actions(ok, g, dtype=torch.int64):
    """A legal action where the row has one, -1 elsewhere."""
    noise = torch.rand(ok.shape, generator=g).masked_fill(~ok, -1.0)
    act = noise.argmax(-1)
    return torch.where(ok.any(-1), act, torch.full_like(act, -1)).to(dtype)


SIZES = [(1, 1), (3, 2), (5, 7), (4, 12), (33, 100), (9, 257), (3, 2047), (4, 9999), (6, 10000), (700, 61), (3, 65536)]


@pytest.mark.parametrize("kind", ["none", "bool", "u8", "bits"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r, a", SIZES)
def test_logprobs_sizes_types_masks(r, a, dtype, kind):
    x, ok, g = _rows(r, a, dtype, seed=r * a)
    act = _actions(torch.ones_like(ok) if kind == "none" else ok, g)
    _check_logprobs(x, ok, act, kind, top=5, t=1.0 if a % 2 else 0.7)


@pytest.mark.parametrize("density", [0.0, 0.003, 0.05, 0.6, 1.0])
@pytest.mark.parametrize("kind", ["u8", "bits"])
@pytest.mark.parametrize("r, a, dtype", [(5, 10000, torch.bfloat16), (3, 10000, torch.float32), (40, 1000, torch.float16)])
def test_logprobs_mask_densities(r, a, dtype, kind, density):
    x, ok, g = _rows(r, a, dtype, density, seed=int(density * 1000))
    if density == 1.0:
        ok[:] = True
    _check_logprobs(x, ok, _actions(ok, g), kind, top=32, t=1.3)


@pytest.mark.parametrize("kind", ["none", "bits", "bool"])
@pytest.mark.parametrize("top", [1, 2, 31, 32])
@pytest.mark.parametrize("order", ["ties", "rising", "falling", "equal"])
def test_top_alternatives_in_every_order(order, top, kind):
    r, a = 6, 1500
    x, ok, g = _rows(r, a, torch.float32, 0.4)
    if order == "ties":
        x = (x * 2).round() / 2
    elif order == "rising":
        x = x.sort(-1)[0]
    elif order == "falling":
        x = x.sort(-1, descending=True)[0]
    else:
        x = torch.full_like(x, 0.25)
    _check_logprobs(x, ok, _actions(torch.ones_like(ok) if kind == "none" else ok, g), kind, top=top, t=1.0)


@pytest.mark.parametrize("index", [torch.int16, torch.int32, torch.int64])
def test_given_actions_that_are_not_legal(index):
    x, ok, g = _rows(8, 10000, torch.bfloat16, 0.01)
    act = _actions(ok, g, index)
    act[3] = -1
    act[4] = -7
    act[5] = 10000
    act[6] = int((~ok[6]).nonzero()[0, 0])
    act[7] = 32767
    out, grad = _check_logprobs(x, ok, act, "bits", top=0, t=1.0)
    assert out.top_action is None and out.top_logprob is None
    assert out.logprob[3].item() == 0.0 and all(out.logprob[i].item() == -INF for i in (4, 5, 6, 7))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["bool", "bits"])
def test_masked_places_may_hold_anything(dtype, kind):
    x, ok, g = _rows(6, 10000, dtype, 0.01, seed=3)
    act = _actions(ok, g)
    dirty = x.clone()
    n = int((~ok).sum())
    bad = torch.tensor([math.nan, INF, -INF, torch.finfo(dtype).max, torch.finfo(dtype).min]).repeat(n // 5 + 1)[:n]
    dirty[~ok] = bad.to(dtype)
    a, ga = _check_logprobs(x, ok, act, kind, top=8, t=1.0)
    b, gb = _check_logprobs(torch.where(ok, x, torch.zeros_like(x)), ok, act, kind, top=8, t=1.0, logits=dirty.to(DEV))
    for p, q in ((a.logprob, b.logprob), (a.entropy, b.entropy), (a.top_action, b.top_action),
                 (a.top_logprob, b.top_logprob), (ga, gb)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("kind", ["none", "bits", "bool"])
def test_lowest_value_and_minus_infinity_as_the_mask(kind):
    """Rows masked inside the logits: the type's lowest value and -inf on legal places have probability 0."""
    x, ok, g = _rows(7, 997, torch.float32, 0.2, seed=9)
    act = _actions(ok, g)
    ok[1, :3] = True
    act[1] = 1
    low = torch.full_like(x, torch.finfo(x.dtype).min)
    low[::2] = -INF
    y = torch.where(ok, x, low)
    legal = ok | (torch.rand(ok.shape, generator=g) < 0.5)
    legal[5] = ok[5]
    if kind == "none":
        legal[:] = True
    _check_logprobs(y, legal, act, kind, top=8, t=1.0)
    # a row that is -inf on every legal place is a row without an action; one of lowest values is uniform
    z = torch.stack([torch.full((997,), -INF), torch.full((997,), torch.finfo(torch.float32).min)])
    all_ok = torch.ones(2, 997, dtype=torch.bool)
    out, grad = _check_logprobs(z, all_ok, torch.tensor([-1, 3]), "none", top=2, t=1.0)
    assert out.top_action.tolist() == [[-1, -1], [0, 1]] and out.entropy[0].item() == 0.0


@pytest.mark.parametrize("kind", ["none", "bits", "bool"])
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_legal_nan_or_infinity_spoils_its_row_alone(bad, kind):
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x, ok, g = _rows(6, 3001, torch.float32, 0.1, seed=4)
    ok[4, 7] = True
    act = _actions(torch.ones_like(ok) if kind == "none" else ok, g)
    dirty = x.clone()
    dirty[4, 7] = bad
    keep = [0, 1, 2, 3, 5]
    res = []
    for v in (x, dirty):
        lx = v.to(DEV).requires_grad_()
        o = action_logprobs(lx, act.to(DEV), _mask_arg(ok, kind), top=3)
        lo = distill_loss(lx, o.top_action, o.top_logprob.detach().nan_to_num(0.0, neginf=-INF), _mask_arg(ok, kind), tail=True)
        gr = torch.autograd.grad([o.logprob, o.entropy, lo], [lx], [torch.ones_like(o.logprob)] * 3)[0]
        res.append((o.logprob.detach(), o.entropy.detach(), o.top_logprob.detach(), lo.detach(), gr))
    for p, q in zip(*res):
        assert torch.equal(p[keep], q[keep])
        assert not p.isnan().any()
    lp, ent, top_lp, lo, gr = res[1]
    assert lp[4].isnan() and ent[4].isnan() and top_lp[4].isnan().all()
    legal = torch.ones(3001, dtype=torch.bool) if kind == "none" else ok[4]
    assert gr[4].cpu()[legal].isnan().all() and (gr[4].cpu()[~legal] == 0).all()


def test_near_certain_action_keeps_its_digits():
    """log p of an action that holds all but 3e-12 of the mass, to float32's relative precision."""
    from ataraxos_b200.policy import action_logprobs

    x = torch.zeros(1, 10000)
    x[0, 77] = 36.0
    out = action_logprobs(x.to(DEV), torch.tensor([77], device=DEV))
    r = 9999 * math.exp(-36.0)
    # relative: exp (4u + 5u * 36), the sum (9999 / 32 + 12) u
    assert abs(out.logprob.item() / -math.log1p(r) - 1) < U * (4 + 180 + 325)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["bits", "bool", "none"])
def test_strides_and_offsets(dtype, kind):
    """Rows that are slices of wider rows, at odd offsets; a transposed tensor; mask rows inside wider rows."""
    for a, pad, off in ((10000, 3, 1), (101, 5, 5), (2500, 8, 8), (63, 1, 1)):
        x, ok, g = _rows(7, a, dtype, 0.2, seed=a)
        wide = torch.full((7, a + pad), 50.0, dtype=dtype, device=DEV)
        wide[:, off:off + a] = x.to(DEV)
        mask = None
        if kind != "none":
            m = _mask_arg(ok, kind)
            wm = torch.full((7, m.shape[1] + 7), 1, dtype=m.dtype, device=DEV)
            wm[:, 3:3 + m.shape[1]] = m
            mask = wm[:, 3:3 + m.shape[1]]
        act = _actions(torch.ones_like(ok) if kind == "none" else ok, g)
        _check_logprobs(x, ok, act, kind, top=4, t=1.0, logits=wide[:, off:off + a], mask=mask)
    x, ok, g = _rows(7, 300, dtype, 0.2, seed=1)
    tr = x.t().contiguous().to(DEV).t()
    assert tr.stride(1) != 1
    _check_logprobs(x, ok, _actions(torch.ones_like(ok) if kind == "none" else ok, g), kind, top=4, t=1.0, logits=tr)


def test_leading_dimensions_and_broadcast():
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x, ok, g = _rows(12, 10000, torch.float32, 0.01)
    act = _actions(ok, g)
    flat = action_logprobs(x.to(DEV), act.to(DEV), ok.to(DEV), top=3)
    for mask in (ok.to(DEV).view(3, 4, 100, 100), _pack(ok).to(DEV).view(3, 4, 1250)):
        o = action_logprobs(x.to(DEV).view(3, 4, 10000), act.to(DEV).view(3, 4), mask, top=3)
        assert o.logprob.shape == (3, 4) and o.top_action.shape == (3, 4, 3)
        assert torch.equal(o.logprob.view(12), flat.logprob) and torch.equal(o.top_action.view(12, 3), flat.top_action)
    one = action_logprobs(x[5].to(DEV), act[5].to(DEV), ok[5].to(DEV), top=3)
    assert one.logprob.shape == () and one.top_action.shape == (3,)
    assert one.logprob.item() == flat.logprob[5].item()
    # one mask for every row, one row of logits for many actions (stride 0)
    m0 = ok[0]
    every = action_logprobs(x.to(DEV).view(3, 4, 10000), None, m0.to(DEV))
    assert every.logprob is None
    want = action_logprobs(x.to(DEV), None, m0.to(DEV).expand(12, 10000).contiguous())
    assert torch.equal(every.entropy.view(12), want.entropy)
    row = x[0].to(DEV).requires_grad_()
    legal = m0.nonzero()[:9, 0].to(DEV)
    many = action_logprobs(row.expand(9, 10000), legal, m0.to(DEV))
    ref = torch.log_softmax(x[0].double().masked_fill(~m0, -INF), -1)[legal.cpu()]
    _close(many.logprob, ref, Policy(x[:1], ok[:1], 1.0).lp_tol[0][legal.cpu()])
    many.logprob.sum().backward()  # the gradients of the nine rows add up
    p = torch.softmax(x[0].double().masked_fill(~m0, -INF), -1)
    hot = torch.zeros(10000, dtype=torch.double)
    hot[legal.cpu()] = 1.0
    _close(row.grad, hot - 9 * p, 9 * p * Policy(x[:1], ok[:1], 1.0).p_rel[0] + 40 * U * (hot + 9 * p))
    loss = distill_loss(x.to(DEV).view(3, 4, 10000), flat.top_action.view(3, 4, 3), flat.top_logprob.view(3, 4, 3),
                        ok.to(DEV).view(3, 4, 100, 100))
    assert loss.shape == (3, 4)


def test_no_rows():
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x = torch.empty((0, 10000), device=DEV, requires_grad=True)
    o = action_logprobs(x, torch.empty(0, dtype=torch.int64, device=DEV), torch.empty((0, 1250), dtype=torch.uint8, device=DEV),
                        top=2)
    lo = distill_loss(x, o.top_action, o.top_logprob.detach())
    assert o.top_action.shape == (0, 2) and lo.shape == (0,)
    (o.logprob.sum() + lo.sum()).backward()
    assert x.grad.shape == (0, 10000)


def test_gradients_of_reductions_and_of_parts():
    """Expanded upstream gradients (sum, mean), strided ones, and outputs that the loss does not use."""
    from ataraxos_b200.policy import action_logprobs

    x, ok, g = _rows(20, 500, torch.float32, 0.3)
    act, m = _actions(ok, g).to(DEV), _pack(ok).to(DEV)
    lx = x.to(DEV).requires_grad_()

    def grad(f):
        return torch.autograd.grad(f(action_logprobs(lx, act, m, top=3)), lx)[0]

    live = torch.isfinite(action_logprobs(lx, act, m, top=3).top_logprob)
    one = grad(lambda o: (o.logprob * torch.ones_like(o.logprob)).sum())
    assert torch.equal(grad(lambda o: o.logprob.sum()), one)
    assert torch.equal(grad(lambda o: o.logprob.mean()), grad(lambda o: (o.logprob * (1 / 20)).sum()))
    ent = grad(lambda o: o.entropy.sum())
    both = grad(lambda o: o.logprob.sum() + o.entropy.sum())
    assert (both - one - ent).abs().max().item() < 16 * U * float(both.abs().max() + one.abs().max() + ent.abs().max())
    wide = torch.randn(20, 2, device=DEV)
    o = action_logprobs(lx, act, m)
    a = torch.autograd.grad(o.logprob, lx, wide[:, 1])[0]
    o = action_logprobs(lx, act, m)
    assert torch.equal(a, torch.autograd.grad(o.logprob, lx, wide[:, 1].contiguous())[0])
    assert grad(lambda o: o.top_logprob[live].sum()).abs().sum().item() > 0


def test_gradient_against_differences():
    """Central differences of the oracle's own forward pass, step h = 1e-5 in 64 bits (error h**2 = 1e-10)."""
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x, ok, g = _rows(5, 40, torch.float32, 0.5)
    act = _actions(ok, g)
    ta, tl = torch.stack([_actions(ok, g) for _ in range(6)], 1), torch.randn((5, 6), generator=g)

    def value(v):
        P = Policy(v, ok, 0.9)
        lp = P.lp.gather(1, act.clamp(min=0)[:, None])[:, 0]
        return (torch.where(act >= 0, lp, torch.zeros_like(lp)).sum() + 0.3 * P.h.sum()
                + 0.7 * _distill_oracle(P, ta, tl, 0.9, False)["loss"].sum())

    lx = x.to(DEV).requires_grad_()
    o = action_logprobs(lx, act.to(DEV), ok.to(DEV), temperature=0.9)
    lo = distill_loss(lx, ta.to(DEV), tl.to(DEV), ok.to(DEV), temperature=0.9)
    (o.logprob.sum() + 0.3 * o.entropy.sum() + 0.7 * lo.sum()).backward()
    h, xd = 1e-5, x.double()
    for i in range(5):
        for j in range(0, 40, 3):
            e = torch.zeros_like(xd)
            e[i, j] = h
            diff = (value(xd + e) - value(xd - e)).item() / (2 * h) if ok[i, j] else 0.0
            assert abs(lx.grad[i, j].item() - diff) < 1e-4 * 0.1 + 1e-5


# -- distillation ---------------------------------------------------------------


def _distill_oracle(P, ta, tl, t, tail):
    """Loss, gradient per unit of upstream gradient, and their bounds."""
    r, k = ta.shape
    a = P.x.shape[1]
    loss, grad = torch.zeros(r).double(), torch.zeros_like(P.p)
    loss_tol, grad_tol = torch.zeros(r).double(), torch.zeros_like(P.p)
    for i in range(r):
        keep = [j for j in range(k) if 0 <= int(ta[i, j]) < a and bool(P.ok[i, int(ta[i, j])]) and float(tl[i, j]) > -INF]
        acts = [int(ta[i, j]) for j in keep]
        v = tl[i, keep].double()
        if tail:
            lq = v
            lq_tol = 3 * U * v.abs() + 4 * U
        elif keep:
            lq = torch.log_softmax(v / t, -1)
            sp = (v / t - (v / t).max()).abs()
            lq_tol = U * (k / 32 + 16 + 5 * float(sp.max())) + U * (5 * sp + 3 * lq.abs() + 3 * math.log(max(k, 2)))
        else:
            continue
        q, q_rel = lq.exp(), lq_tol + 6 * U
        sq = float(q.sum())
        dq = float((q * q_rel).sum()) + U * (k / 32 + 12) * sq
        lp, lpt = P.lp[i, acts], P.lp_tol[i, acts]
        loss[i] = (q * (lq - lp)).sum()
        loss_tol[i] = (q * ((lq - lp).abs() * (q_rel + U * (k / 32 + 16)) + lq_tol + lpt + 2 * U * (lq.abs() + lp.abs()))).sum()
        listed = torch.zeros(a, dtype=torch.bool)
        listed[acts] = True
        free = P.ok[i] & ~listed
        total, share, share_tol = sq, 0.0, 0.0
        if tail:
            pr = float(P.p[i][free].sum())
            if pr > 0:
                sp = float(P.p[i][listed].sum())
                qr = max(0.0, 1.0 - sq)
                lpr_tol = (float(P.z_rel[i]) * 2 + U * (30 + 5 * float(P.d[i][free & (P.p[i] > 0)].abs().min()) + 6 * float(P.logz[i]))
                           + (2 * sp * float(P.p_rel[i][listed & (P.p[i] > 0)].max()) if sp > 0 else 0.0))
                dq += 2 * U
                ratio = abs(math.log(max(qr, dq) / pr)) + 2
                loss[i] += qr * math.log(qr / pr) if qr > 0 else 0.0
                loss_tol[i] += dq * ratio + qr * (lpr_tol + 3 * U * ratio)
                share = qr / pr
                share_tol = dq / pr + share * (lpr_tol + 8 * U)
                total += qr
        wt = torch.zeros(a).double()
        wt_tol = torch.zeros(a).double()
        for n, j in enumerate(acts):
            wt[j] += q[n]
            wt_tol[j] += q[n] * (q_rel[n] + k * U)
        p, prel = P.p[i], P.p_rel[i]
        grad[i] = torch.where(listed, p * total - wt, p * (total - share)) / t
        grad_tol[i] = (p * (total * prel + 2 * dq + 4 * U * total) + wt_tol + 4 * U * wt
                       + torch.where(listed, torch.zeros_like(p), p * (share * prel + share_tol))) / t
        grad[i][~P.ok[i]] = 0
    return {"loss": loss, "grad": grad, "loss_tol": loss_tol, "grad_tol": grad_tol}


def _check_distill(x, ok, ta, tl, kind, t, tail, logits=None):
    from ataraxos_b200.policy import distill_loss

    okk = torch.ones_like(ok) if kind == "none" else ok
    ref = _distill_oracle(Policy(x, okk, t), ta, tl, t, tail)
    lx = (x.to(DEV) if logits is None else logits).detach().requires_grad_()
    loss = distill_loss(lx, ta.to(DEV), tl.to(DEV), _mask_arg(ok, kind), temperature=t, tail=tail)
    _close(loss, ref["loss"], ref["loss_tol"])
    w = torch.linspace(-1, 2, x.shape[0]).double()
    grad = torch.autograd.grad(loss, lx, w.float().to(DEV))[0]
    assert grad.dtype == lx.dtype
    w = w.float().double()[:, None]
    _close(grad, ref["grad"] * w, ref["grad_tol"] * w.abs() + 2 * U * (ref["grad"] * w).abs(), lx.dtype)
    return loss, grad


def _teacher(x, ok, k, g, tail, t, index=torch.int64):
    """A teacher near the student: its k likeliest legal actions, -1 past the last."""
    r, a = x.shape
    y = (x.double() + torch.randn(x.shape, generator=g).double()).masked_fill(~ok, -INF)
    if tail:
        y = torch.log_softmax(y / t, -1).nan_to_num(nan=-INF)
    v, i = y.topk(min(k, a), -1)
    ta = torch.full((r, k), -1, dtype=index)
    tl = torch.zeros(r, k)
    ta[:, :v.shape[1]] = torch.where(v > -INF, i, torch.full_like(i, -1)).to(index)
    tl[:, :v.shape[1]] = torch.where(v > -INF, v, torch.zeros_like(v)).float()
    return ta, tl


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r, a, k", [(1, 1, 1), (3, 2, 2), (5, 7, 9), (20, 100, 8), (9, 257, 33), (4, 9999, 16), (6, 10000, 32),
                                     (300, 61, 5), (3, 10000, 512), (3, 65536, 100)])
def test_distill_sizes_types_masks(r, a, k, dtype, kind, tail):
    x, ok, g = _rows(r, a, dtype, 0.3, seed=r + a + k)
    t = 1.0 if k % 2 else 1.7
    ta, tl = _teacher(x, torch.ones_like(ok) if kind == "none" else ok, k, g, tail, t)
    _check_distill(x, ok, ta, tl, kind, t, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["bool", "bits", "none"])
@pytest.mark.parametrize("index", [torch.int16, torch.int32])
def test_distill_entries_left_out_and_listed_twice(kind, tail, index):
    x, ok, g = _rows(10, 10000, torch.float32, 0.004, seed=5)
    okk = torch.ones_like(ok) if kind == "none" else ok
    ta, tl = _teacher(x, okk, 12, g, tail, 1.0, index)
    ta[3, 4] = ta[3, 0]                                   # twice, with another weight
    ta[4, 1:5] = ta[4, 0]                                 # five times
    if tail:
        tl[4, 1:5] = -6.0
    ta[5, ::2] = -1                                       # padding
    ta[6, 0] = 10000                                      # past the last action
    if kind != "none":
        ta[7, 2] = int((~ok[7]).nonzero()[3, 0])          # not legal
    tl[8, 1:] = -INF                                      # weight zero
    ta[9] = -1                                            # nothing left
    ta[0, 11] = -5
    loss, grad = _check_distill(x, ok, ta, tl, kind, 1.0, tail)
    assert loss[9].item() == 0.0 and not grad[9].any()


@pytest.mark.parametrize("kind", ["bool", "bits", "none"])
def test_distill_tail_when_everything_is_listed(kind):
    """No unlisted legal action: the mass that rounding leaves over is dropped, not set against nothing."""
    x, ok, g = _rows(8, 24, torch.float32, 0.5, seed=6)
    ta, tl = _teacher(x, torch.ones_like(ok) if kind == "none" else ok, 24, g, True, 1.0)
    loss, _ = _check_distill(x, ok, ta, tl, kind, 1.0, True)
    assert torch.isfinite(loss).all()


@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("a", [50, 600, 10000])
@pytest.mark.parametrize("density", [0.05, 0.7])
def test_distill_tail_with_a_near_certain_rest(a, density, kind):
    """The listed actions hold nearly all of the student's mass, and one unlisted action nearly all of what is left."""
    g = torch.Generator().manual_seed(a)
    ok = torch.rand((6, a), generator=g) < density
    ok[:, :4] = True
    x = -12.0 + 0.1 * torch.randn((6, a), generator=g)
    x[:, :3] = torch.tensor([9.0, 8.0, 10.0])
    x[:, 3] = 5.0
    ta = torch.tensor([[0, 1, 2]]).expand(6, 3).contiguous()
    tl = torch.log(torch.tensor([[0.5, 0.2, 0.1]])).expand(6, 3).contiguous()
    _check_distill(x, ok, ta, tl, kind, 1.0, True)


@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("a, density", [(60, 0.5), (700, 0.02), (700, 0.8), (10000, 0.8)])
def test_confident_rows(a, density, kind):
    """One action holds all but a little of the mass: its log-probability, the entropy and the gradient of the rest."""
    g = torch.Generator().manual_seed(a)
    ok = torch.rand((5, a), generator=g) < density
    ok[:, 1] = True
    x = torch.randn((5, a), generator=g)
    x[:, 1] = torch.tensor([14.0, 20.0, 30.0, 60.0, 300.0])
    _check_logprobs(x, ok, torch.ones(5, dtype=torch.int64), kind, top=3, t=1.0)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["none", "bool", "bits"])
@pytest.mark.parametrize("a, k", [(100, 40), (900, 70), (10000, 200), (20000, 65)])
def test_distill_entries_listed_again_far_apart(a, k, kind, tail):
    """The same action in different groups of 32 entries, with different weights; entries left out in between."""
    x, ok, g = _rows(5, a, torch.float32, 0.5 if a < 10000 else 0.02, seed=k)
    ta, tl = _teacher(x, torch.ones_like(ok) if kind == "none" else ok, k, g, tail, 1.3)
    ta[0, 33:37] = ta[0, 0:4]
    ta[3, k - 1] = ta[3, 0]
    ta[3, k // 2] = ta[3, 0]
    ta[4, 5::7] = -1
    if tail:
        tl[:, 32:] -= 1.0                                # the weights stay below 1 in sum
    _check_distill(x, ok, ta, tl, kind, 1.3, tail)


@pytest.mark.parametrize("kind", ["bits", "bool", "none"])
@pytest.mark.parametrize("dtype, density", [(torch.bfloat16, 0.5), (torch.float32, 0.02), (torch.float16, 1.0)])
def test_batches_of_more_than_a_thousand_rows(dtype, density, kind):
    """Where a gradient row is one warp's."""
    x, ok, g = _rows(1300, 2600, dtype, density, seed=21)
    _check_logprobs(x, ok, _actions(torch.ones_like(ok) if kind == "none" else ok, g), kind, top=0, t=1.0)


def test_second_derivatives_are_refused():
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x = torch.randn(4, 30, device=DEV, requires_grad=True)
    act = torch.zeros(4, dtype=torch.int64, device=DEV)
    for y in (action_logprobs(x, act).logprob, action_logprobs(x, act, top=2).entropy,
              distill_loss(x, act[:, None], torch.zeros(4, 1, device=DEV))):
        first = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            first.square().sum().backward()


def test_distill_of_itself_is_zero():
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x, ok, g = _rows(30, 10000, torch.float32, 0.003, seed=8)
    m, lx = _pack(ok).to(DEV), x.to(DEV).requires_grad_()
    P = Policy(x, ok, 1.5)
    for tail in (False, True):
        # 16 of about 30 moves; without the tail both sides would have to be cut off alike
        best = action_logprobs(lx.detach(), None, m, top=16, temperature=1.5)
        if not tail:
            keep = torch.zeros_like(ok)
            keep.scatter_(1, best.top_action.cpu().clamp(min=0), True)
            keep &= ok
        loss = distill_loss(lx, best.top_action, best.top_logprob * (1.0 if tail else 1.5),
                            m if tail else _pack(keep).to(DEV), temperature=1.5, tail=tail)
        assert loss.abs().max().item() < 4 * float(P.lp_tol.max()) + 64 * U
        grad = torch.autograd.grad(loss.sum(), lx)[0]
        assert grad.abs().max().item() < 4 * float(P.lp_tol.max()) + 64 * U


@pytest.mark.parametrize("teacher", [torch.float32, torch.bfloat16, torch.float16])
def test_distill_teacher_types_and_strides(teacher):
    x, ok, g = _rows(9, 1000, torch.bfloat16, 0.1, seed=2)
    ta, tl = _teacher(x, ok, 8, g, False, 2.0)
    tl = tl.to(teacher)
    _check_distill(x, ok, ta, tl, "bits", 2.0, False)
    from ataraxos_b200.policy import distill_loss

    want = distill_loss(x.to(DEV), ta.to(DEV), tl.to(DEV), _pack(ok).to(DEV), temperature=2.0)
    wa, wl = ta.to(DEV).t().contiguous().t(), tl.to(DEV).t().contiguous().t()
    assert torch.equal(distill_loss(x.to(DEV), wa, wl, _pack(ok).to(DEV), temperature=2.0), want)


# -- large offsets, streams, graphs ------------------------------------------------


def test_offsets_past_32_bits():
    """215,000 rows of 10,000 (2.15e9 elements): the last rows are read and written at 64-bit offsets."""
    from ataraxos_b200.policy import action_logprobs, distill_loss

    r, n = 215_000, 5
    x, ok, g = _rows(n, 10000, torch.bfloat16, 0.005, seed=11)
    act = _actions(ok, g)
    big = torch.zeros((r, 10000), dtype=torch.bfloat16, device=DEV)
    big[-n:] = x.to(DEV)
    bits = torch.zeros((r, 1250), dtype=torch.uint8, device=DEV)
    bits[-n:] = _pack(ok).to(DEV)
    acts = torch.full((r,), -1, dtype=torch.int64, device=DEV)
    acts[-n:] = act.to(DEV)
    lx = big.requires_grad_()
    o = action_logprobs(lx, acts, bits, top=2)
    lo = distill_loss(lx, o.top_action, o.top_logprob.detach(), bits, tail=True)
    P = Policy(x, ok, 1.0)
    _close(o.logprob[-n:], torch.where(act >= 0, P.lp.gather(1, act.clamp(min=0)[:, None])[:, 0], torch.zeros_like(P.h)),
           P.lp_tol.gather(1, act.clamp(min=0)[:, None])[:, 0])
    assert not o.logprob[:-n].any() and not lo[:-n].any()
    grad = torch.autograd.grad(o.logprob.sum(), lx)[0]
    hot = torch.zeros_like(P.p).scatter_(1, act.clamp(min=0)[:, None], (act >= 0).double()[:, None])
    want = hot - P.p * (act >= 0).double()[:, None]
    _close(grad[-n:], want, P.p * P.p_rel + 8 * U, torch.bfloat16)
    for i in range(0, r - n, 20_000):
        assert not grad[i:min(i + 20_000, r - n)].any()


def test_many_small_rows():
    """More rows than a grid of one dimension is given at once, each a row of its own."""
    from ataraxos_b200.policy import action_logprobs

    r = 1_300_001
    x = torch.randn((r, 3), device=DEV)
    act = torch.randint(0, 3, (r,), device=DEV)
    lx = x.clone().requires_grad_()
    o = action_logprobs(lx, act, top=3)
    ref = torch.log_softmax(x.double(), -1)
    assert (o.logprob.double() - ref.gather(1, act[:, None])[:, 0]).abs().max().item() < 64 * U * 4
    assert torch.equal(o.top_action, x.argsort(-1, descending=True))
    o.logprob.sum().backward()
    want = torch.nn.functional.one_hot(act, 3).double() - ref.exp()
    assert (lx.grad.double() - want).abs().max().item() < 64 * U


def test_side_stream_and_graph_replay():
    """Forward and backward captured together and replayed on new values, beside a living eager graph of the same
    logits (of its own leaf: torch ties a leaf's gradient to the stream that first used it, and ends a capture that
    meets such a leaf's older graph)."""
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x, ok, g = _rows(16, 10000, torch.float32, 0.01, seed=12)
    act, bits = _actions(ok, g).to(DEV), _pack(ok).to(DEV)
    leaf = x.to(DEV).requires_grad_()
    one = torch.ones(16, device=DEV)

    def both(v):
        o = action_logprobs(v, act, bits, top=4)
        lo = distill_loss(v, o.top_action, o.top_logprob.detach() * 0.9, bits)
        gr = torch.autograd.grad([o.logprob, o.entropy, lo], [v], [one, one, one])[0]
        return o.logprob.detach(), o.entropy.detach(), o.top_action, lo.detach(), gr

    eager = action_logprobs(leaf.detach().requires_grad_(), act, bits)  # its graph stays alive over the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both(leaf.detach().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    want = [v.clone() for v in both(leaf.detach().requires_grad_())]
    for p, q in zip(first, want):
        assert torch.equal(p, q)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    other = (x * 0.5).to(DEV).requires_grad_()
    with torch.cuda.graph(graph):
        outs = both(leaf)
    with torch.cuda.graph(graph2):  # two graphs, no workspace between them
        outs2 = both(other)
    want2 = [v.clone() for v in both(other.detach().requires_grad_())]
    graph.replay()
    graph2.replay()
    torch.cuda.synchronize()
    for p, q in zip((*outs, *outs2), (*want, *want2)):
        assert torch.equal(p, q)
    with torch.no_grad():
        leaf.copy_((x * 1.25).to(DEV))
    graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(outs, both(leaf.detach().requires_grad_())):
        assert torch.equal(p, q)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        eager.logprob.sum().backward()  # autograd saw the leaf change


def test_results_do_not_depend_on_the_batch():
    """A row's bits are the same alone, in a small batch and in a large one, and from run to run."""
    from ataraxos_b200.policy import action_logprobs, distill_loss

    for a, dens in ((10000, 0.004), (100, 0.5)):
        x, ok, g = _rows(3000, a, torch.bfloat16, dens, seed=13)
        act, bits, lx = _actions(ok, g).to(DEV), _pack(ok).to(DEV), x.to(DEV)
        ta, tl = _teacher(x, ok, 8, g, True, 1.0)
        ta, tl = ta.to(DEV), tl.to(DEV)

        def run(i, j):
            v = lx[i:j].detach().requires_grad_()
            o = action_logprobs(v, act[i:j], bits[i:j], top=4)
            lo = distill_loss(v, ta[i:j], tl[i:j], bits[i:j], tail=True)
            gr = torch.autograd.grad(o.logprob.sum() + lo.sum(), v)[0]
            return [o.logprob, o.entropy, o.top_action, o.top_logprob, lo, gr]

        whole, again = run(0, 3000), run(0, 3000)
        for p, q in zip(whole, again):
            assert torch.equal(p, q)
        for i, j in ((0, 1), (17, 18), (5, 69), (2900, 3000)):
            tol = 0  # the same arithmetic for every batch size
            for p, q in zip(whole, run(i, j)):
                assert torch.equal(p[i:j], q), tol


# -- with the simulator -------------------------------------------------------------


def test_step_logprob_is_the_operators():
    """The step kernel samples with these log-probabilities; they agree with its own."""
    from ataraxos_b200 import StrategoRolloutBuffer
    from ataraxos_b200.policy import action_logprobs

    n = 256
    b = StrategoRolloutBuffer(n, 0, seed=3, pool_size=512)
    b.reset_all_from_pool()
    for t in range(40):
        logits = torch.randn((n, 10000), device=DEV)
        bits = b.compute_legal_action_mask_bits()
        u8 = b.compute_legal_action_mask()
        out = b.step(None, policy="gumbel", logits=logits)
        r = action_logprobs(logits, out.action, bits, top=4)
        assert (r.logprob - out.logprob).abs().max().item() < 2e-5
        r8 = action_logprobs(logits, out.action, u8, top=4)
        assert torch.equal(r.top_action, r8.top_action)
        assert (r.logprob - r8.logprob).abs().max().item() < 2e-6
        assert u8.view(n, -1).gather(1, r.top_action.clamp(min=0)).view(n, 4)[r.top_action >= 0].all()


@pytest.mark.parametrize("mask_format", ["bits", "u8"])
def test_policy_gradient_step_from_the_ring(mask_format):
    """A ring's recorded games scored under a network's logits, slot by slot and all at once, with the gradient."""
    from ataraxos_b200 import StrategoRolloutBuffer
    from ataraxos_b200.policy import action_logprobs
    from ataraxos_b200.trajectory import TrajectoryBuffer

    n, T = 24, 6
    b = StrategoRolloutBuffer(n, 0, seed=5, pool_size=64, max_game_length=4)
    b.reset_all_from_pool()
    ring = TrajectoryBuffer(b, T, obs_dtype=None, mask_format=mask_format)
    ring.prime()
    ring.rollout(T - 1, auto_reset=False)
    assert (ring.action == -1).any() and (ring.action >= 0).any()
    logits = torch.randn((T, n, 10000), device=DEV).bfloat16().requires_grad_()
    r = ring.action_logprobs(logits, top=2)
    assert r.logprob.shape == (T, n) and r.top_logprob.shape == (T, n, 2)
    assert (r.logprob[ring.action < 0] == 0).all() and (r.logprob[ring.action >= 0] < 0).all()
    one = ring.action_logprobs(logits[2:4], slice(2, 4))
    assert torch.equal(one.logprob, r.logprob[2:4])
    adv = torch.randn((T, n), device=DEV)
    (-(adv * r.logprob).mean() - 0.01 * r.entropy.mean()).backward()
    ok = torch.from_numpy(np.unpackbits(ring.mask.cpu().numpy(), axis=-1, bitorder="little")).bool() \
        if mask_format == "bits" else ring.mask.cpu().bool().flatten(-2)
    ok, x = ok.view(T * n, 10000), logits.detach().cpu().view(T * n, 10000)
    ref = action_logprobs(logits.detach().view(T * n, 10000), ring.action.view(-1), ok.to(DEV))
    assert torch.equal(ref.logprob.view(T, n), r.logprob.detach()) or \
        (ref.logprob.view(T, n) - r.logprob).abs().max().item() < 2e-6
    P = Policy(x, ok, 1.0)
    act = ring.action.cpu().long().view(-1)
    w = -(adv.cpu().double() / (T * n)).view(-1) * (act >= 0)
    hot = torch.zeros_like(P.p).scatter_(1, act.clamp(min=0)[:, None], w[:, None])
    gh = -0.01 / (T * n)
    want = hot - P.p * (w[:, None] + gh * (torch.where(P.p > 0, P.lp, torch.zeros_like(P.lp)) + P.h[:, None]))
    _close(logits.grad.view(T * n, 10000), want, 2e-6 * (hot.abs() + P.p * w.abs()[:, None] + abs(gh)), torch.bfloat16)


def test_search_teaches_the_network():
    """Search policy -> its likeliest moves -> distillation at the roots, gradients from both operators."""
    from ataraxos_b200 import StrategoRolloutBuffer
    from ataraxos_b200.policy import action_logprobs, distill_loss
    from ataraxos_b200.search import BatchedSearch

    n = 4
    b = StrategoRolloutBuffer(n, 0, seed=9, pool_size=64)
    b.reset_all_from_pool()
    for _ in range(30):
        b.step(None)
    table = torch.randn(10000, device=DEV)

    def net(info):
        return torch.randn((info.shape[0], 3), device=DEV), table.expand(info.shape[0], 10000)

    res = BatchedSearch(net, n_rollouts=60, depth=3).search(b)
    ta, tl = res.teacher(16)
    pol = res.policy.cpu()
    assert torch.equal(ta.cpu(), _top_of(pol.log().float().double(), pol > 0, 16))
    mask = b.compute_legal_action_mask_bits()
    logits = table.expand(n, 10000).clone().requires_grad_()
    loss = distill_loss(logits, ta, tl, mask, tail=True)
    ok = torch.from_numpy(np.unpackbits(mask.cpu().numpy(), axis=1, bitorder="little")).bool()
    ref = _distill_oracle(Policy(logits.detach().cpu(), ok, 1.0), ta.cpu(), tl.cpu(), 1.0, True)
    _close(loss, ref["loss"], ref["loss_tol"])
    loss.sum().backward()
    _close(logits.grad, ref["grad"], ref["grad_tol"])
    # a step against the gradient brings the student nearer
    with torch.no_grad():
        moved = logits - 0.1 * logits.grad
    best = action_logprobs(moved, ta[:, 0], mask)
    assert torch.isfinite(best.logprob).all()
    assert (distill_loss(moved, ta, tl, mask, tail=True) <= loss).all()
