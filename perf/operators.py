"""The policy operators' workloads: their inputs, their plain forms and the
framework's own calls, for timing and comparison.

``logprobs`` is ``ataraxos_b200.policy.action_logprobs`` (log-probabilities of
given actions under the legal softmax, with entropy and top alternatives) and
``distill`` is ``ataraxos_b200.policy.distill_loss`` (divergence from a
teacher's top actions); both with their gradients where ``train`` is set.
``own`` chooses between the plain torch form and the framework's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

NUM_ACTIONS = 10000  # flat moves src * 100 + dst
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
MOVES = 30           # legal moves of a usual position, as prepare() deals them
MOST_CELLS = 65536 * NUM_ACTIONS


def _case(name, op, rows, actions=NUM_ACTIONS, dtype="f32", mask="bits", legal="moves", train=False, temperature=1.0,
          top=0, listed=0, tail=False, pad=0):
    c = {"op": op, "rows": rows, "actions": actions, "dtype": dtype, "mask": mask, "legal": legal, "train": train,
         "temperature": temperature, "top": top, "listed": listed, "tail": tail, "pad": pad}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one position asked for the probability of a move, its five best moves and its entropy (analysis of a game)
        _case("logprobs one position", "logprobs", 1, top=5),
        # the 64 roots of a search batch: the network's 32 best moves as the start of a teacher's list
        _case("logprobs 64 roots", "logprobs", 64, mask="u8", top=32),
        # one ply of 4096 self-play games scored under another network, the step's own u8 masks
        _case("logprobs self-play ply", "logprobs", 4096, dtype="bf16", mask="u8"),
        # a policy-gradient minibatch: 8 plies of 1536 games from the bit-masked trajectory ring, with its gradient
        _case("logprobs minibatch train", "logprobs", 8 * 1536, dtype="bf16", train=True),
        # an unroll of 128 plies of 512 games at once, with its gradient
        _case("logprobs unroll train", "logprobs", 128 * 512, dtype="bf16", train=True, temperature=0.8),
        # a head over the 100 squares (which piece moves), a slice of a wider output, no mask
        _case("logprobs squares train", "logprobs", 200003, actions=100, dtype="f16", mask="none", train=True, pad=3),
        # a whole unmasked head of an odd width with its eight best
        _case("logprobs unmasked odd", "logprobs", 2049, actions=9999, mask="none", top=8),
        # the 64 roots of a search batch distilled at once: the search policy's 32 best moves and the rest as one
        _case("distill 64 roots train", "distill", 64, listed=32, tail=True, train=True),
        # 4096 searched positions with their u8 masks, every listed move's weight renormalised
        _case("distill positions train", "distill", 4096, dtype="bf16", mask="u8", listed=32, train=True),
        # a large replay batch, bit masks
        _case("distill replay train", "distill", 32768, dtype="bf16", listed=32, tail=True, train=True),
        # a teacher network's 16 best of the whole unmasked head, softened
        _case("distill network train", "distill", 4096, dtype="f16", mask="none", listed=16, tail=True, train=True,
              temperature=2.0),
        # the loss alone on held-out rows of a narrower head with half of it legal
        _case("distill held-out", "distill", 5000, actions=2500, legal="half", listed=20, temperature=1.5),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "distill"])
    actions = NUM_ACTIONS if rng.random() < 0.6 else _log_uniform(rng, 12, NUM_ACTIONS)
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    cells = MOST_CELLS // (2 if op == "logprobs" else 4) // (2 if dtype == "f32" else 1)
    mask = rng.choice(["bits", "bits", "u8", "none"])
    legal = "moves" if actions == NUM_ACTIONS and rng.random() < 0.8 else "half"
    train = rng.random() < 0.6
    return _case(None, op, _log_uniform(rng, 1, min(200000, cells // actions)), actions, dtype, mask, legal, train,
                 rng.choice([1.0, 1.0, 0.5 + round(rng.random() * 2, 2)]),
                 rng.choice([0, 1, 5, 8, 20, 32]) if op == "logprobs" else 0,
                 rng.choice([1, 7, 16, 32, 50]) if op == "distill" else 0,
                 rng.random() < 0.5 if op == "distill" else False, rng.choice([0, 0, 1, 3]))


def _legal(case, g, dev):
    """The legal actions as bool [R, A]: about 30 moves of about 12 pieces to
    neighbouring squares and along lines, or half of all; one row in 64 empty
    (a game that is over) when there are at least 64 rows."""
    r, a = case["rows"], case["actions"]
    if case["legal"] == "moves":
        ok = torch.zeros((r, a), dtype=torch.bool, device=dev)
        src = torch.randint(0, 100, (r, 12, 1), generator=g, device=dev)
        step = torch.tensor([1, -1, 10, -10, 2, 20], device=dev)
        dst = src + step
        take = (torch.rand(dst.shape, generator=g, device=dev) < torch.tensor([.6, .6, .6, .6, .15, .15], device=dev))
        take &= (dst >= 0) & (dst < 100)
        flat = torch.where(take, src * 100 + dst, src * 100 + src)  # no piece moves to its own square
        ok.scatter_(1, flat.reshape(r, -1), True)
        ok.view(r, 100, 100).diagonal(dim1=1, dim2=2).fill_(False)
    else:
        ok = torch.empty((r, a), dtype=torch.bool, device=dev)
        for i in range(0, r, 8192):
            ok[i:i + 8192] = torch.rand((min(8192, r - i), a), generator=g, device=dev) < 0.5
    if r >= 64:
        ok[::64] = False
    return ok


def _pack(ok):
    r, a = ok.shape
    w = (a + 7) // 8
    full = torch.zeros((r, w * 8), dtype=torch.uint8, device=ok.device)
    full[:, :a] = ok
    full = full.view(r, w, 8)
    bits = torch.zeros((r, w), dtype=torch.uint8, device=ok.device)
    for j in range(8):
        bits |= full[..., j] << j
    return bits


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r, a, t = case["rows"], case["actions"], case["temperature"]
    wide = torch.empty((r, a + case["pad"]), dtype=DTYPES[case["dtype"]], device=dev)
    for i in range(0, r, 8192):  # a policy head's logits: a few units of spread
        wide[i:i + 8192] = 2.5 * torch.randn((min(8192, r - i), a + case["pad"]), generator=g, device=dev)
    logits = wide[:, case["pad"]:].detach()
    ok = None if case["mask"] == "none" else _legal(case, g, dev)
    s = {"case": case, "logits": logits.requires_grad_(case["train"]), "mask": None}
    n = case["listed"] if case["op"] == "distill" else 1
    acts = torch.full((r, n), -1, dtype=torch.int64, device=dev)
    vals = torch.zeros((r, n), device=dev)
    for i in range(0, r, 8192):  # the teacher is another network: its logits lie near the student's
        x = logits[i:i + 8192].detach().float()
        x = (x + torch.randn(x.shape, generator=g, device=dev)) / (t if case["tail"] else 1.0)
        if ok is not None:
            x = x.masked_fill(~ok[i:i + 8192], float("-inf"))
        if case["tail"]:
            x = torch.log_softmax(x, dim=-1).nan_to_num(nan=float("-inf"))
        if case["op"] == "distill":
            v, k = x.topk(min(n, a), dim=-1)
        else:  # an action sampled from the policy
            k = (x - torch.empty_like(x).exponential_(generator=g).log()).argmax(-1, keepdim=True)
            v = x.gather(1, k)
        live = v > float("-inf")
        acts[i:i + 8192, :k.shape[1]] = torch.where(live, k, -1)
        vals[i:i + 8192, :k.shape[1]] = torch.where(live, v, torch.zeros_like(v))
    scale = 32.0 if case["dtype"] == "f16" else 1.0 / r  # a mean over rows; 16-bit floats of 5 exponent bits scale the loss up
    if case["op"] == "distill":
        s["teacher_actions"], s["teacher_logits"] = acts, vals
        s["g_loss"] = scale * torch.rand((r,), generator=g, device=dev)   # a weight for each position
    else:
        s["actions"] = acts[:, 0].contiguous()
        s["g_logprob"] = scale * torch.randn((r,), generator=g, device=dev)  # minus the advantage
        s["g_entropy"] = torch.full((r,), -0.01 * scale, device=dev)         # an entropy bonus
    if ok is not None:
        s["mask"] = _pack(ok) if case["mask"] == "bits" else ok
    return s


def _rows_legal(s):
    x, m = s["logits"].detach(), s["mask"]
    if m is None:
        return torch.ones(x.shape, dtype=torch.bool, device=x.device)
    if m.dtype == torch.bool:
        return m
    bit = torch.arange(8, device=m.device, dtype=torch.uint8)
    return ((m[:, :, None] >> bit) & 1).bool().view(m.shape[0], -1)[:, :x.shape[1]]


def _softmax_parts(x, ok, t):
    """Whether a row has a legal entry, its shifted logits d = (x - max) / T,
    exp(d) on the legal entries, and their sum Z and log Z (summed and held in
    64 bits: the losses are differences of such logs)."""
    top = x.masked_fill(~ok, float("-inf")).amax(-1, keepdim=True)
    some = top > float("-inf")
    top = torch.where(some, top, torch.zeros_like(top))
    d = ((x - top) / t).masked_fill(~ok, 0.0)
    e = torch.exp(d).masked_fill(~ok, 0.0)
    z = e.sum(-1, keepdim=True, dtype=torch.float64)
    z = torch.where(some, z, torch.ones_like(z))
    return some, d, e, z, torch.log(z)


def _top(x, ok, k):
    """The k largest legal logits by value and then by lower index."""
    bits = x.contiguous().view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 20) + (x.shape[1] - torch.arange(x.shape[1], device=x.device))
    key = key.masked_fill(~ok, -(1 << 62))
    n = min(k, x.shape[1])
    best, idx = key.topk(n, dim=-1)
    idx = torch.where(best > -(1 << 62), idx, -1)
    return torch.nn.functional.pad(idx, (0, k - n), value=-1)


def _plain_logprobs(s):
    c = s["case"]
    x, ok, t = s["logits"].detach().float(), _rows_legal(s), c["temperature"]
    some, d, e, z, logz = _softmax_parts(x, ok, t)
    a = s["actions"]
    has = (a >= 0).unsqueeze(1)
    at = a.clamp(min=0).unsqueeze(1)
    lp = torch.where(has, d.gather(1, at) - logz, torch.zeros_like(logz))
    h = torch.where(some, logz - (e * d).sum(-1, keepdim=True) / z, torch.zeros_like(logz))
    out = {"logprob": lp.squeeze(1).float(), "entropy": h.squeeze(1).float()}
    if c["top"]:
        k = _top(x, ok, c["top"])
        out["top_action"] = k
        out["top_logprob"] = torch.where(k >= 0, d.gather(1, k.clamp(min=0)) - logz, float("-inf")).float()
    if c["train"]:
        gl = torch.where(has, s["g_logprob"].unsqueeze(1), 0.0)
        p = e / z.float()
        grad = -p * (gl + s["g_entropy"].unsqueeze(1) * (d + (h - logz).float()))
        grad.scatter_add_(1, at, gl)
        out["grad"] = (grad / t).to(s["logits"].dtype)
    return out


def _plain_distill(s):
    c = s["case"]
    x, ok, t = s["logits"].detach().float(), _rows_legal(s), c["temperature"]
    some, d, e, z, logz = _softmax_parts(x, ok, t)
    k, v = s["teacher_actions"], s["teacher_logits"].double()
    at = k.clamp(min=0)
    keep = (k >= 0) & ok.gather(1, at)
    if c["tail"]:
        logq = v
    else:
        u = (v / t).masked_fill(~keep, float("-inf"))
        top = u.amax(-1, keepdim=True)
        u = u - torch.where(top > float("-inf"), top, torch.zeros_like(top))
        logq = u - torch.log(torch.exp(u).sum(-1, keepdim=True).clamp(min=1e-30))
    q = torch.exp(logq).masked_fill(~keep, 0.0)
    logq = logq.masked_fill(~keep, 0.0)
    logp = (d.gather(1, at) - logz).masked_fill(~keep, 0.0)
    loss = (q * (logq - logp)).sum(-1, keepdim=True)
    total = q.sum(-1, keepdim=True)
    rest = torch.zeros_like(loss)
    if c["tail"]:
        # unlisted legal actions as one: no action is listed twice here
        free = ok.to(torch.int8).scatter_add_(1, at, -keep.to(torch.int8)) > 0
        pr = e.masked_fill(~free, 0.0).sum(-1, keepdim=True, dtype=torch.float64) / z
        left = pr > 0
        qr = torch.where(left, (1.0 - total).clamp(min=0.0), torch.zeros_like(total))
        term = qr * (torch.log(qr.clamp(min=1e-38)) - torch.log(torch.where(left, pr, torch.ones_like(pr))))
        loss = loss + torch.where(qr > 0, term, torch.zeros_like(term))
        rest = torch.where(left, qr / torch.where(left, pr, torch.ones_like(pr)), torch.zeros_like(pr))
        total = total + qr
    out = {"loss": loss.squeeze(1).float()}
    if c["train"]:
        p = e / z.float()
        grad = p * total.float()
        if c["tail"]:
            grad = torch.where(free, p * (total - rest).float(), grad)
        grad.scatter_add_(1, at, -q.float())
        out["grad"] = (grad * (s["g_loss"].unsqueeze(1) / t)).to(s["logits"].dtype)
    return out


def run(state):
    c = state["case"]
    if not own:
        return _plain_logprobs(state) if c["op"] == "logprobs" else _plain_distill(state)
    from ataraxos_b200.policy import action_logprobs, distill_loss

    x = state["logits"]
    if c["op"] == "logprobs":
        r = action_logprobs(x, state["actions"], state["mask"], top=c["top"], temperature=c["temperature"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if c["top"]:
            out["top_action"], out["top_logprob"] = r.top_action, r.top_logprob
        if c["train"]:
            out["grad"] = torch.autograd.grad([r.logprob, r.entropy], [x], [state["g_logprob"], state["g_entropy"]])[0]
        return out
    loss = distill_loss(x, state["teacher_actions"], state["teacher_logits"], state["mask"],
                        temperature=c["temperature"], tail=c["tail"])
    out = {"loss": loss}
    if c["train"]:
        out["grad"] = torch.autograd.grad([loss], [x], [state["g_loss"]])[0]
    return out


def work(case):
    """Every mask byte and the legal logits are read (a scattered one costs its
    32-byte sector), the outputs and, in training, the whole gradient written."""
    r, a, size = case["rows"], case["actions"], SIZES[case["dtype"]]
    row = a * size
    legal = a
    if case["mask"] != "none":
        legal = MOVES if case["legal"] == "moves" else a / 2
    per = min(row, legal * 32)
    per += {"none": 0, "u8": a, "bits": (a + 7) // 8}[case["mask"]]
    if case["op"] == "logprobs":
        per += 8 + 8 + 12 * case["top"] + (8 if case["train"] else 0)
    else:
        per += 12 * case["listed"] + 4 + (4 if case["train"] else 0)
    if case["train"]:
        per += row
    return {"bytes": r * per, "flops": r * legal * (12 if case["train"] else 6)}


def _exact_rows(case, x, ok, s, i, j):
    """The definition by torch's own log-softmax in 64 bits; gradients by differentiating it."""
    t = case["temperature"]
    x = x.double().requires_grad_(case["train"])
    some = ok.any(-1, keepdim=True)
    z = torch.where(ok | ~some, x / t, torch.full_like(x, float("-inf")))
    logp = torch.log_softmax(z, dim=-1)
    finite = torch.where(ok, logp, torch.zeros_like(logp))
    some = some.squeeze(1)
    if case["op"] == "logprobs":
        a = s["actions"][i:j]
        has = (a >= 0) & some
        lp = torch.where(has, finite.gather(1, a.clamp(min=0)[:, None])[:, 0], torch.zeros((), dtype=x.dtype, device=x.device))
        h = -(torch.where(ok, finite.exp(), torch.zeros_like(finite)) * finite).sum(-1)
        out = {"logprob": lp, "entropy": h}
        if case["top"]:
            out["top_action"] = None
            n = min(case["top"], x.shape[1])
            v = torch.where(ok, logp, torch.full_like(logp, float("-inf"))).detach().sort(-1, descending=True)[0][:, :n]
            out["top_logprob"] = torch.nn.functional.pad(v, (0, case["top"] - n), value=float("-inf"))
        pull = (lp * s["g_logprob"][i:j].double() + h * s["g_entropy"][i:j].double()).sum()
    else:
        k, v = s["teacher_actions"][i:j], s["teacher_logits"][i:j].double()
        at = k.clamp(min=0)
        keep = (k >= 0) & ok.gather(1, at)
        if case["tail"]:
            logq = torch.where(keep, v, torch.full_like(v, float("-inf")))
        else:
            logq = torch.where(keep, v / t, torch.full_like(v, float("-inf")))
            none = ~keep.any(-1, keepdim=True)
            logq = logq - torch.where(none, torch.zeros_like(logq[:, :1]), torch.logsumexp(logq, -1, keepdim=True))
        q = logq.exp()
        gap = torch.where(keep, logq, torch.zeros_like(logq)) - torch.where(keep, finite.gather(1, at), torch.zeros_like(logq))
        loss = (q * gap).sum(-1)
        if case["tail"]:
            free = ok.clone()
            rows, cols = keep.nonzero(as_tuple=True)
            free[rows, at[rows, cols]] = False
            left = free.any(-1)
            qr = torch.where(left, (1 - q.sum(-1)).clamp(min=0), torch.zeros_like(loss))
            lpr = torch.logsumexp(torch.where(free | ~left[:, None], logp, torch.full_like(logp, float("-inf"))), -1)
            on = qr > 0
            loss = loss + torch.where(on, qr * (torch.where(on, qr, torch.ones_like(qr)).log() - torch.where(on, lpr, torch.zeros_like(lpr))),
                                      torch.zeros_like(qr))
        out = {"loss": loss}
        pull = (loss * s["g_loss"][i:j].double()).sum()
    if case["train"]:
        out["grad"] = torch.autograd.grad(pull, x)[0]
    return {n: v if v is None else v.detach() for n, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    step = max(1, (1 << 27) // case["actions"])
    x = s["logits"].detach()
    whole = None
    for i in range(0, case["rows"], step):
        j = min(case["rows"], i + step)
        part = dict(s, logits=x[i:j], mask=None if s["mask"] is None else s["mask"][i:j])
        got = _exact_rows(case, x[i:j], _rows_legal(part), s, i, j)
        if whole is None:
            whole = {n: v if v is None else torch.empty((case["rows"], *v.shape[1:]), dtype=v.dtype, device=v.device)
                     for n, v in got.items()}
        for n, v in got.items():
            if v is not None:
                whole[n][i:j] = v
    return whole
