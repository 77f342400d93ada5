"""The language-model operators as they are measured: token log probabilities, distillation from a
teacher's top logits, and the gated linear recurrence, each forward, backward and in the small
form a decoding step calls.

`run` computes them in plain torch operations, or, where `own` is true, through
`harp_amd.operators` on a device handle that queues on torch's stream.
"""

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -1
_handles = {}


def listed():
    return [
        # one decoding step of a small serving batch: the drawn tokens' scores and the 20 best alternatives
        {"name": "score, decoding step", "op": "score", "rows": 8, "vocab": 32000, "dtype": "bf16", "top": 20, "masked": 0, "scale": 1.0},
        # the tokens of one long prompt under a vocabulary of odd size whose last entries are never produced
        {"name": "score, prompt, odd vocab", "op": "score", "rows": 1021, "vocab": 50257, "dtype": "f16", "top": 5, "masked": 17, "scale": 0.7},
        # log probabilities and entropies of a batch of sampled answers
        {"name": "score, batch of answers", "op": "score", "rows": 8192, "vocab": 32000, "dtype": "f32", "top": 0, "masked": 0, "scale": 1.0},
        # gradient of a policy's objective (log probability and entropy) with respect to the logits
        {"name": "score gradient, batch", "op": "score_grad", "rows": 8192, "vocab": 65536, "dtype": "bf16", "masked": 0, "scale": 1.0},
        # distillation of a small student on a small batch, f32 as the front end computes
        {"name": "distill, small batch", "op": "distill", "rows": 64, "vocab": 8192, "dtype": "f32", "teacher": 16, "padded": False, "temperature": 2.0},
        # a large training batch: loss and gradient in one call
        {"name": "distill, training batch", "op": "distill", "rows": 8192, "vocab": 128000, "dtype": "bf16", "teacher": 64, "padded": True, "temperature": 1.0},
        # the gradient alone, as an autograd engine calls it after the loss
        {"name": "distill gradient, odd vocab", "op": "distill_grad", "rows": 2047, "vocab": 50257, "dtype": "f32", "teacher": 20, "padded": True, "temperature": 1.5},
        # one token for every sequence of a serving batch
        {"name": "scan, one token", "op": "scan", "batch": 64, "time": 1, "width": 2048, "dtype": "bf16", "log_gate": True, "ragged": False, "state": True},
        # a layer's forward pass in training
        {"name": "scan, training layer", "op": "scan", "batch": 8, "time": 4096, "width": 2048, "dtype": "bf16", "log_gate": True, "ragged": False, "state": False},
        # its backward pass
        {"name": "scan gradient, training", "op": "scan_grad", "batch": 8, "time": 4096, "width": 2048, "dtype": "bf16", "log_gate": True, "ragged": False, "state": False},
        # one long document, few channels: the sequence itself has to be split
        {"name": "scan, long document", "op": "scan", "batch": 1, "time": 131072, "width": 512, "dtype": "f32", "log_gate": False, "ragged": False, "state": True},
        # the backward pass of a padded batch of uneven sequences with an odd number of channels
        {"name": "scan gradient, padded, odd", "op": "scan_grad", "batch": 13, "time": 1999, "width": 717, "dtype": "f16", "log_gate": False, "ragged": True, "state": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "score", "score_grad", "distill", "distill_grad", "scan", "scan", "scan_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op.startswith("scan"):
        width = _log_uniform(rng, 8, 4096)
        time = 1 if op == "scan" and rng.random() < 0.2 else _log_uniform(rng, 2, 131072)
        batch = _log_uniform(rng, 1, 256)
        while batch * time * width > 60_000_000:
            batch, time = max(1, batch // 2), time if batch > 1 else time // 2
        return {"op": op, "batch": batch, "time": time, "width": width, "dtype": dtype, "log_gate": rng.random() < 0.5,
                "ragged": rng.random() < 0.4, "state": rng.random() < 0.5}
    vocab = _log_uniform(rng, 500, 150_000)
    if rng.random() < 0.5:
        vocab += -vocab % 64
    rows = _log_uniform(rng, 1, 8192)
    while rows * vocab > (200_000_000 if op == "score" else 500_000_000):
        rows //= 2
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype}
    if op == "score":
        return {**case, "top": rng.choice([0, 1, 5, 20, 32]), "masked": rng.choice([0, 0, rng.randrange(1, 200)]), "scale": rng.choice([1.0, 0.7, 1.25])}
    if op == "score_grad":
        return {**case, "masked": rng.choice([0, 0, rng.randrange(1, 200)]), "scale": rng.choice([1.0, 0.7, 1.25])}
    return {**case, "teacher": _log_uniform(rng, 1, 128), "padded": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.5, 2.0, 4.0])}


def _lengths(case):
    """Steps of each sequence: all of them, or uneven ones from none to all in a padded batch."""
    b, t = case["batch"], case["time"]
    return [t - (i * 7919) % (t + 1) for i in range(b)] if case["ragged"] else [t] * b


def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"].startswith("scan"):
        steps = sum(_lengths(case)) * case["width"]
        ends = 4 * case["batch"] * case["width"] * (2 if case["state"] else 1)
        if case["op"] == "scan":
            return {"bytes": 3 * s * steps + ends, "flops": 2 * steps}
        return {"bytes": 5 * s * steps + ends, "flops": 3 * steps}
    n, v = case["rows"], case["vocab"]
    if case["op"] == "score":
        return {"bytes": s * n * v + n * (8 + 12 + 8 * case["top"]), "flops": 5 * n * v}
    if case["op"] == "score_grad":
        return {"bytes": 2 * s * n * v + n * (8 + 16), "flops": 6 * n * v}
    k = case["teacher"]
    if case["op"] == "distill":
        return {"bytes": 2 * s * n * v + n * (8 * k + 12), "flops": 6 * n * v}
    return {"bytes": 2 * s * n * v + n * (8 * k + 8), "flops": 4 * n * v}


# ---- inputs -----------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"].startswith("scan"):
        b, t, d = case["batch"], case["time"], case["width"]
        # decays between 0.6 and 0.999, as gates of a trained layer spread
        log_a = -torch.exp(normal(b, t, d) * 1.2 - 3.0).clamp_(1e-3, 0.5)
        st = {"case": case, "gate": (log_a if case["log_gate"] else log_a.exp()).to(dt),
              "lengths": torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None,
              "state": normal(b, d) if case["state"] else None}
        del log_a
        if case["op"] == "scan":
            st["x"] = normal(b, t, d, dtype=dt)
            st["out"] = torch.zeros(b, t, d, device="cuda", dtype=dt)
            st["final"] = torch.empty(b, d, device="cuda")
            return st
        # the states that the forward pass left are of the size that its sums reach
        st["h"] = (normal(b, t, d) * 2.5).to(dt)
        st["grad_h"] = normal(b, t, d, dtype=dt)
        st["grad_gate"] = torch.zeros(b, t, d, device="cuda", dtype=dt)
        st["grad_x"] = torch.zeros(b, t, d, device="cuda", dtype=dt)
        st["grad_state"] = torch.empty(b, d, device="cuda") if case["state"] else None
        return st
    n, v = case["rows"], case["vocab"]
    logits = normal(n, v, dtype=dt).mul_(2.5)
    st = {"case": case, "logits": logits}
    if case["op"].startswith("score"):
        if case["masked"]:
            logits[:, v - case["masked"]:] = -math.inf
        live = v - case["masked"]
        st["targets"] = torch.randint(0, live, (n,), generator=gen, device="cuda")
        # the target is among the likelier tokens, as a sampled one is
        logits.scatter_add_(1, st["targets"][:, None], normal(n, 1).abs().mul_(4.0).to(dt))
        if n > 8:
            st["targets"][3::11] = IGNORE
        if case["op"] == "score":
            k = case["top"]
            st["logp"], st["entropy"] = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
            st["norm"] = torch.empty(n, 2, device="cuda")
            st["top_logp"] = torch.empty(n, k, device="cuda") if k else None
            st["top_ids"] = torch.empty(n, k, device="cuda", dtype=torch.int32) if k else None
            return st
        m = logits.amax(1, keepdim=True)
        lp = (logits.double() if n * v <= 20_000_000 else logits.float()).sub(m).mul_(case["scale"])
        log_s = torch.logsumexp(lp, 1, keepdim=True)
        st["norm"] = torch.cat([m.float(), log_s.float()], 1)
        lp -= log_s
        st["entropy"] = -(lp.exp() * lp.clamp_(min=-1e4)).sum(1).float()
        st["grad_logp"], st["grad_entropy"] = normal(n), normal(n).mul_(0.01)
        st["grad"] = torch.empty_like(logits)
        return st
    k = case["teacher"]
    st["teacher"] = torch.sort(normal(n, k).mul_(3.0), dim=1, descending=True).values
    # a teacher's tokens are all different: an arithmetic progression from a place of the row's own
    step = max(1, v // (k + 1))
    first = torch.randint(0, max(1, v - step * (k - 1)), (n, 1), generator=gen, device="cuda") if k <= v else torch.zeros(n, 1, device="cuda", dtype=torch.int64)
    st["ids"] = ((first + step * torch.arange(k, device="cuda")[None, :]) % v).to(torch.int32)
    logits.scatter_add_(1, st["ids"].long(), st["teacher"].clamp(min=0).to(dt))
    if case["padded"]:
        st["ids"][torch.arange(k, device="cuda")[None, :] >= torch.randint(0, k + 1, (n, 1), generator=gen, device="cuda")] = -1
    st["weight"] = torch.rand(n, generator=gen, device="cuda").add_(0.5)
    st["grad"] = torch.empty_like(logits)
    if case["op"] == "distill":
        st["loss"], st["norm"] = torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda")
    else:
        m = logits.amax(1, keepdim=True)
        u = (logits.double() if n * v <= 20_000_000 else logits.float()).sub(m).div_(case["temperature"])
        st["norm"] = torch.cat([m.float(), torch.logsumexp(u, 1, keepdim=True).float()], 1)
    return st


# ---- one pass ---------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return {"score": _score, "score_grad": _score_grad, "distill": _distill, "distill_grad": _distill_grad, "scan": _scan, "scan_grad": _scan_grad}[state["case"]["op"]](state)


def _device(x):
    """The device handle of the stream that torch works on now, on the GPU of `x`.  (The stream as a number: as an object of
    torch's it takes 2.7 us, a third of the smallest calls.)"""
    index = x.get_device()
    stream = torch._C._cuda_getCurrentRawStream(index)
    handle = _handles.get((index, stream))
    if handle is None:
        from harp_amd.backend import HipDevice
        handle = _handles[index, stream] = HipDevice(index, stream=stream)
    return handle


def _own(st):
    from harp_amd import operators as ops
    case = st["case"]
    dev = _device(st["gate"] if "gate" in st else st["logits"])
    op = case["op"]
    if op == "score":
        out = ops.Logprobs(st["logp"], st["entropy"], st["norm"], st["top_logp"], st["top_ids"])
        ops.token_logprobs(dev, st["logits"], st["targets"], top=case["top"], scale=case["scale"], ignore_index=IGNORE, out=out)
        return {"logp": out.logp, "entropy": out.entropy, "norm": out.norm, "top_logp": out.top_logp, "top_ids": out.top_ids}
    if op == "score_grad":
        ops.token_logprobs_backward(dev, st["logits"], st["targets"], st["norm"], st["entropy"], st["grad_logp"], st["grad_entropy"],
                                    scale=case["scale"], ignore_index=IGNORE, out=st["grad"])
        return {"grad": st["grad"]}
    if op == "distill":
        out = ops.Distilled(st["loss"], st["norm"], st["grad"])
        ops.distill_loss(dev, st["logits"], st["teacher"], st["ids"], temperature=case["temperature"], row_weight=st["weight"], grad=True, out=out)
        return {"loss": out.loss, "norm": out.norm, "grad": out.grad}
    if op == "distill_grad":
        ops.distill_loss_backward(dev, st["logits"], st["teacher"], st["ids"], st["norm"], st["weight"], temperature=case["temperature"], out=st["grad"])
        return {"grad": st["grad"]}
    if op == "scan":
        ops.gated_scan(dev, st["gate"], st["x"], state=st["state"], lengths=st["lengths"], log_gate=case["log_gate"], out=st["out"], final=st["final"])
        return {"h": st["out"], "final": st["final"]}
    ops.gated_scan_backward(dev, st["gate"], st["h"], st["grad_h"], state=st["state"], lengths=st["lengths"], log_gate=case["log_gate"],
                            out=ops.ScanGrads(st["grad_gate"], st["grad_x"], st["grad_state"]))
    return {"grad_gate": st["grad_gate"], "grad_x": st["grad_x"], "grad_state": st["grad_state"]}


def _softmax_parts(z, scale):
    """Row maximum m, scale (z - m), its exponentials, and the logarithm of their sum."""
    m = z.amax(1, keepdim=True)
    d = (z - m) * scale
    e = torch.exp(d)
    return m, d, e, torch.log(e.sum(1, keepdim=True))


def _score(st):
    case = st["case"]
    z = st["logits"].float()
    m, d, e, log_s = _softmax_parts(z, case["scale"])
    entropy = log_s - (torch.where(e > 0, d, 0.0) * e).sum(1, keepdim=True) / torch.exp(log_s)
    t = st["targets"]
    logp = torch.where(t != IGNORE, d.gather(1, t.clamp(min=0)[:, None])[:, 0] - log_s[:, 0], 0.0)
    top_logp = top_ids = None
    if case["top"]:
        # one whole number for each entry, its value above its place counted from the end: equal values go to the lowest place
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -2147483648 - bits, bits)
        place = torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
        best = (key * 4294967296 + place).topk(case["top"], 1).indices
        top_ids = best.int()
        top_logp = d.gather(1, best) - log_s
    return {"logp": logp, "entropy": entropy[:, 0], "norm": torch.cat([m, log_s], 1), "top_logp": top_logp, "top_ids": top_ids}


def _log_probabilities(st, scale):
    m, log_s = st["norm"][:, :1], st["norm"][:, 1:]
    return (st["logits"].float() - m) * scale - log_s


def _score_grad(st):
    case = st["case"]
    lp = _log_probabilities(st, case["scale"])
    p = torch.exp(lp)
    t = st["targets"]
    g = torch.where(t != IGNORE, st["grad_logp"], 0.0)
    grad = -p * (g[:, None] + st["grad_entropy"][:, None] * (torch.where(p > 0, lp, 0.0) + st["entropy"][:, None]))
    grad.scatter_add_(1, t.clamp(min=0)[:, None], g[:, None])
    return {"grad": (grad * case["scale"]).to(st["logits"].dtype)}


def _teacher(st):
    """The teacher's probabilities over the tokens it names (0 where it names none), and their logarithms."""
    named = st["ids"] >= 0
    v = torch.where(named, st["teacher"].float() / st["case"]["temperature"], -math.inf)
    m = v.amax(1, keepdim=True)
    v = v - torch.where(m == -math.inf, 0.0, m)
    s = torch.exp(v).sum(1, keepdim=True)
    q = torch.where(named, torch.exp(v) / s, 0.0)
    return q, torch.where(named, v - torch.log(s), 0.0)


def _distill(st):
    case = st["case"]
    temp, dt = case["temperature"], st["logits"].dtype
    m, d, e, log_s = _softmax_parts(st["logits"].float(), 1.0 / temp)
    q, log_q = _teacher(st)
    ids = st["ids"].clamp(min=0).long()
    log_p = d.gather(1, ids) - log_s
    loss = temp * temp * (torch.where(q > 0, log_q - log_p, 0.0) * q).sum(1)
    grad = e.mul_(q.sum(1, keepdim=True) / torch.exp(log_s)).scatter_add_(1, ids, -q)
    return {"loss": loss, "norm": torch.cat([m, log_s], 1), "grad": (grad.mul_(temp * st["weight"][:, None])).to(dt)}


def _distill_grad(st):
    temp, dt = st["case"]["temperature"], st["logits"].dtype
    p = torch.exp(_log_probabilities(st, 1.0 / temp))
    q, _ = _teacher(st)
    grad = p.mul_(q.sum(1, keepdim=True)).scatter_add_(1, st["ids"].clamp(min=0).long(), -q)
    return {"grad": grad.mul_(temp * st["weight"][:, None]).to(dt)}


def _gates(st):
    a = st["gate"].float()
    return torch.exp(a) if st["case"]["log_gate"] else a


def _valid(st, like):
    """Which steps a sequence has, as a mask over [batch, time, 1]; None where all have all."""
    if st["lengths"] is None:
        return None
    return (torch.arange(like.shape[1], device=like.device)[None, :] < st["lengths"][:, None])[:, :, None]


def _recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t along dimension 1, h_(-1) = 0, by doubling the reach of each step's sum."""
    reach = 1
    while reach < a.shape[1]:
        b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _scan(st):
    a, x = _gates(st), st["x"].float()
    ok = _valid(st, x)
    if st["state"] is not None:
        x = torch.cat([x[:, :1] + a[:, :1] * st["state"][:, None], x[:, 1:]], 1)
    h = _recurrence(a, x)
    if ok is None:
        return {"h": h.to(st["x"].dtype), "final": h[:, -1]}
    last = (st["lengths"].long() - 1).clamp(min=0)[:, None, None].expand(-1, 1, h.shape[2])
    start = torch.zeros_like(h[:, 0]) if st["state"] is None else st["state"]
    final = torch.where(st["lengths"][:, None] > 0, h.gather(1, last)[:, 0], start)
    return {"h": torch.where(ok, h, 0.0).to(st["x"].dtype), "final": final}


def _scan_grad(st):
    a, g = _gates(st), st["grad_h"].float()
    dt = st["grad_h"].dtype
    ok = _valid(st, g)
    if ok is not None:
        a, g = torch.where(ok, a, 0.0), torch.where(ok, g, 0.0)
    # the gate that carries a gradient from step t + 1 to step t, both in reverse order
    carry = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    lam = _recurrence(carry.flip(1), g.flip(1)).flip(1)
    start = torch.zeros_like(lam[:, 0]) if st["state"] is None else st["state"]
    grad_gate = lam * torch.cat([start[:, None], st["h"][:, :-1].float()], 1)
    if st["case"]["log_gate"]:
        grad_gate = grad_gate * a
    if ok is not None:
        grad_gate = torch.where(ok, grad_gate, 0.0)
    return {"grad_gate": grad_gate.to(dt), "grad_x": lam.to(dt), "grad_state": None if st["state"] is None else a[:, 0] * lam[:, 0]}


# ---- the definition in 64 bits -------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"].startswith("scan"):
        return _exact_scan(case, st)
    n = st["logits"].shape[0]
    step = max(1, 200_000_000 // st["logits"].shape[1])
    parts = [_exact_rows(case, st, slice(i, min(n, i + step))) for i in range(0, n, step)]
    return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_rows(case, st, rows):
    z = st["logits"][rows].double()
    v = z.shape[1]
    if case["op"].startswith("score"):
        t = st["targets"][rows]
        live = t != IGNORE
        if case["op"] == "score":
            u = z * case["scale"]
            lse = torch.logsumexp(u, 1)
            lp = u - lse[:, None]
            p = torch.exp(lp)
            entropy = -torch.nansum(p * lp, 1)
            logp = torch.where(live, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
            top_logp = top_ids = None
            if case["top"]:
                order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : case["top"]]
                top_logp, top_ids = lp.gather(1, order), order.int()
            largest = z.max(1).values
            return {"logp": logp, "entropy": entropy, "norm": torch.stack([largest, lse - largest * case["scale"]], 1), "top_logp": top_logp, "top_ids": top_ids}
        norm = st["norm"][rows].double()
        lp = case["scale"] * (z - norm[:, :1]) - norm[:, 1:]
        p = torch.exp(lp)
        g = torch.where(live, st["grad_logp"][rows].double(), 0.0)[:, None]
        hot = torch.arange(v, device=z.device)[None, :] == t[:, None]
        bonus = torch.nan_to_num(p * (lp + st["entropy"][rows].double()[:, None]), nan=0.0)
        return {"grad": case["scale"] * (g * (hot.double() - p) - st["grad_entropy"][rows].double()[:, None] * bonus)}
    temp = case["temperature"]
    ids = st["ids"][rows].long()
    w = st["weight"][rows].double()
    teacher = torch.where(ids >= 0, st["teacher"][rows].double() / temp, -math.inf)
    q = torch.nan_to_num(torch.softmax(teacher, 1), nan=0.0)
    if case["op"] == "distill":
        largest = z.max(1).values[:, None]
        log_s = torch.logsumexp((z - largest) / temp, 1, keepdim=True)
    else:
        largest, log_s = st["norm"][rows].double().split(1, 1)
    log_p = (z - largest) / temp - log_s
    spread = torch.zeros_like(z)
    spread.scatter_add_(1, ids.clamp(min=0), q)
    grad = (w * temp)[:, None] * (torch.exp(log_p) * q.sum(1)[:, None] - spread)
    if case["op"] == "distill_grad":
        return {"grad": grad}
    kl = (torch.xlogy(q, q) - q * log_p.gather(1, ids.clamp(min=0))).sum(1)
    return {"loss": temp * temp * kl, "norm": torch.cat([largest, log_s], 1), "grad": grad}


def _exact_scan(case, st):
    """Blocks of the sequence one after another; within a block, step by step over all of them at once."""
    a = st["gate"].double()
    if case["log_gate"]:
        a = torch.exp(a)
    b, t, d = a.shape
    lengths = _lengths(case)
    steps = torch.arange(t, device=a.device)[None, :, None]
    inside = steps < torch.tensor(lengths, device=a.device)[:, None, None]
    zero = torch.zeros(b, d, device=a.device, dtype=torch.float64)
    start = zero if st["state"] is None else st["state"].double()
    if case["op"] == "scan":
        # behind a sequence's end the state stays as it is
        h = _exact_states(torch.where(inside, a, 1.0), torch.where(inside, st["x"].double(), 0.0), start)
        return {"h": torch.where(inside, h, 0.0), "final": h[:, -1]}
    g = torch.where(inside, st["grad_h"].double(), 0.0)
    a = torch.where(inside, a, 0.0)
    nxt = torch.zeros_like(a)
    nxt[:, :-1] = a[:, 1:]
    lam = torch.flip(_exact_states(torch.flip(nxt, [1]), torch.flip(g, [1]), zero), [1])
    before = torch.empty_like(lam)
    before[:, 0], before[:, 1:] = start, st["h"][:, :-1].double()
    grad_gate = torch.where(inside, lam * before * (a if case["log_gate"] else 1.0), 0.0)
    return {"grad_gate": grad_gate, "grad_x": lam, "grad_state": None if st["state"] is None else a[:, 0] * lam[:, 0]}


def _exact_states(a, x, start):
    b, t, d = a.shape
    block = max(1, int(math.sqrt(t)))
    count = -(-t // block)
    over = count * block - t
    if over:
        a = torch.cat([a, torch.ones(b, over, d, device=a.device, dtype=a.dtype)], 1)
        x = torch.cat([x, torch.zeros(b, over, d, device=a.device, dtype=a.dtype)], 1)
    a, x = a.reshape(b, count, block, d), x.reshape(b, count, block, d)
    h, reach = torch.empty_like(x), torch.empty_like(x)
    state, left = torch.zeros_like(x[:, :, 0]), torch.ones_like(x[:, :, 0])
    for i in range(block):
        state = a[:, :, i] * state + x[:, :, i]
        left = left * a[:, :, i]
        h[:, :, i], reach[:, :, i] = state, left
    carry = start
    for j in range(count):
        h[:, j] += reach[:, j] * carry[:, None]
        carry = h[:, j, -1]
    return h.reshape(b, count * block, d)[:, :t]
