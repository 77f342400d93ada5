"""The front end's operators on the CPU oracle: their definitions (include/eclat_hip.h) in 64 bits, rounded to f32 at the end.
Test infrastructure, like the rest of this package."""

from __future__ import annotations

import numpy as np

_NP = {"f32": np.float32, "i32": np.int32, "i64": np.int64}


def _array(item):
    buf, shape, dtype = item
    return np.frombuffer(buf.read_to_host(), dtype=_NP[dtype.name]).reshape(shape)


def _log_softmax(z, scale):
    """Largest logit, log of the sum, log probabilities (-inf throughout a row without a logit above -infinity)."""
    m = z.max(1, keepdims=True)
    empty = m == -np.inf
    d = scale * (z - np.where(empty, 0.0, m))
    log_s = np.log(np.exp(d).sum(1, keepdims=True))
    return m, log_s, np.where(empty, -np.inf, d - log_s)


def _times_log(p, x):
    """p x, 0 where p is 0."""
    return np.where(p == 0, 0.0, p * x)


def _teacher(u, ids, v, temperature):
    named = (ids >= 0) & (ids < v)
    x = np.where(named, u.astype(np.float64) / temperature, -np.inf)
    m = x.max(1, keepdims=True)
    e = np.where(named, np.exp(x - np.where(np.isfinite(m), m, 0.0)), 0.0)
    s = e.sum(1, keepdims=True)
    return e / np.where(s > 0, s, 1.0)


def compute(name, attrs, arrays):
    with np.errstate(all="ignore"):
        return _compute(name, attrs, arrays)


def _compute(name, attrs, arrays):
    f = [a.astype(np.float64) if a.dtype.kind == "f" else a for a in arrays]
    if name.startswith("token_logprobs"):
        z, t = f[0], f[1]
        c, (n, v) = attrs["scale"], z.shape
        live = t != attrs["ignore_index"]
        inside = (t >= 0) & (t < v)
        at = np.where(inside, t, 0)
        if name == "token_logprobs":
            m, log_s, lp = _log_softmax(z, c)
            p = np.exp(lp)
            return [np.where(live, np.where(inside, lp[np.arange(n), at], np.nan), 0.0), -_times_log(p, lp).sum(1), np.concatenate([m, log_s], 1)]
        norm, entropy, grads = f[2], f[3], list(f[4:])
        g = np.where(live, grads.pop(0), 0.0) if attrs["logp"] else np.zeros(n)
        g = np.where(live & ~inside, np.nan, g)
        e = grads.pop(0) if attrs["entropy"] else np.zeros(n)
        empty = (norm == -np.inf).all(1)
        lp = c * (z - norm[:, :1]) - norm[:, 1:]
        p = np.exp(lp)
        hot = np.zeros_like(z)
        hot[np.arange(n), at] = live & inside
        grad = c * (g[:, None] * (hot - p) - e[:, None] * _times_log(p, lp + entropy[:, None]))
        return [np.where(empty[:, None], 0.0, grad)]
    if name.startswith("distill_loss"):
        z, u, ids = f[0], f[1], f[2]
        n, v = z.shape
        temp = attrs["temperature"]
        q = _teacher(u, ids, v, temp)
        none = (q == 0).all(1)
        at = np.clip(ids, 0, v - 1)
        if name == "distill_loss":
            m, log_s, lp = _log_softmax(z, 1.0 / temp)
            lp = np.take_along_axis(lp, at, 1)
            loss = temp * temp * _times_log(q, np.log(q) - lp).sum(1)
            return [np.where(none, 0.0, loss), np.concatenate([m, log_s], 1)]
        norm, g = f[3], f[4]
        grad = np.exp((z - norm[:, :1]) / temp - norm[:, 1:])
        np.add.at(grad, (np.arange(n)[:, None], at), -q)
        return [np.where((none | (norm == -np.inf).all(1))[:, None], 0.0, g[:, None] * temp * grad)]
    gate = np.exp(f[0]) if attrs["log_gate"] else f[0]
    b, t, d = gate.shape
    if name == "gated_scan":
        h, out = f[2] if len(f) > 2 else np.zeros((b, d)), np.zeros((b, t, d))
        for i in range(t):
            h = gate[:, i] * h + f[1][:, i]
            out[:, i] = h
        return [out]
    if name == "gated_scan_backward":
        h, g = f[1], f[2]
        first = f[3] if len(f) > 3 else np.zeros((b, d))
        carry, dg, dx = np.zeros((b, d)), np.zeros((b, t, d)), np.zeros((b, t, d))
        for i in range(t - 1, -1, -1):
            dx[:, i] = g[:, i] + carry
            dg[:, i] = dx[:, i] * (h[:, i - 1] if i else first) * (gate[:, i] if attrs["log_gate"] else 1.0)
            carry = gate[:, i] * dx[:, i]
        return [dg, dx, carry][: 3 if len(f) > 3 else 2]
    raise ValueError(f"no operator '{name}'")


def run(allocate, name, attrs, inputs, outputs):
    results = []
    for value, (shape, dtype) in zip(compute(name, attrs, [_array(i) for i in inputs]), outputs):
        buf = allocate(shape, dtype)
        buf.write_from_host(np.ascontiguousarray(value.reshape(shape), dtype=_NP[dtype.name]).tobytes())
        results.append(buf)
    return results
