"""Plain 64-bit forms of the language-model operators (numpy), with the rounding errors that an f32
evaluation of them may have: what the kernels are held to.

u = 2^-24 is half a step of f32.  The error bounds are sums of the roundings along each value's way:
an exponential's argument is computed in at most four roundings and exp2 is good to one step, so a
term exp(x) carries (4 |x| + 2) u; a sum of n terms by 256 threads or fewer of a row carries
n / 64 + 64 roundings (a thread's chain, then trees); a logarithm of the sum takes that as an absolute error.
"""

import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
SMALLEST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}     # results below are rounded absolutely (or flushed)


def rounding(dtype, want):
    """What the one rounding of a result to `dtype` may move it."""
    return HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]


def _row_parts(z, scale):
    z = z.astype(np.float64)
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        d = np.where(m == -np.inf, -np.inf, (z - m) * scale)
        e = np.where(d == -np.inf, 0.0, np.exp(d))
        s = e.sum(1, keepdims=True)
        log_s = np.log(s)
    return m, d, e, s, log_s


def sum_error(d, n):
    """Bound of |log S - its f32 value| for a row with arguments d <= 0: the terms' errors, weighted by the terms."""
    e = np.where(np.isfinite(d), np.exp(np.where(np.isfinite(d), d, 0.0)), 0.0)
    x = np.where(e > 0, -np.where(np.isfinite(d), d, 0.0), 0.0)
    s = np.maximum(e.sum(1), 1e-300)
    return ((e * (4 * x + 2)).sum(1) / s + n / 64 + 64) * U


def score(z, targets, ignore, scale, top):
    """dict of results and, under the same names with _tol, how far f32 may be off."""
    scale = float(np.float32(scale))
    n, v = z.shape
    m, d, e, s, log_s = _row_parts(z, scale)
    empty = s[:, 0] == 0
    err = sum_error(d, v)
    with np.errstate(all="ignore"):
        lp = np.where(empty[:, None], -np.inf, d - log_s)
        p = e / s
        ent = np.where(empty, 0.0, log_s[:, 0] - np.where(e > 0, d * e, 0.0).sum(1) / s[:, 0])
    t = np.asarray(targets)
    inside = (t >= 0) & (t < v)
    logp = np.where(t == ignore, 0.0, np.where(inside, lp[np.arange(n), np.clip(t, 0, v - 1)], np.nan))
    out = {"logp": logp, "entropy": ent, "norm": np.concatenate([m, log_s], 1)}
    fin = np.where(np.isfinite(lp), np.abs(lp), 0.0)
    out["logp_tol"] = err + 4 * U * (np.where(np.isfinite(logp), np.abs(logp), 0) + np.abs(np.where(np.isfinite(log_s[:, 0]), log_s[:, 0], 0)) + 1)
    # the two parts of H carry the sums' error, relative to themselves, twice over
    out["entropy_tol"] = 4 * (err + 4 * U) * (1 + np.abs(ent) + np.abs(np.where(np.isfinite(log_s[:, 0]), log_s[:, 0], 0)))
    out["norm_tol"] = np.stack([np.zeros(n), err + 4 * U * (1 + np.abs(np.where(np.isfinite(log_s[:, 0]), log_s[:, 0], 0)))], 1)
    if top:
        key = np.where(np.isnan(z), -np.inf, z.astype(np.float64)) + 0.0
        order = np.argsort(-key, axis=1, kind="stable")[:, :top]
        out["top_ids"] = order
        out["top_logp"] = np.take_along_axis(lp, order, 1)
        out["top_logp_tol"] = (err + 4 * U * (1 + np.abs(np.where(np.isfinite(log_s[:, 0]), log_s[:, 0], 0))))[:, None] + 4 * U * np.take_along_axis(fin, order, 1)
    return out


def score_grad(z, targets, ignore, scale, norm, entropy, g, h):
    scale = float(np.float32(scale))
    n, v = z.shape
    z = z.astype(np.float64)
    m, log_s = norm[:, :1].astype(np.float64), norm[:, 1:].astype(np.float64)
    empty = (m == -np.inf) & (log_s == -np.inf)
    with np.errstate(all="ignore"):
        lp = np.where(empty, -np.inf, (z - m) * scale - log_s)
        p = np.where(lp == -np.inf, 0.0, np.exp(lp))
    t = np.asarray(targets)
    gg = np.where(t == ignore, 0.0, 0.0 if g is None else g.astype(np.float64))
    hh = np.zeros(n) if h is None else h.astype(np.float64)
    ent = np.zeros(n) if entropy is None else entropy.astype(np.float64)
    x = np.where(np.isfinite(lp), lp, 0.0)
    hot = np.zeros((n, v))
    live = (t != ignore) & (t >= 0) & (t < v)
    hot[np.arange(n)[live], t[live]] = 1.0
    want = scale * (gg[:, None] * (hot - p) - hh[:, None] * p * (x + ent[:, None]))
    want = np.where(empty, 0.0, want)
    # p carries its argument's error, which is that of (z - m) scale and of log S; the sums of a product a few roundings each
    arg = (4 * (np.abs(x) + np.abs(np.where(np.isfinite(log_s), log_s, 0.0))) + 8) * U
    tol = scale * p * (np.abs(gg)[:, None] + np.abs(hh)[:, None] * (np.abs(x) + np.abs(ent)[:, None] + 1)) * (2 * arg + 8 * U) + scale * hot * np.abs(gg)[:, None] * 4 * U
    bad = (t != ignore) & ((t < 0) | (t >= v))
    want[bad] = np.nan
    want[empty[:, 0]] = 0.0
    return want, tol


def teacher_of(u, ids, v, temperature):
    temperature = float(np.float32(temperature))
    named = (ids >= 0) & (ids < v)
    x = np.where(named, u.astype(np.float64) / temperature, -np.inf)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        x = np.where(m == -np.inf, -np.inf, x - m)
        q = np.where(x == -np.inf, 0.0, np.exp(x))
        s = q.sum(1, keepdims=True)
        q = np.where(s > 0, q / np.where(s > 0, s, 1), 0.0)
        log_q = np.where(q > 0, x - np.log(np.where(s > 0, s, 1)), 0.0)
    rel = (4 * np.where(np.isfinite(x), -x, 0.0) + x.shape[1] / 8 + 80) * U        # of q, and absolute of log q
    return q, log_q, rel


def distill(z, u, ids, temperature, weight, norm=None):
    """(loss, loss_tol, norm, norm_tol, grad, grad_tol); the gradient for the given `norm` where there is one."""
    n, v = z.shape
    temp = float(np.float32(temperature))
    m, d, e, s, log_s = _row_parts(z, 1.0 / temp)
    err = sum_error(d, v)
    empty = s[:, 0] == 0
    if norm is not None:
        m, log_s = norm[:, :1].astype(np.float64), norm[:, 1:].astype(np.float64)
        empty = (m[:, 0] == -np.inf) & (log_s[:, 0] == -np.inf)
        err = np.zeros(n)
        with np.errstate(all="ignore"):
            d = (z.astype(np.float64) - m) / temp
    q, log_q, rel = teacher_of(u, ids, v, temp)
    with np.errstate(all="ignore"):
        lp = np.where(empty[:, None], -np.inf, d - log_s)
        p = np.where(lp == -np.inf, 0.0, np.exp(lp))
    at = np.clip(ids, 0, v - 1)
    lp_at = np.take_along_axis(lp, at, 1)
    with np.errstate(all="ignore"):
        terms = np.where(q > 0, q * (log_q - lp_at), 0.0)
    loss = temp * temp * terms.sum(1)
    fin = np.where(np.isfinite(lp_at), np.abs(lp_at), 0.0)
    ls = np.abs(np.where(np.isfinite(log_s), log_s, 0.0))
    loss_tol = temp * temp * (q * ((np.abs(log_q) + fin + 1) * (rel + ids.shape[1] / 16 * U + 16 * U) + err[:, None] + 4 * U * (fin + ls))).sum(1)
    spread = np.zeros((n, v))
    spread_tol = np.zeros((n, v))
    np.add.at(spread, (np.arange(n)[:, None], at), q)
    np.add.at(spread_tol, (np.arange(n)[:, None], at), q * (rel + 8 * U))
    total = (q.sum(1) > 0).astype(np.float64)[:, None]
    w = (np.ones(n) if weight is None else weight.astype(np.float64))[:, None] * temp
    grad = np.where(empty[:, None], 0.0, w * (total * p - spread))
    x = np.where(np.isfinite(lp), np.abs(lp), 0.0)
    grad_tol = np.abs(w) * (total * p * (((4 * (x + ls) + 16) * U + err[:, None])) + spread_tol + 4 * U * np.abs(total * p - spread))
    norm_tol = np.stack([np.zeros(n), err + 4 * U * (1 + ls[:, 0])], 1)
    return loss, loss_tol, np.concatenate([m, log_s], 1), norm_tol, grad, grad_tol


def scan(gate, x, state, lengths, log_gate):
    """(h, h_tol, final, final_tol): a step's product and sum are two roundings on everything summed so far (and
    those of its gate), joining pieces of the sequence a fixed number more."""
    g = gate.astype(np.float64)
    a = np.exp(g) if log_gate else g
    per = 4 + (4 * np.abs(np.where(np.isfinite(g), g, 0.0)) + 4 if log_gate else 0)
    b, t, d = g.shape
    n = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    h = np.zeros((b, d)) if state is None else state.astype(np.float64)
    mag, err = np.abs(h), np.zeros((b, d))
    hs, tol = np.zeros((b, t, d)), np.zeros((b, t, d))
    for i in range(t):
        live = (i < n)[:, None]
        p = per[:, i] if log_gate else per
        h = np.where(live, a[:, i] * h + x[:, i], h)
        err = np.where(live, np.abs(a[:, i]) * (err + p * mag), err)
        mag = np.where(live, np.abs(a[:, i]) * mag + np.abs(x[:, i].astype(np.float64)), mag)
        hs[:, i], tol[:, i] = h, (err + 64 * mag) * U
    return hs, tol, h, (err + 64 * mag) * U


def scan_grad(gate, h, grad_h, state, lengths, log_gate, grad_final):
    """((grad_gate, grad_x, grad_state), the same with tolerances)."""
    g = gate.astype(np.float64)
    a = np.exp(g) if log_gate else g
    b, t, d = g.shape
    n = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    zero = np.zeros((b, d))
    before0 = zero if state is None else state.astype(np.float64)
    carry = zero if grad_final is None else grad_final.astype(np.float64)
    mag, err = np.abs(carry), np.zeros((b, d))
    dg, dx = np.zeros((b, t, d)), np.zeros((b, t, d))
    dg_tol, dx_tol = np.zeros((b, t, d)), np.zeros((b, t, d))
    for i in range(t - 1, -1, -1):
        live = (i < n)[:, None]
        p = 4 + (4 * np.abs(np.where(np.isfinite(g[:, i]), g[:, i], 0.0)) + 4 if log_gate else 0)
        lam = carry + grad_h[:, i]
        lmag = mag + np.abs(grad_h[:, i].astype(np.float64))
        before = before0 if i == 0 else h[:, i - 1].astype(np.float64)
        tol = (err + 64 * lmag) * U
        scale = a[:, i] if log_gate else np.ones((b, d))
        dx[:, i], dx_tol[:, i] = np.where(live, lam, 0), np.where(live, tol, 0)
        dg[:, i] = np.where(live, lam * before * scale, 0)
        dg_tol[:, i] = np.where(live, np.abs(before * scale) * (tol + (8 + p) * U * np.abs(lam)), 0)
        carry = np.where(live, a[:, i] * lam, carry)
        err = np.where(live, np.abs(a[:, i]) * (err + p * lmag), err)
        mag = np.where(live, np.abs(a[:, i]) * lmag, mag)
    return (dg, dx, carry), (dg_tol, dx_tol, (err + 64 * mag) * U)
