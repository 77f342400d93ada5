"""The language-model operators as nodes of the front end's graphs: values, gradients, training, on the
CPU oracle and (the same tests, marked gpu) as kernels on the GPU."""

import numpy as np
import pytest

import operator_oracle as oracle


@pytest.fixture(params=["c", pytest.param("hip:0", marks=pytest.mark.gpu)])
def fe(request, frontend):
    if request.param.startswith("hip"):
        request.getfixturevalue("hip")
    frontend.set_device_str(request.param)
    yield frontend
    from harp_amd.frontend.tensor import _INPUT_BUFFER_CACHE
    _INPUT_BUFFER_CACHE.clear()
    frontend.clear_default_device()


def tensor(fe, a, grad=False):
    kind = {"float32": "f32", "int32": "i32", "int64": "i64"}[a.dtype.name]
    t = fe.Tensor.input(list(a.shape), fe.DType(kind)).requires_grad_(grad)
    t.set_data(a)
    return t


def values(t):
    t.realize()
    return t.to_numpy().reshape(t.shape())


def gradients(fe, loss, params, exact=True):
    """Each gradient on its own, as the reference realizes them; lowered in the mode they were built in."""
    with fe.exact_mode(exact):
        loss.backward_with_params(params)
        return [values(p.grad()) for p in params]


def central(f, arrays, k, e=1e-5):
    """Central differences of f (in 64 bits) by the elements of arrays[k]."""
    base = [a.astype(np.float64) if a.dtype.kind == "f" else a for a in arrays]
    out = np.zeros(base[k].shape)
    for at in np.ndindex(out.shape):
        hi, lo = [b.copy() for b in base], [b.copy() for b in base]
        hi[k][at] += e
        lo[k][at] -= e
        out[at] = (f(*hi) - f(*lo)) / (2 * e)
    return out


@pytest.mark.parametrize("exact", [True, False])
def test_scores_and_their_gradient(fe, exact):
    rng = np.random.default_rng(0)
    z, t = rng.normal(0, 2, (5, 23)).astype(np.float32), np.array([0, 22, -1, 7, 7], np.int64)
    logits, targets = tensor(fe, z, True), tensor(fe, t)
    logp, entropy = fe.nn.token_logprobs(logits, targets, scale=0.8)
    want = oracle.score(z, t, -1, 0.8, 0)
    assert np.all(np.abs(values(logp) - want["logp"]) <= want["logp_tol"] + 2.0 ** -24 * np.abs(want["logp"]))
    assert np.all(np.abs(values(entropy) - want["entropy"]) <= want["entropy_tol"] + 2.0 ** -24 * np.abs(want["entropy"]))
    # used together: one backward call for both; a difference step of 1e-5 is off by its square times third
    # derivatives (below 10), and by 1e-15 * 20 / 1e-5
    for loss, f in (((logp + entropy).sum(0), lambda r: (r["logp"] + r["entropy"]).sum()), (logp.sum(0), lambda r: r["logp"].sum()),
                    (entropy.sum(0), lambda r: r["entropy"].sum())):
        got = gradients(fe, loss, [logits], exact)[0]
        want = central(lambda x: f(oracle.score(x, t, -1, 0.8, 0)), [z], 0)
        assert np.all(np.abs(got - want) <= 1e-8 + 2e-6)


def test_cross_entropy_is_the_negated_score(fe):
    """`nn.cross_entropy_loss` with a one-hot tensor and the scores of the same tokens: the same loss and gradient."""
    rng = np.random.default_rng(1)
    z, t = rng.normal(0, 2, (6, 19)).astype(np.float32), rng.integers(0, 19, 6).astype(np.int32)
    one_hot = np.zeros((6, 19), np.float32)
    one_hot[np.arange(6), t] = 1
    a, b = tensor(fe, z, True), tensor(fe, z, True)
    plain = fe.nn.cross_entropy_loss(a, tensor(fe, one_hot), exact=True)
    scored = fe.nn.token_logprobs(b, tensor(fe, t))[0].sum(0).scale_exact(-1.0 / 6)
    # both losses and gradients below 10 and 1 in size, a few dozen f32 roundings each
    assert abs(values(plain) - values(scored)) < 1e-5
    assert np.all(np.abs(gradients(fe, plain, [a])[0] - gradients(fe, scored, [b])[0]) < 1e-5)


@pytest.mark.parametrize("exact", [True, False])
def test_distillation_and_its_gradient(fe, exact):
    rng = np.random.default_rng(2)
    z, u = rng.normal(0, 2, (4, 31)).astype(np.float32), rng.normal(0, 2, (4, 6)).astype(np.float32)
    ids = rng.integers(0, 31, (4, 6)).astype(np.int32)
    ids[1, 3:] = -1
    ids[2] = -1
    ids[3, 1] = ids[3, 0]
    logits = tensor(fe, z, True)
    loss = fe.nn.distill_loss(logits, tensor(fe, u), tensor(fe, ids), temperature=2.0)
    want, tol = oracle.distill(z, u, ids, 2.0, None)[:2]
    assert np.all(np.abs(values(loss) - want) <= tol + 2.0 ** -24 * np.abs(want))
    weight = tensor(fe, rng.random(4).astype(np.float32))
    w = weight.to_numpy().astype(np.float64)
    got = gradients(fe, (loss * weight).sum(0), [logits], exact)[0]
    assert np.all(np.abs(got - central(lambda x: (w * oracle.distill(x, u, ids, 2.0, None)[0]).sum(), [z], 0)) <= 1e-8 + 2e-6)


@pytest.mark.parametrize("log_gate", [False, True])
def test_recurrence_and_its_gradient(fe, log_gate):
    rng = np.random.default_rng(3)
    g = rng.uniform(0.2, 0.95, (2, 6, 3)).astype(np.float32)
    g = np.log(g) if log_gate else g
    x, s = rng.normal(0, 1, (2, 6, 3)).astype(np.float32), rng.normal(0, 1, (2, 3)).astype(np.float32)
    w = rng.normal(0, 1, (2, 6, 3)).astype(np.float32)
    arrays = [g, x, s]
    params = [tensor(fe, a, True) for a in arrays]
    h = fe.nn.gated_scan(params[0], params[1], params[2], log_gate=log_gate)
    want, tol, _, _ = oracle.scan(g, x, s, None, log_gate)
    assert np.all(np.abs(values(h) - want) <= tol + 2.0 ** -24 * np.abs(want))
    got = gradients(fe, (h * tensor(fe, w)).sum(2).sum(1).sum(0), params)
    for k in range(3):
        assert np.all(np.abs(got[k] - central(lambda *v: (w * oracle.scan(*v, None, log_gate)[0]).sum(), arrays, k)) <= 1e-8 + 1e-5)


def test_gates_of_one_are_a_cumulative_sum(fe):
    x = np.random.default_rng(4).normal(0, 1, 40).astype(np.float32)
    ones = fe.Tensor.ones([1, 40, 1])
    got, plain = values(fe.nn.gated_scan(ones, tensor(fe, x.reshape(1, 40, 1)))).ravel(), values(tensor(fe, x).cumsum(0))
    assert np.all(np.abs(got - plain) <= 2 * 40 * 2.0 ** -24 * np.abs(x).cumsum())


def test_sources_of_any_shape_of_graph(fe):
    """Operators on views, on reductions, on constants, on each other, and one tensor as several sources."""
    rng = np.random.default_rng(5)
    a = rng.uniform(0.1, 0.9, (4, 3, 2)).astype(np.float32)
    t = tensor(fe, a)
    g = t.permute([1, 0, 2])                                       # [3,4,2], strided
    h = fe.nn.gated_scan(g, g)
    h2 = fe.nn.gated_scan(fe.nn.sigmoid(h), h * h, h.max(1))
    got = values(h2.sum(2).max(1))
    at = a.transpose(1, 0, 2).astype(np.float64)
    w1 = oracle.scan(at, at, None, None, False)[0]
    w2 = oracle.scan(1 / (1 + np.exp(-w1)), w1 * w1, w1.max(1), None, False)[0]
    assert np.all(np.abs(got - w2.sum(2).max(1)) <= 1e-4)          # values of about 10, under 1e3 roundings of 2^-24
    assert np.all(np.abs(values(h2) - w2) <= 1e-4)
    wide = fe.Tensor.ones([3, 4, 2])
    assert np.all(np.abs(values(fe.nn.gated_scan(wide, wide) + wide) - (np.arange(1, 5)[None, :, None] + 1)) <= 1e-5)


def recurrent_model(fe, params, x, width):
    """Two gated recurrences over [1,T,D] between linear layers, logits [T,V]: what `nn.linear` and the operators
    make together."""
    w_gate, w_in, w_out, b_out = params
    t, d = x.shape()
    gate = fe.nn.sigmoid(fe.nn.linear(x, w_gate)).reshape([1, t, width])
    h = fe.nn.gated_scan(gate, fe.nn.linear(x, w_in).reshape([1, t, width]))
    h = fe.nn.gated_scan(gate, h * (fe.Tensor.ones_like(gate) - gate)).reshape([t, width])
    return fe.nn.linear(h, w_out, b_out)


def numpy_model(params, x):
    w_gate, w_in, w_out, b_out = params
    gate = 1 / (1 + np.exp(-(x @ w_gate.T)))
    h = oracle.scan(gate[None], (x @ w_in.T)[None], None, None, False)[0]
    h = oracle.scan(gate[None], h * (1 - gate[None]), None, None, False)[0][0]
    return h @ w_out.T + b_out


def test_a_recurrent_model_learns_from_a_teacher(fe):
    """The operators together, as a training step uses them: loss and gradients of every parameter against the
    formula's by differences, then steps of SGD on the device, then the scores of tokens under the result."""
    rng = np.random.default_rng(6)
    t, d, width, v, k = 7, 3, 4, 11, 3
    x = rng.normal(0, 1, (t, d)).astype(np.float32)
    arrays = [rng.normal(0, 0.7, s).astype(np.float32) for s in ((width, d), (width, d), (v, width), (v,))]
    u, ids = rng.normal(0, 2, (t, k)).astype(np.float32), np.stack([rng.permutation(v)[:k] for _ in range(t)]).astype(np.int32)

    def total(*p):
        return oracle.distill(numpy_model(p, x.astype(np.float64)), u, ids, 1.5, None)[0].sum() / t
    with fe.exact_mode():
        params = [fe.layers.Parameter(n, a.shape, a) for n, a in zip("abcd", arrays)]
        opt = fe.optim.SGD(params, lr=0.1)
        for step in range(3):
            logits = recurrent_model(fe, [p.tensor() for p in params], tensor(fe, x), width)
            loss = fe.nn.distill_loss(logits, tensor(fe, u), tensor(fe, ids), temperature=1.5).sum(0).scale_exact(1.0 / t)
            loss.backward_with_params([p.tensor() for p in params])
            now = [p.to_numpy() for p in params]
            if step == 0:
                for i, p in enumerate(params):
                    got = values(p.tensor().grad().contiguous())
                    # f32 through four linear layers and two scans: gradients below 3, under 1e3 roundings
                    assert np.all(np.abs(got - central(total, now, i)) <= 3 * 1000 * 2.0 ** -24), i
            opt.step(also=[loss])
            assert abs(float(loss.to_numpy()[0]) - total(*[n.astype(np.float64) for n in now])) < 1e-5
        tokens = ids[:, 0].copy()
        logits = recurrent_model(fe, [p.tensor() for p in params], tensor(fe, x), width)
        logp, entropy = fe.nn.token_logprobs(logits, tensor(fe, tokens))
        z = numpy_model([p.to_numpy().astype(np.float64) for p in params], x.astype(np.float64))
        lp = z - z.max(1, keepdims=True)
        lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
        fe.tensor.realize_many([logp, entropy])
        assert np.all(np.abs(logp.to_numpy() - lp[np.arange(t), tokens]) < 1e-4)
        assert np.all(np.abs(entropy.to_numpy() + (np.exp(lp) * lp).sum(1)) < 1e-4)


def many(fe, *tensors):
    """Realized together; each as its shape says."""
    fe.tensor.realize_many(tensors)
    return [t.to_numpy().reshape(t.shape()) for t in tensors]


def test_views_of_outputs_realized_with_other_roots(fe):
    """A root that is a view of an operator's output, or of what one is computed into, has its own values, in the
    view's order, whatever else is realized with it."""
    rng = np.random.default_rng(7)
    z, t = rng.normal(0, 2, (4, 9)).astype(np.float32), np.array([0, 3, 8, 5], np.int32)
    logp, entropy = fe.nn.token_logprobs(tensor(fe, z), tensor(fe, t))
    lp, as_square, total, e = many(fe, logp, logp.reshape([2, 2]), logp + entropy, entropy)
    assert np.array_equal(as_square, lp.reshape(2, 2)) and np.array_equal(total, lp + e)
    a = rng.uniform(0.1, 0.9, (2, 3, 4)).astype(np.float32)
    g = tensor(fe, a)
    h = fe.nn.gated_scan(g, g)
    want = values(h)
    twice = h + h
    views = [h.permute([0, 2, 1]), twice.permute([2, 1, 0]), h.reshape([6, 4]), h.unsqueeze(0).expand(0, 2), -h.permute([1, 0, 2])]
    wanted = [want.transpose(0, 2, 1), (want + want).transpose(2, 1, 0), want.reshape(6, 4), np.stack([want, want]), -want.transpose(1, 0, 2)]
    for got, w in zip(many(fe, *views, h * h, h), wanted + [want * want, want]):
        assert np.array_equal(got, w)
    for v, w in zip(views, wanted):                                  # and alone
        v.clear_buffer()
        assert np.array_equal(values(v), w)


def test_an_operators_source_and_its_views_as_roots(fe):
    """What an operator reads is computed before it; as a root, and as a view in a root, it is still found, and so is
    a view of an input.  What is computed of inputs alone is what it is without operators."""
    rng = np.random.default_rng(8)
    a, b = rng.uniform(0.1, 0.9, (2, 3, 4)).astype(np.float32), rng.uniform(0.1, 0.9, (2, 3, 4)).astype(np.float32)
    ta, tb = tensor(fe, a), tensor(fe, b)
    gate = ta * tb
    h = fe.nn.gated_scan(gate, tb)
    flat, swapped = gate.reshape([6, 4]), gate.permute([0, 2, 1])
    swapped.realize()
    before = swapped.to_numpy()
    swapped.clear_buffer()
    fe.tensor.realize_many([gate, flat, swapped, tb.reshape([4, 6]), h, h + gate])
    x = a * b
    assert np.array_equal(gate.to_numpy().reshape(x.shape), x) and np.array_equal(flat.to_numpy(), x.ravel())
    assert np.array_equal(swapped.to_numpy(), before)
    got = many(fe, tb.reshape([4, 6]), ta.permute([2, 0, 1]), h * h, h)
    assert np.array_equal(got[0], b.reshape(4, 6)) and np.array_equal(got[1], a.transpose(2, 0, 1)) and np.array_equal(got[2], got[3] * got[3])


@pytest.mark.parametrize("exact", [True, False])
def test_a_view_read_by_an_operator_and_by_others(fe, exact):
    """One strided view as an operator's source, as a root, and inside another source and another root: each has its
    elements (in both modes, though a view with several readers is lowered differently in them)."""
    rng = np.random.default_rng(12)
    a, b = rng.uniform(0.1, 0.9, (2, 4, 3)).astype(np.float32), rng.uniform(0.1, 0.9, (2, 3, 4)).astype(np.float32)
    with fe.exact_mode(exact):
        p = tensor(fe, a).permute([0, 2, 1])
        h = fe.nn.gated_scan(-p, p)
        q = h.permute([2, 0, 1])
        got_h, got_q, got_n = many(fe, h, q, -(q * tensor(fe, b.transpose(2, 0, 1).copy())))
    at = a.transpose(0, 2, 1)
    want, tol, _, _ = oracle.scan(-at, at, None, None, False)
    assert np.all(np.abs(got_h - want) <= tol + 2.0 ** -24 * np.abs(want))
    assert np.array_equal(got_q, got_h.transpose(2, 0, 1)) and np.array_equal(got_n, -(got_h * b).transpose(2, 0, 1))


@pytest.mark.parametrize("exact", [True, False])
def test_gradients_behind_a_reshape_realized_together(fe, exact):
    """The gradients of a step, which are views of one backward call's outputs, from one `realize_many`."""
    rng = np.random.default_rng(9)
    a, b, w = (rng.uniform(0.2, 0.9, (4, 2)).astype(np.float32) for _ in range(3))
    params = [tensor(fe, x, True) for x in (a, b, w)]
    with fe.exact_mode(exact):
        h = fe.nn.gated_scan(params[0].reshape([1, 4, 2]), params[1].reshape([1, 4, 2])).reshape([4, 2])
        loss = (h * params[2]).sum(1).sum(0)
        loss.backward_with_params(params)
        together = many(fe, *[p.grad() for p in params], loss)
    states = oracle.scan(a[None], b[None], None, None, False)[0][0]
    dg, dx, _ = oracle.scan_grad(a[None], states[None], w[None].astype(np.float64), None, None, False, None)[0]
    # sums of four terms below 4, a dozen roundings each
    for got, want in zip(together, (dg[0], dx[0], states, (states * w).sum())):
        assert np.all(np.abs(got - want) <= 12 * 4 * 2.0 ** -24)


@pytest.mark.parametrize("exact", [True, False])
def test_second_derivatives_are_refused(fe, exact):
    """A gradient's own gradient through an operator is not there; the terms are not left out silently."""
    rng = np.random.default_rng(10)
    z, x = tensor(fe, rng.normal(0, 1, (3, 5)).astype(np.float32), True), tensor(fe, rng.uniform(0.2, 0.9, (1, 3, 2)).astype(np.float32), True)
    w = tensor(fe, rng.normal(0, 1, (3, 5)).astype(np.float32), True)
    one, other = tensor(fe, np.array([4, 0, 2], np.int32)), tensor(fe, np.array([[1, 2], [0, 3], [4, -1]], np.int32))
    teacher = tensor(fe, rng.normal(0, 1, (3, 2)).astype(np.float32))

    def total(t):
        return t.reshape([int(np.prod(t.shape()))]).sum(0)
    for p, y in ((z, fe.nn.token_logprobs(z, one)[0]), (z, fe.nn.token_logprobs(z, one)[1]), (z, fe.nn.distill_loss(z, teacher, other)),
                 (x, fe.nn.gated_scan(x, x))):
        with fe.exact_mode(exact):
            p.zero_grad()
            total(y * y).backward_with_params([p])
            again = total(p.grad() * p.grad())
            with pytest.raises(NotImplementedError, match="_backward' has no derivative"):
                again.backward_with_params([p])
            # by what the gradient does not depend on through the operator: ordinary
            if p is z:
                total(p.grad() * w).backward_with_params([w])
                assert np.array_equal(values(w.grad()), values(p.grad().contiguous()))


def same(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    with np.errstate(invalid="ignore"):
        return np.all((np.isnan(got) & np.isnan(want)) | (got == want) | (np.abs(got - want) <= tol + 2.0 ** -24 * np.abs(want)))


def test_masked_rows_and_ids_outside_the_vocabulary(fe):
    """Tokens that cannot occur, rows of nothing else, targets that are no token, rows without the teacher's entries."""
    rng = np.random.default_rng(11)
    z = rng.normal(0, 2, (6, 13)).astype(np.float32)
    z[0, ::2] = -np.inf
    z[1] = -np.inf
    z[2, 1:] = -np.inf
    t = np.array([1, 4, 0, 13, -7, -1], np.int64)
    logits = tensor(fe, z, True)
    logp, entropy = fe.nn.token_logprobs(logits, tensor(fe, t))
    want = oracle.score(z, t, -1, 1.0, 0)
    assert same(values(logp), want["logp"], want["logp_tol"]) and same(values(entropy), want["entropy"], want["entropy_tol"])
    g, e = rng.normal(0, 1, 6).astype(np.float32), rng.normal(0, 1, 6).astype(np.float32)
    with fe.exact_mode():
        got = gradients(fe, (logp * tensor(fe, g) + entropy * tensor(fe, e)).sum(0), [logits])[0]
    # the norm and the entropy that it reads are within their own bounds of these, and p |log p + H| is below 20
    norm, ent = want["norm"].astype(np.float32), want["entropy"].astype(np.float32)
    grad, tol = oracle.score_grad(z, t, -1, 1.0, norm, ent, g, e)
    off = (np.abs(g) + 20 * np.abs(e))[:, None] * (want["norm_tol"][:, 1:] + want["entropy_tol"][:, None] + 2 * 2.0 ** -24 * 20)
    assert same(got, grad, tol + off)

    u, ids = rng.normal(0, 2, (6, 3)).astype(np.float32), np.array([[1, 3, 5], [0, 1, 2], [0, -1, 13], [2, 2, 3], [-1, 13, -9], [4, 5, -1]], np.int32)
    z[4, 3] = np.nan
    z[5, 4] = -np.inf
    u[5, 0] = -np.inf
    logits = tensor(fe, z, True)
    loss = fe.nn.distill_loss(logits, tensor(fe, u), tensor(fe, ids))
    want, loss_tol, _, norm_tol, grad, tol = oracle.distill(np.where(np.isnan(z), 0, z), u, ids, 1.0, None)
    assert want[4] == 0 and want[1] == np.inf and np.isfinite(want[[0, 2, 3, 5]]).all() and not grad[[1, 4]].any()
    assert same(values(loss), want, loss_tol)
    with fe.exact_mode():
        got = gradients(fe, loss.sum(0), [logits])[0]
    assert same(got, grad, tol + norm_tol[:, 1:] + 2.0 ** -24 * 20)        # p is at most 1, its argument off by the norm's rounding


@pytest.mark.parametrize("bad", [
    lambda fe, z, t, s: fe.nn.token_logprobs(z, t.cast(fe.F32)),
    lambda fe, z, t, s: fe.nn.token_logprobs(z, tensor(fe, np.zeros(3, np.int32))),
    lambda fe, z, t, s: fe.nn.token_logprobs(z.sum(0), t),
    lambda fe, z, t, s: fe.nn.distill_loss(z, z, t),
    lambda fe, z, t, s: fe.nn.distill_loss(z, z, tensor(fe, np.zeros((4, 5), np.int32))),
    lambda fe, z, t, s: fe.nn.gated_scan(s, z),
    lambda fe, z, t, s: fe.nn.gated_scan(s, s, s),
    lambda fe, z, t, s: fe.nn.gated_scan(s, s.cast(fe.I32)),
])
def test_refused_shapes_and_types(fe, bad):
    z, t = tensor(fe, np.zeros((4, 6), np.float32)), tensor(fe, np.zeros(4, np.int32))
    with pytest.raises(ValueError):
        bad(fe, z, t, tensor(fe, np.zeros((2, 3, 4), np.float32)))


def test_an_input_without_a_buffer(fe):
    from harp_amd.frontend.executor import ExecutionError, execute_graph
    logp, _ = fe.nn.token_logprobs(fe.Tensor.input([2, 3], fe.F32), fe.Tensor.input([2], fe.DType("i64")))
    with pytest.raises(ExecutionError, match="MissingInput"):
        execute_graph([logp.graph], {})


def test_programs_and_backends_without_operators(fe):
    from harp_amd.frontend.lowerer import LoweringError, lower_graph
    s = tensor(fe, np.ones((1, 2, 3), np.float32))
    h = fe.nn.gated_scan(s, s)
    with pytest.raises(LoweringError, match="gated_scan"):
        lower_graph([(h + h).graph])
    dev = fe.get_default_device()

    class Bare:
        kind = "bare"

        def __getattr__(self, name):
            if name in ("run_operator", "compile_program"):
                raise AttributeError(name)
            return getattr(dev.backend, name)
    old, dev.backend = dev.backend, Bare()
    try:
        with pytest.raises(fe.ExecutionError, match="no operators"):
            h.realize()
    finally:
        dev.backend = old
    assert np.array_equal(values(h).ravel(), np.repeat([1, 2], 3).astype(np.float32))
