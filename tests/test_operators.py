"""The language-model operators on the GPU against their plain 64-bit forms (operator_oracle.py)."""

import itertools

import numpy as np
import pytest

import operator_oracle as oracle

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    from harp_amd import backend as hb
    if hb.device_count() == 0:
        pytest.skip("no HIP device")
    return hb.HipDevice(0, stream=torch.cuda.current_stream().cuda_stream)


@pytest.fixture(scope="module")
def ops():
    from harp_amd import operators
    return operators


def on_gpu(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(DT[dtype])).cuda()


def host(t):
    return t.detach().double().cpu().numpy()


def rows_of(n, v, dtype, seed, spread=3.0, stride=None):
    """Logits as the GPU holds them (values of `dtype`), [n, v] with rows `stride` elements apart."""
    z = np.random.default_rng(seed).normal(0, spread, (n, stride or v)).astype(np.float32)
    return on_gpu(z, dtype)[:, :v]


def close(got, want, tol, what):
    """NaN and infinities in the same places, everything else within the bound.  (A result beyond f32's largest
    number, (2 - 2^-23) 2^127, by half a step or more rounds to infinity: such a log probability is one of a lowest
    value times a scale above 1.)"""
    got = np.asarray(got, np.float64)
    want = np.where(np.abs(want) >= (2 - 2.0 ** -24) * 2.0 ** 127, np.copysign(np.inf, want), want)
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(all="ignore"):
        off = np.where(same, 0.0, np.abs(got - want) - tol)
    worst = np.nanargmax(np.where(np.isnan(off), np.inf, off)) if off.size else 0
    assert off.size == 0 or bool(np.all(off <= 0)), (what, np.unravel_index(worst, off.shape), got.flat[worst], want.flat[worst], np.broadcast_to(tol, off.shape).flat[worst])


def check_score(dev, ops, z, targets, top=0, scale=1.0, ignore=-1, entropy=True, workspace=None):
    n, v = z.shape
    out = ops.Logprobs(torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda") if entropy else None,
                       torch.full((n, 2), 7.0, device="cuda"), torch.full((n, top), 7.0, device="cuda") if top else None,
                       torch.full((n, top), 7, device="cuda", dtype=torch.int32) if top else None)
    ops.token_logprobs(dev, z, targets, top=top, scale=scale, ignore_index=ignore, out=out, workspace=workspace)
    want = oracle.score(host(z), targets.cpu().numpy(), ignore, scale, top)
    close(host(out.logp), want["logp"], want["logp_tol"], "logp")
    close(host(out.norm), want["norm"], want["norm_tol"], "norm")
    if entropy:
        close(host(out.entropy), want["entropy"], want["entropy_tol"], "entropy")
    if top:
        assert np.array_equal(out.top_ids.cpu().numpy(), want["top_ids"])
        close(host(out.top_logp), want["top_logp"], want["top_logp_tol"], "top_logp")
    return out


SIZES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 255), (4, 257), (9, 1000), (3, 4097), (2, 8191), (1, 40000), (7, 33333), (1100, 131)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", SIZES)
def test_score_sizes(dev, ops, n, v, dtype):
    z = rows_of(n, v, dtype, seed=n * 7919 + v)
    t = on_gpu(np.random.default_rng(5).integers(0, v, n))
    check_score(dev, ops, z, t, top=min(v, 5))
    check_score(dev, ops, z, t.int(), top=0, scale=0.7, entropy=False)
    check_score(dev, ops, z, t, top=min(v, 32), scale=1.6)


@pytest.mark.parametrize("dtype,n,v", [("f32", 1, 140001), ("bf16", 2, 300003), ("f32", 60, 131080), ("f32", 260, 2001), ("f32", 260, 8003),
                                       ("f32", 260, 16001), ("bf16", 2050, 33001), ("f16", 70, 270000)])
def test_score_of_every_launch_shape(dev, ops, dtype, n, v):
    """Rows of one to sixteen waves, rows in segments, aligned and not."""
    z = rows_of(n, v, dtype, seed=v)
    t = on_gpu(np.random.default_rng(5).integers(0, v, n))
    check_score(dev, ops, z, t, top=20)
    check_score(dev, ops, z, t, top=0, entropy=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,shift", [(3, 1001, 1), (5, 4099, 3), (2, 33000, 5)])
def test_score_rows_at_any_alignment(dev, ops, n, v, shift, dtype):
    wide = rows_of(n, v + shift + 6, dtype, seed=v)
    z = wide[:, shift:shift + v]
    assert z.stride(0) == v + shift + 6
    check_score(dev, ops, z, on_gpu(np.arange(n)), top=7)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [64, 5000, 70000])
def test_score_of_ties(dev, ops, v, dtype):
    """All equal, few values, one value below a plateau, signed zeros: equal logits go by their id."""
    rng = np.random.default_rng(v)
    z = np.zeros((5, v), np.float32)
    z[1] = rng.integers(0, 3, v)
    z[2, :] = 1.0
    z[2, rng.integers(0, v, 40)] = 0.5
    z[3] = np.where(rng.random(v) < 0.5, 0.0, -0.0)
    z[4] = -np.arange(v) // 16
    check_score(dev, ops, on_gpu(z, dtype), on_gpu(np.full(5, v - 1)), top=32)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [50, 3000, 60000])
def test_score_of_sorted_rows(dev, ops, v, dtype):
    up = np.linspace(-20, 20, v, dtype=np.float32)
    z = np.stack([up, up[::-1], np.concatenate([up[v // 2:], up[:v // 2]])])
    check_score(dev, ops, on_gpu(z, dtype), on_gpu(np.array([0, v // 2, v - 1])), top=20)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [9, 2048, 50001])
def test_score_of_masked_rows(dev, ops, v, dtype):
    """Entries of -infinity, of the type's lowest value, rows of nothing else, one live entry."""
    low = float(torch.finfo(DT[dtype]).min)
    z = np.random.default_rng(v).normal(0, 2, (7, v)).astype(np.float32)
    z[0] = -np.inf
    z[1, :] = -np.inf
    z[1, v // 2] = -3.0
    z[2] = low
    z[3, ::2] = low
    z[4, 1:] = -np.inf
    z[5, : v - 1] = -np.inf
    z[6, ::2] = -np.inf
    t = on_gpu(np.array([0, v // 2, v - 1, 0, 0, 0, 0]))
    gpu = on_gpu(z, dtype)
    gpu[2] = low
    gpu[3, ::2] = low
    for scale in (1.0, 0.5, 1.7):
        out = check_score(dev, ops, gpu, t, top=min(9, v), scale=scale)
        grad = ops.token_logprobs_backward(dev, gpu, t, out.norm, out.entropy, on_gpu(np.ones(7, np.float32)), on_gpu(np.full(7, 0.25, np.float32)),
                                           scale=scale, out=torch.full_like(gpu, 9.0))
        want, tol = oracle.score_grad(host(gpu), t.cpu().numpy(), -1, scale, host(out.norm), host(out.entropy), np.ones(7), np.full(7, 0.25))
        close(host(grad), want, tol + oracle.rounding(dtype, want), "grad")
        assert not host(grad)[0].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [100, 40000])
def test_score_of_nan_and_infinity(dev, ops, v, dtype):
    z = np.random.default_rng(v).normal(0, 2, (4, v)).astype(np.float32)
    z[0, v // 3] = np.nan
    z[1, v - 1] = np.inf
    z[2] = np.nan
    z[2, 5] = 1.0
    gpu, t = on_gpu(z, dtype), on_gpu(np.array([1, v - 1, 5, -1]))
    out = ops.token_logprobs(dev, gpu, t, top=3, out=ops.Logprobs(*(torch.empty(s, device="cuda") for s in ((4,), (4,), (4, 2), (4, 3))),
                                                                  torch.empty(4, 3, device="cuda", dtype=torch.int32)))
    assert np.isnan(host(out.logp)[:3]).all() and np.isnan(host(out.entropy)[:3]).all() and np.isnan(host(out.top_logp)[:3]).all()
    ids = out.top_ids.cpu().numpy()
    clean = np.where(np.isnan(host(gpu)), -np.inf, host(gpu))
    assert np.array_equal(ids[0], np.argsort(-clean[0], kind="stable")[:3])
    assert ids[1, 0] == v - 1 and list(ids[2]) == [5, -1, -1]
    assert host(out.logp)[3] == 0.0 and np.isfinite(host(out.entropy)[3])


def test_score_ids_outside_the_vocabulary(dev, ops):
    z = rows_of(6, 513, "f32", 3)
    for dt in (torch.int32, torch.int64):
        t = torch.tensor([-1, 513, -2, 2 ** 31 - 1, 512, -100], device="cuda").to(dt)
        out = check_score(dev, ops, z, t)
        assert np.array_equal(np.isnan(host(out.logp)), [False, True, True, True, False, True])
        out = check_score(dev, ops, z, t, ignore=-100)
        assert host(out.logp)[5] == 0.0 and np.isnan(host(out.logp)[0])
        grad = ops.token_logprobs_backward(dev, z, t, out.norm, None, on_gpu(np.ones(6, np.float32)), ignore_index=-100, out=torch.empty_like(z))
        assert np.array_equal(np.isnan(host(grad)).all(1), [True, True, True, True, False, False])
        assert not host(grad)[5].any()
    big = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 2 ** 32 + 5, 0, 1], device="cuda")
    assert np.array_equal(np.isnan(host(check_score(dev, ops, z, big).logp)), [True] * 4 + [False] * 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", SIZES)
def test_score_gradient(dev, ops, n, v, dtype):
    rng = np.random.default_rng(n + v)
    z = rows_of(n, v, dtype, seed=v, stride=v + 3)
    t = on_gpu(np.where(rng.random(n) < 0.2, -1, rng.integers(0, v, n)))
    g, h = rng.normal(0, 1, n).astype(np.float32), rng.normal(0, 0.3, n).astype(np.float32)
    s = check_score(dev, ops, z, t, scale=0.8)
    for gg, hh in ((g, h), (g, None), (None, h), (None, None)):
        out = torch.full((n, v + 5), 5.0, device="cuda", dtype=DT[dtype])
        ops.token_logprobs_backward(dev, z, t, s.norm, s.entropy, None if gg is None else on_gpu(gg), None if hh is None else on_gpu(hh),
                                    scale=0.8, out=out[:, :v])
        want, tol = oracle.score_grad(host(z), t.cpu().numpy(), -1, 0.8, host(s.norm), host(s.entropy), gg, hh)
        close(host(out[:, :v]), want, tol + oracle.rounding(dtype, want), "grad")
        assert bool((out[:, v:] == 5.0).all())


def test_score_gradient_against_differences(dev, ops):
    """Central differences of the oracle's own sum: a step e has an error of e^2 / 6 times the third
    derivative (below 8 for log p and H at these sizes) and of the sum's rounding over e."""
    rng = np.random.default_rng(1)
    n, v, scale = 4, 37, 1.3
    z = rng.normal(0, 1.5, (n, v)).astype(np.float32)
    t = np.array([3, 36, -1, 0])
    g, h = rng.normal(0, 1, n).astype(np.float32), rng.normal(0, 1, n).astype(np.float32)
    zg, tg = on_gpu(z), on_gpu(t)
    s = check_score(dev, ops, zg, tg, scale=scale)
    grad = host(ops.token_logprobs_backward(dev, zg, tg, s.norm, s.entropy, on_gpu(g), on_gpu(h), scale=scale, out=torch.empty_like(zg)))

    def total(x):
        r = oracle.score(x, t, -1, scale, 0)
        return (g * r["logp"] + h * r["entropy"]).sum()
    e = 1e-4
    for i, j in itertools.product(range(n), range(v)):
        a, b = z.astype(np.float64), z.astype(np.float64)
        a[i, j] += e
        b[i, j] -= e
        assert abs((total(a) - total(b)) / (2 * e) - grad[i, j]) < 8 * 8 * e * e / 6 + 1e-10 / e + 2e-5


def check_distill(dev, ops, z, u, ids, temperature, weight, dtype, workspace=None):
    n, v = z.shape
    grad = torch.full((n, v + 3), 5.0, device="cuda", dtype=DT[dtype])
    out = ops.Distilled(torch.full((n,), 7.0, device="cuda"), torch.full((n, 2), 7.0, device="cuda"), grad[:, :v])
    w = None if weight is None else on_gpu(weight)
    ops.distill_loss(dev, z, u, ids, temperature=temperature, row_weight=w, grad=True, out=out, workspace=workspace)
    loss, loss_tol, norm, norm_tol, want, tol = oracle.distill(host(z), host(u), ids.cpu().numpy(), temperature, weight)
    close(host(out.loss), loss, loss_tol, "loss")
    close(host(out.norm), norm, norm_tol, "norm")
    close(host(out.grad), want, tol + oracle.rounding(dtype, want), "grad")
    assert bool((grad[:, v:] == 5.0).all())
    alone = ops.Distilled(torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda"), None)
    ops.distill_loss(dev, z, u, ids, temperature=temperature, out=alone, workspace=workspace)
    close(host(alone.loss), loss, loss_tol, "loss alone")                # (sums in another order than with the gradient)
    close(host(alone.norm), norm, norm_tol, "norm alone")
    later = ops.distill_loss_backward(dev, z, u, ids, out.norm, w, temperature=temperature, out=torch.full((n, v), 5.0, device="cuda", dtype=DT[dtype]))
    _, _, _, _, want, tol = oracle.distill(host(z), host(u), ids.cpu().numpy(), temperature, weight, norm=host(out.norm))
    close(host(later), want, tol + oracle.rounding(dtype, want), "later gradient")
    return out


DISTILL = [(1, 1, 1), (1, 5, 3), (3, 64, 7), (2, 1000, 100), (6, 2051, 1), (1, 50000, 40), (9, 9000, 257), (3, 1100, 1024), (1030, 97, 5)]
DISTILL_SHAPES = [("f32", 3, 16001, 30), ("f32", 520, 4001, 3), ("bf16", 520, 16003, 70), ("f32", 520, 32001, 5), ("f32", 3, 60001, 1024), ("bf16", 2, 131075, 65),
                  ("f32", 70, 70001, 20), ("f16", 2, 140003, 200), ("f32", 2, 140001, 20), ("bf16", 1, 300000, 300),
                  ("f16", 520, 1003, 8), ("bf16", 520, 3001, 9), ("f32", 520, 7001, 4), ("f16", 3, 196613, 1024), ("f32", 3, 98304, 9), ("f32", 70, 98410, 5), ("bf16", 2, 131079, 3)]


@pytest.mark.parametrize("dtype,n,v,k", DISTILL_SHAPES)
def test_distill_of_every_launch_shape(dev, ops, dtype, n, v, k):
    """Rows held by 64 to 1024 threads, rows read twice, rows in segments."""
    rng = np.random.default_rng(v + k)
    ids = rng.integers(0, v, (n, k))
    ids[:, k // 2:][rng.random((n, k - k // 2)) < 0.3] = v - 1                   # the last element, often
    check_distill(dev, ops, rows_of(n, v, dtype, seed=v), on_gpu(rng.normal(0, 3, (n, k)).astype(np.float32)), on_gpu(ids), 1.5, rng.random(n).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", DISTILL)
def test_distill(dev, ops, n, v, k, dtype):
    rng = np.random.default_rng(v + k)
    z = rows_of(n, v, dtype, seed=v + n, stride=v + 5)
    u = on_gpu(rng.normal(0, 3, (n, k)).astype(np.float32), dtype if v % 2 else None)
    ids = rng.integers(0, v, (n, k))                                   # a token may be named twice
    ids[rng.random((n, k)) < 0.2] = -1
    wide = on_gpu(np.concatenate([ids, ids], 1))
    check_distill(dev, ops, z, u, wide[:, :k] if k % 2 else wide[:, :k].int(), 2.0, rng.random(n).astype(np.float32), dtype)
    check_distill(dev, ops, z, u, on_gpu(ids), 1.0, None, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [40, 30000])
def test_distill_edges(dev, ops, v, dtype):
    """No entry, the same token everywhere, entries outside the vocabulary, a teacher's -infinity and
    lowest values, a student's masked rows."""
    rng = np.random.default_rng(v)
    k = 6
    low = float(torch.finfo(DT[dtype]).min)
    z, u, ids = rng.normal(0, 2, (10, v)).astype(np.float32), rng.normal(0, 2, (10, k)).astype(np.float32), rng.integers(0, v, (10, k))
    ids[0] = -1
    ids[1] = v - 1
    ids[2] = [v, -5, 2 ** 31 - 1, -2 ** 31, 3, v + 1]
    u[3, 2:] = -np.inf
    u[4] = -np.inf
    z[5] = -np.inf
    z[6] = -np.inf
    ids[6] = -1
    z[7, ids[7, 1]] = -np.inf
    z[8, ::2] = -np.inf
    ids[8] = np.arange(k) * 2 + 1
    gz, gu = on_gpu(z, dtype), on_gpu(u, dtype)
    gz[9] = low
    gu[2, 4] = low
    out = check_distill(dev, ops, gz, gu, on_gpu(ids), 1.5, rng.random(10).astype(np.float32), dtype)
    loss, grad = host(out.loss), host(out.grad)
    assert loss[0] == 0 and not grad[0].any() and loss[4] == 0 and not grad[4].any()
    assert loss[5] == np.inf and not grad[5].any() and loss[6] == 0 and not grad[6].any() and loss[7] == np.inf


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", [(6, 40), (6, 5003), (6, 60000), (6, 400007), (300, 200003)])
def test_distill_rows_without_entries_may_hold_anything(dev, ops, n, v, dtype):
    """Loss 0 and gradient 0, held in registers, in segments, and read twice: NaN, infinities, all of one kind."""
    z = rows_of(n, v, dtype, 5)
    ids = torch.full((n, 3), -1, device="cuda")
    ids[:, 1:] = torch.tensor([v, -7], device="cuda")
    ids[2] = torch.tensor([0, 1, 2], device="cuda")            # (no entry either: the teacher's logits are -infinity)
    ids[5] = torch.tensor([v - 1, 3, 3], device="cuda")        # the one row with entries
    u = on_gpu(np.random.default_rng(0).normal(0, 1, (n, 3)).astype(np.float32))
    u[2] = -np.inf
    z[0, v // 2] = np.nan
    z[1] = np.nan
    z[2, 1] = np.inf
    z[3] = np.inf
    z[4] = -np.inf
    weight = on_gpu(np.linspace(-1, 2, n).astype(np.float32))
    full = lambda *s, dt=torch.float32: torch.full(s, 7.0, device="cuda", dtype=dt)  # noqa: E731
    out = ops.Distilled(full(n), full(n, 2), full(n, v, dt=DT[dtype]))
    ops.distill_loss(dev, z, u, ids, temperature=1.5, row_weight=weight, grad=True, out=out)
    alone = ops.Distilled(full(n), full(n, 2), None)
    ops.distill_loss(dev, z, u, ids, temperature=1.5, out=alone)
    later = ops.distill_loss_backward(dev, z, u, ids, out.norm, weight, temperature=1.5, out=full(n, v, dt=DT[dtype]))
    none = [i for i in range(n) if i != 5]
    for loss in (out.loss, alone.loss):
        assert not host(loss)[none].any() and np.isfinite(host(loss)[5]) and host(loss)[5] != 0
    for grad, norm in ((out.grad, None), (later, host(out.norm[5:6]))):
        assert not bool(grad[none].any())
        want, tol = oracle.distill(host(z[5:6]), host(u[5:6]), ids[5:6].cpu().numpy(), 1.5, host(weight[5:6]), norm=norm)[4:]
        close(host(grad[5:6]), want, tol + oracle.rounding(dtype, want), "grad")


def test_distill_gradient_against_differences(dev, ops):
    """As for the scores; the third derivative of T^2 KL by a logit is below 1 / T."""
    rng = np.random.default_rng(2)
    n, v, k, temp = 3, 29, 5, 1.7
    z, u = rng.normal(0, 1.5, (n, v)).astype(np.float32), rng.normal(0, 2, (n, k)).astype(np.float32)
    ids = rng.integers(0, v, (n, k))
    ids[1, 2] = ids[1, 0]
    w = rng.random(n).astype(np.float32)
    out = check_distill(dev, ops, on_gpu(z), on_gpu(u), on_gpu(ids), temp, w, "f32")
    grad, e = host(out.grad), 1e-4

    def total(x):
        return (w * oracle.distill(x, u, ids, temp, None)[0]).sum()
    for i, j in itertools.product(range(n), range(v)):
        a, b = z.astype(np.float64), z.astype(np.float64)
        a[i, j] += e
        b[i, j] -= e
        assert abs((total(a) - total(b)) / (2 * e) - grad[i, j]) < e * e + 1e-10 / e + 2e-5


def sequences(b, t, d, dtype, seed, log_gate, layout="btd"):
    rng = np.random.default_rng(seed)
    lg = -np.minimum(np.exp(rng.normal(0, 1.2, (b, t, d)) - 3), 0.7).astype(np.float32)
    gate = (lg if log_gate else np.exp(lg)).astype(np.float32)
    arrays = [gate] + [rng.normal(0, 1, (b, t, d)).astype(np.float32) for _ in range(2)]
    out = []
    for a in arrays:
        if layout == "tbd":
            out.append(on_gpu(a.transpose(1, 0, 2), dtype).permute(1, 0, 2))
        elif layout == "wide":
            out.append(on_gpu(np.concatenate([a, a, a[..., :1]], 2), dtype)[:, :, d:2 * d])
        else:
            out.append(on_gpu(a, dtype))
    return out


def check_scan(dev, ops, b, t, d, dtype, log_gate, lengths=None, state=True, layout="btd", seed=0, ends=True):
    gate, x, grad_h = sequences(b, t, d, dtype, seed + b * t + d, log_gate, layout)
    rng = np.random.default_rng(seed)
    s = rng.normal(0, 2, (b, d)).astype(np.float32) if state else None
    gs = None if s is None else on_gpu(s)
    gl = None if lengths is None else on_gpu(np.asarray(lengths, np.int32))
    n = np.full(b, t) if lengths is None else np.clip(np.asarray(lengths), 0, t)
    for i in range(b):                                         # what lies behind a sequence is not looked at
        for a in (gate, x, grad_h):
            a[i, n[i]:] = float("nan")
    live = np.arange(t)[None, :, None] < n[:, None, None]

    def blank():
        base = torch.full((t, b, d) if layout == "tbd" else (b, t, 2 * d + 1), 3.0, device="cuda", dtype=DT[dtype])
        return base.permute(1, 0, 2) if layout == "tbd" else base[:, :, d:2 * d]
    out, final = blank(), torch.full((b, d), 9.0, device="cuda") if ends else None
    ops.gated_scan(dev, gate, x, state=gs, lengths=gl, log_gate=log_gate, out=out, final=final)
    clean = [np.where(live, host(a), 0.0) for a in (gate, x, grad_h)]
    h, tol, fin, fin_tol = oracle.scan(clean[0], clean[1], s, lengths, log_gate)
    close(np.where(live, host(out), 0), np.where(live, h, 0), np.where(live, tol + oracle.rounding(dtype, h), 0), "h")
    assert bool((out[torch.from_numpy(np.broadcast_to(~live, out.shape).copy()).cuda()] == 3.0).all())
    if ends:
        close(host(final), fin, fin_tol + oracle.rounding("f32", fin), "final")
    gf = rng.normal(0, 1, (b, d)).astype(np.float32) if ends else None
    grads = ops.ScanGrads(blank(), blank(), torch.full((b, d), 9.0, device="cuda") if state else None)
    ops.gated_scan_backward(dev, gate, out, grad_h, state=gs, lengths=gl, log_gate=log_gate, grad_final=None if gf is None else on_gpu(gf), out=grads)
    want, tols = oracle.scan_grad(clean[0], np.where(live, host(out), 0), clean[2], s, lengths, log_gate, gf)
    for name, got, w, tl in zip(("grad_gate", "grad_x"), grads[:2], want, tols):
        close(np.where(live, host(got), 0), w, tl + np.where(live, oracle.rounding(dtype, w), 0), name)
        assert bool((got[torch.from_numpy(np.broadcast_to(~live, got.shape).copy()).cuda()] == 3.0).all())
    if state:
        close(host(grads.grad_state), want[2], tols[2] + oracle.rounding("f32", want[2]), "grad_state")


SCANS = [(1, 1, 1), (3, 1, 64), (2, 2, 7), (1, 5, 65), (2, 63, 130), (3, 64, 8), (1, 129, 256), (2, 300, 33), (1, 1027, 96), (1, 5000, 24), (40, 17, 100)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,t,d", SCANS)
def test_scan(dev, ops, b, t, d, dtype):
    check_scan(dev, ops, b, t, d, dtype, log_gate=False)
    check_scan(dev, ops, b, t, d, dtype, log_gate=True, state=False, ends=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["tbd", "wide"])
def test_scan_layouts(dev, ops, layout, dtype):
    check_scan(dev, ops, 3, 200, 72, dtype, log_gate=True, layout=layout)
    check_scan(dev, ops, 2, 513, 41, dtype, log_gate=False, layout=layout)


@pytest.mark.parametrize("log_gate", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scan_last_channels(dev, ops, dtype, log_gate):
    """Rows that end inside a vector, in many workgroups at once: with every count of channels in the last one."""
    check_scan(dev, ops, 6, 1030, 717, dtype, log_gate, lengths=[1030, 1, 513, 1029, 700, 1030])
    check_scan(dev, ops, 16, 600, 717, dtype, log_gate)       # (more workgroups than the device runs one a compute unit)
    check_scan(dev, ops, 5, 1100, 1408, dtype, log_gate)
    check_scan(dev, ops, 2, 1021, 203, dtype, log_gate)
    for width in (65, 74, 83, 92, 102, 111):
        check_scan(dev, ops, 3, 530, width, dtype, log_gate)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [1, 8, 9, 16, 17, 31])
def test_scan_of_few_channels(dev, ops, width, dtype):
    """Rows of less than a cache line: more steps go to a workgroup, in one piece and in several."""
    check_scan(dev, ops, 9, 130, width, dtype, log_gate=True)
    check_scan(dev, ops, 2, 4300, width, dtype, log_gate=False, lengths=[4300, 2049])
    check_scan(dev, ops, 3, 1100, width, dtype, log_gate=True, layout="wide", state=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scan_lengths(dev, ops, dtype):
    """Sequences of no steps, one, all, and lengths outside the array; NaN behind them stays there."""
    check_scan(dev, ops, 7, 150, 48, dtype, log_gate=True, lengths=[0, 1, 150, 149, -3, 1000, 64])
    check_scan(dev, ops, 3, 700, 5, dtype, log_gate=False, lengths=[512, 0, 513], state=False)
    check_scan(dev, ops, 2, 1, 300, dtype, log_gate=False, lengths=[0, 1])


def test_scan_gates_of_zero_and_one(dev, ops):
    """A gate of exactly 0 (exp(-infinity)) forgets everything, a gate of 1 forgets nothing."""
    b, t, d = 2, 400, 9
    x = np.random.default_rng(0).normal(0, 1, (b, t, d)).astype(np.float32)
    lg = np.zeros((b, t, d), np.float32)
    lg[0, ::50] = -np.inf
    for log_gate in (True, False):
        g = lg if log_gate else np.exp(lg)
        out = ops.gated_scan(dev, on_gpu(g), on_gpu(x), log_gate=log_gate, out=torch.empty(b, t, d, device="cuda"))
        h, tol, _, _ = oracle.scan(g, x, None, None, log_gate)
        close(host(out), h, tol, "h")


def test_scan_in_pieces(dev, ops):
    """A prompt in one call, then token by token with the state handed on, gives the states of one long call."""
    b, t, d = 3, 40, 70
    gate, x, _ = sequences(b, t, d, "f32", 11, True)
    whole = ops.gated_scan(dev, gate, x, log_gate=True, out=torch.empty_like(x))
    state, got = torch.zeros(b, d, device="cuda"), []
    for lo, hi in [(0, 33)] + [(i, i + 1) for i in range(33, 40)]:
        nxt = torch.empty(b, d, device="cuda")
        got.append(ops.gated_scan(dev, gate[:, lo:hi], x[:, lo:hi], state=state, log_gate=True, out=torch.empty(b, hi - lo, d, device="cuda"), final=nxt))
        state = nxt
    h, tol, fin, fin_tol = oracle.scan(host(gate), host(x), None, None, True)
    close(host(torch.cat(got, 1)), h, tol, "pieces")
    close(host(whole), h, tol, "whole")
    close(host(state), fin, fin_tol, "state")


def test_scan_gradient_against_differences(dev, ops):
    """The sum of the outputs is linear in every single gate and input: central differences of it are exact but
    for rounding (1e-13 of sums of about 1e2, over the step)."""
    rng = np.random.default_rng(4)
    b, t, d = 1, 9, 2
    gate, x = rng.uniform(0.3, 0.99, (b, t, d)).astype(np.float32), rng.normal(0, 1, (b, t, d)).astype(np.float32)
    s, w = rng.normal(0, 1, (b, d)).astype(np.float32), rng.normal(0, 1, (b, t, d)).astype(np.float32)
    gg, gx, gs = on_gpu(gate), on_gpu(x), on_gpu(s)
    h = ops.gated_scan(dev, gg, gx, state=gs, out=torch.empty_like(gx))
    got = ops.gated_scan_backward(dev, gg, h, on_gpu(w), state=gs, out=ops.ScanGrads(torch.empty_like(gx), torch.empty_like(gx), torch.empty_like(gs)))

    def total(g, v, s0):
        return (w * oracle.scan(g, v, s0, None, False)[0]).sum()
    base = [gate.astype(np.float64), x.astype(np.float64), s.astype(np.float64)]
    for k, grad in enumerate(got):
        for at in np.ndindex(base[k].shape):
            hi, lo = [v.copy() for v in base], [v.copy() for v in base]
            hi[k][at] += 1e-3
            lo[k][at] -= 1e-3
            assert abs((total(*hi) - total(*lo)) / 2e-3 - host(grad)[at]) < 1e-8 + 200 * oracle.U * 50


# ---- how calls are made ------------------------------------------------------------------------------


def test_results_as_buffers(ops):
    """Arrays of the library's own on a handle with its own stream; outputs allocated by the call."""
    from harp_amd import backend as hb
    from harp_amd.frontend import F32, I32
    d = hb.HipDevice(0)
    rng = np.random.default_rng(0)
    z, t = rng.normal(0, 2, (6, 900)).astype(np.float32), rng.integers(0, 900, 6).astype(np.int32)
    bz, bt = hb.HipBuffer(d, [6, 900], F32), hb.HipBuffer(d, [6], I32)
    bz.write_array(z)
    bt.write_array(t)
    out = ops.token_logprobs(d, bz, bt, top=4)
    want = oracle.score(z, t, -1, 1.0, 4)
    close(out.logp.read_array(np.float32), want["logp"], want["logp_tol"], "logp")
    assert np.array_equal(out.top_ids.read_array(np.int32, (6, 4)), want["top_ids"])
    # a view into the middle of a larger buffer: rows 1 to 4, columns 100 on
    part = ops.View(bz, [4, 700], F32, offset=4 * (900 + 100), strides=[900, 1])
    lp = hb.HipBuffer(d, [10], F32)
    lp.write_array(np.full(10, 5, np.float32))
    ops.token_logprobs(d, part, ops.View(bt, [4], I32, offset=0), scale=2.0, out=ops.Logprobs(ops.View(lp, [4], F32, offset=12), None, hb.HipBuffer(d, [4, 2], F32), None, None))
    want = oracle.score(z[1:5, 100:800], np.where(t[:4] < 700, t[:4], -2), -1, 2.0, 0)
    got = lp.read_array(np.float32)
    close(got[3:7], want["logp"], want["logp_tol"], "logp")
    assert (got[[0, 1, 2, 7, 8, 9]] == 5).all()
    g = rng.uniform(0, 1, (2, 50, 12)).astype(np.float32)
    bg, bx = hb.HipBuffer(d, [2, 50, 12], F32), hb.HipBuffer(d, [2, 50, 12], F32)
    bg.write_array(g)
    bx.write_array(g)
    h = ops.gated_scan(d, bg, bx)
    want, tol, _, _ = oracle.scan(g, g, None, None, False)
    close(h.read_array(np.float32, (2, 50, 12)), want, tol, "h")
    # an output nothing has written yet, of which the call writes a part: the rest reads as zeros
    lens = hb.HipBuffer(d, [2], I32)
    lens.write_array(np.array([50, 20], np.int32))
    h = ops.gated_scan(d, bg, bx, lengths=lens).read_array(np.float32, (2, 50, 12))
    assert not h[1, 20:].any() and h[1, :20].any()


def test_no_rows_and_no_steps(dev, ops):
    z = torch.empty(0, 50, device="cuda")
    none = torch.empty(0, device="cuda")
    ops.token_logprobs(dev, z, none.long(), out=ops.Logprobs(none, None, torch.empty(0, 2, device="cuda"), None, None))
    ops.token_logprobs_backward(dev, z, none.long(), torch.empty(0, 2, device="cuda"), out=torch.empty_like(z))
    ops.distill_loss(dev, z, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, device="cuda").int(), grad=True,
                     out=ops.Distilled(none, torch.empty(0, 2, device="cuda"), torch.empty_like(z)))
    g, s, f = torch.empty(2, 0, 5, device="cuda"), torch.randn(2, 5, device="cuda"), torch.empty(2, 5, device="cuda")
    ops.gated_scan(dev, g, g, state=s, out=g, final=f)
    assert torch.equal(f, s)
    e = torch.randn(2, 5, device="cuda")
    ops.gated_scan_backward(dev, g, g, g, state=s, grad_final=e, out=ops.ScanGrads(g, g, f))
    assert torch.equal(f, e)
    torch.cuda.synchronize()


def _all_calls(dev, ops, seed, n=5, v=270000, k=9, b=2, t=1300, d=40):
    """One call of each operator on inputs of the seed: (a function that runs them, their outputs, workspaces)."""
    rng = np.random.default_rng(seed)
    z = rows_of(n, v, "bf16", seed)
    ids, u = on_gpu(rng.integers(0, v, (n, k))), on_gpu(rng.normal(0, 2, (n, k)).astype(np.float32))
    tg = ids[:, 0].contiguous()
    gate, x, gh = sequences(b, t, d, "f32", seed, True)
    e = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    sc = ops.Logprobs(e(n), e(n), e(n, 2), e(n, 6), e(n, 6, dt=torch.int32))
    di = ops.Distilled(e(n), e(n, 2), torch.zeros_like(z))
    sg, h, fin = torch.zeros_like(z), torch.zeros_like(x), e(b, d)
    gr = ops.ScanGrads(torch.zeros_like(x), torch.zeros_like(x), None)
    ones = torch.ones(n, device="cuda")
    ws = [torch.empty(max(nb, 1), device="cuda", dtype=torch.uint8) for nb in (
        ops.token_logprobs_workspace(dev, z, top=6), ops.distill_loss_workspace(dev, z), ops.gated_scan_workspace(dev, gate),
        ops.gated_scan_backward_workspace(dev, gate))]

    def go(handle, given=True):
        w = ws if given else [None] * 4
        ops.token_logprobs(handle, z, tg, top=6, out=sc, workspace=w[0])
        ops.token_logprobs_backward(handle, z, tg, sc.norm, sc.entropy, ones, ones, out=sg)
        ops.distill_loss(handle, z, u, ids, grad=True, out=di, workspace=w[1])
        ops.gated_scan(handle, gate, x, log_gate=True, out=h, final=fin, workspace=w[2])
        ops.gated_scan_backward(handle, gate, h, gh, log_gate=True, out=gr, workspace=w[3])
    outs = [*sc, sg, *di, h, fin, gr.grad_gate, gr.grad_x]
    return go, outs


def test_same_bits_every_time(dev, ops):
    go, outs = _all_calls(dev, ops, 3)
    go(dev)
    first = [o.clone() for o in outs]
    for given in (True, False, True):
        for o in outs:
            o.fill_(7)
        go(dev, given)
        for a, b in zip(first, outs):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(dev, ops):
    """Two handles on streams of their own, workspaces from each handle's pool, calls interleaved."""
    from harp_amd import backend as hb
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    handles = [hb.HipDevice(0, stream=s.cuda_stream) for s in streams]
    calls = [_all_calls(dev, ops, 21), _all_calls(dev, ops, 22)]
    want = []
    for go, outs in calls:
        go(dev)
        want.append([o.clone() for o in outs])
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for h, (go, _) in zip(handles, calls):
            go(h, given=False)
    torch.cuda.synchronize()
    for (_, outs), w in zip(calls, want):
        for a, b in zip(outs, w):
            assert torch.equal(a, b)


def test_captured_and_replayed(ops):
    """All operators in one graph of the caller's, replayed between eager work on the same stream; every replay is
    checked against the eager results of the inputs it finds."""
    from harp_amd import backend as hb
    s = torch.cuda.Stream()
    h = hb.HipDevice(0, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        go, outs = _all_calls(h, ops, 31)
        go2, outs2 = _all_calls(h, ops, 32)
        go(h)
        want = [o.clone() for o in outs]
        go2(h)
        want2 = [o.clone() for o in outs2]
    torch.cuda.synchronize()
    graphs = []
    for g in (go, go2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            g(h)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(s):
            for o in outs + outs2:
                o.fill_(7)
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs + outs2, want + want2):
            assert torch.equal(a, b)


def test_capture_needs_the_callers_workspace(ops):
    from harp_amd import backend as hb
    from harp_amd._lib import EhError
    s = torch.cuda.Stream()
    h = hb.HipDevice(0, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        z = torch.randn(2, 300000, device="cuda")
        t = torch.zeros(2, device="cuda", dtype=torch.int64)
        out = ops.Logprobs(torch.empty(2, device="cuda"), None, torch.empty(2, 2, device="cuda"), None, None)
        assert ops.token_logprobs_workspace(h, z) > 0
        small = torch.empty(8, device="cuda", dtype=torch.uint8)
        ok = torch.empty(2, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        with pytest.raises(EhError, match="workspace"):
            ops.token_logprobs(h, z, t, out=out)
        with pytest.raises(EhError, match="workspace"):
            ops.token_logprobs(h, z, t, out=out, workspace=small)
        ok.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((ok == 1).all())


def test_the_current_device_and_stream_stay(dev, ops):
    before = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    check_score(dev, ops, rows_of(2, 100, "f32", 0), on_gpu(np.zeros(2, np.int64)))
    assert (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream) == before


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_far_apart_in_a_large_array(dev, ops, dtype):
    """Offsets beyond 2^32 bytes (and, in bf16, beyond 2^31 elements)."""
    stride = 1_300_000_000
    base = torch.zeros(2 * stride + 5000, device="cuda", dtype=DT[dtype])
    z = base.as_strided((3, 4999), (stride, 1))
    z.copy_(rows_of(3, 4999, dtype, 9))
    check_score(dev, ops, z, on_gpu(np.array([0, 4998, 77])), top=3)
    seq = base.as_strided((1, 3, 600), (0, stride, 1))
    out = ops.gated_scan(dev, torch.full((1, 3, 600), 0.5, device="cuda", dtype=DT[dtype]), seq, out=torch.empty(1, 3, 600, device="cuda", dtype=DT[dtype]))
    h, tol, _, _ = oracle.scan(np.full((1, 3, 600), 0.5), host(seq), None, None, False)
    close(host(out), h, tol + oracle.rounding(dtype, h), "h")


def test_an_earlier_calls_error_is_reported_once(dev, ops):
    """A refused call of HIP leaves its error with the thread: neither an operator nor another library takes it for its own."""
    from harp_amd import backend as hb
    from harp_amd import frontend as fe
    a = fe.Tensor.input([256])
    blob = hb.HipKernel(dev, fe.lower_graph([(a * a).graph])[0]).get_binary()
    z, t = rows_of(4, 30, "f32", 0), on_gpu(np.array([1, 2, 3, 4]))
    for after in (lambda: check_score(dev, ops, z, t), lambda: torch.ones(3, device="cuda").sum().item()):
        with pytest.raises(hb.EhError):
            hb.HipModule(dev, blob, "no_such_entry")
        after()


def test_gradients_of_more_vectors_than_a_launch_has_threads(dev, ops):
    """2^32 vectors and more of one gradient (69 GB, of a row that all share): every row has the same."""
    n, v = 262150, 131072
    row = rows_of(1, v, "bf16", 4)
    z, out = row.expand(n, v), torch.empty(n, v, device="cuda", dtype=torch.bfloat16)
    t = torch.full((1,), 77, device="cuda")
    score = ops.Logprobs(*(torch.empty(1, device="cuda") for _ in range(2)), torch.empty(1, 2, device="cuda"), None, None)
    ops.token_logprobs(dev, row, t, out=score)
    e = torch.full((n,), 0.5, device="cuda")
    one = torch.empty(1, v, device="cuda", dtype=torch.bfloat16)

    def same(want):
        assert not bool(torch.isnan(want).any())
        for lo in range(0, n, 8192):
            assert bool((out[lo:lo + 8192] == want).all()), lo
        out.fill_(float("nan"))
    ops.token_logprobs_backward(dev, row, t, score.norm, score.entropy, e[:1], e[:1], out=one)
    ops.token_logprobs_backward(dev, z, t.expand(n).contiguous(), score.norm.expand(n, 2).contiguous(), score.entropy.expand(n).contiguous(), e, e, out=out)
    same(one)
    u, ids = torch.zeros(1, 2, device="cuda"), torch.tensor([[5, v - 1]], device="cuda")
    loss = ops.Distilled(torch.empty(1, device="cuda"), torch.empty(1, 2, device="cuda"), None)
    ops.distill_loss(dev, row, u, ids, out=loss)
    ops.distill_loss_backward(dev, row, u, ids, loss.norm, out=one)
    ops.distill_loss_backward(dev, z, u.expand(n, 2), ids.expand(n, 2), loss.norm.expand(n, 2).contiguous(), out=out)
    same(one)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_few_channels_with_steps_far_apart(dev, ops, dtype):
    """Steps of megabytes, so that a piece reaches beyond 32-bit offsets, in the workspace that was asked for."""
    t, d, step = (2500, 8, 1_200_000) if dtype == "f16" else (1000, 64, 2_100_000)
    base = torch.zeros(t * step + 1000, device="cuda", dtype=DT[dtype])
    gate, x, gh = sequences(1, t, d, dtype, 3, True)
    far = [base[i * 64:].as_strided((1, t, d), (0, step, 1)) for i in range(6)]
    for a, b in zip(far, (gate, x, gh)):
        a.copy_(b)
    h, gg, gx = far[3:]
    ws = torch.empty(ops.gated_scan_workspace(dev, gate), device="cuda", dtype=torch.uint8)
    ops.gated_scan(dev, far[0], far[1], log_gate=True, out=h, workspace=ws)
    want, tol, _, _ = oracle.scan(host(gate), host(x), None, None, True)
    close(host(h), want, tol + oracle.rounding(dtype, want), "h")
    ws = torch.empty(ops.gated_scan_backward_workspace(dev, gate), device="cuda", dtype=torch.uint8)
    ops.gated_scan_backward(dev, far[0], h, far[2], log_gate=True, out=ops.ScanGrads(gg, gx, None), workspace=ws)
    want, tols = oracle.scan_grad(host(gate), host(h), host(gh), None, None, True, None)
    for name, got, w, tl in zip(("grad_gate", "grad_x"), (gg, gx), want, tols):
        close(host(got), w, tl + oracle.rounding(dtype, w), name)


def test_a_wait_given_up_is_reported(dev, ops, monkeypatch):
    """A scan whose first piece is left out (by the host), so that the others wait for it in vain: the call ends, what
    follows is NaN, and the handle says so once, wherever it next waits or scans."""
    from harp_amd import backend as hb
    from harp_amd.frontend import F32
    gate, x, grad_h = sequences(1, 2000, 64, "f32", 5, True)
    h, fin = torch.zeros_like(x), torch.zeros(1, 64, device="cuda")
    monkeypatch.setenv("ECLAT_HIP_LOSE_WAITS", "1")
    mine = hb.HipDevice(0, stream=torch.cuda.current_stream().cuda_stream)
    monkeypatch.delenv("ECLAT_HIP_LOSE_WAITS")
    some = hb.HipBuffer(mine, [4], F32)
    some.write_array(np.zeros(4, np.float32))

    def scan():
        ops.gated_scan(mine, gate, x, log_gate=True, out=h, final=fin)

    def back():
        ops.gated_scan_backward(mine, gate, x, grad_h, log_gate=True, out=ops.ScanGrads(torch.empty_like(x), h, fin))
    scan()
    with pytest.raises(hb.EhError, match="in vain"):
        mine.sync()
    mine.sync()
    assert not bool(h[:, :512].any()) and bool(torch.isnan(h[:, 512:]).all()) and bool(torch.isnan(fin).all())
    back()
    with pytest.raises(hb.EhError, match="in vain"):
        some.read_array(np.float32)
    some.read_array(np.float32)
    assert bool(torch.isnan(h[:, :1536]).all()) and bool(torch.isnan(fin).all())
    for call in (scan, back):                                      # and the next scan is not queued
        scan()
        torch.cuda.synchronize()
        h.zero_()
        with pytest.raises(hb.EhError, match="in vain"):
            call()
        mine.sync()
        assert not bool(h.any())
    # another handle has lost nothing, nor does NaN in the data look like a lost wait, whatever its bits
    x.view(torch.int32)[0, 3, :7] = -1
    ops.gated_scan(dev, gate, x, log_gate=True, out=h, final=fin)
    dev.sync()
    assert bool(torch.isnan(fin[0, :7]).all())
    want, tol, _, _ = oracle.scan(host(gate), np.nan_to_num(host(x)), None, None, True)
    close(host(h)[..., 7:], want[..., 7:], tol[..., 7:], "h")
    ops.gated_scan(dev, gate, x, state=x[:, 3].contiguous(), log_gate=True, out=h, final=fin)
    dev.sync()


REFUSED = [
    ("overlap", lambda o, d, z, t, e: o.token_logprobs_backward(d, z, t, e(4, 2), out=z)),
    ("overlap", lambda o, d, z, t, e: o.gated_scan(d, z[None], z[None], out=z[None])),
    ("overlap", lambda o, d, z, t, e: o.gated_scan(d, z[None], z[None], out=e(1, 1, 100).expand(1, 4, 100))),
    ("overlap", lambda o, d, z, t, e: o.gated_scan(d, z[None], z[None], out=e(500).as_strided((2, 2, 100), (150, 60, 1))[:, :, :100].reshape(1, 4, 100) if False else e(500).as_strided((1, 4, 100), (0, 60, 1)))),
    ("out of range", lambda o, d, z, t, e: o.token_logprobs(d, z, t, top=33)),
    ("out of range", lambda o, d, z, t, e: o.token_logprobs(d, z[:, :3], t, top=4)),
    ("positive", lambda o, d, z, t, e: o.token_logprobs(d, z, t, scale=0.0)),
    ("positive", lambda o, d, z, t, e: o.token_logprobs(d, z, t, scale=float("nan"))),
    ("positive", lambda o, d, z, t, e: o.distill_loss(d, z, z[:, :3], t[:, None].expand(4, 3).contiguous(), temperature=-1.0)),
    ("out of range", lambda o, d, z, t, e: o.distill_loss(d, e(4, 2000), e(4, 1025), torch.zeros(4, 1025, device="cuda", dtype=torch.int32))),
    ("type", lambda o, d, z, t, e: o.gated_scan(d, z[None], z[None].half(), out=e(1, 4, 100))),
    ("shape", lambda o, d, z, t, e: o.token_logprobs(d, z, t[:3])),
    ("host", lambda o, d, z, t, e: o.token_logprobs(d, z.cpu(), t)),
    ("contiguous", lambda o, d, z, t, e: o.token_logprobs(d, z.t(), torch.zeros(100, device="cuda", dtype=torch.int64))),
    ("f32, bf16", lambda o, d, z, t, e: o.token_logprobs(d, z.long(), t)),
    ("i32 or i64", lambda o, d, z, t, e: o.token_logprobs(d, z, z[:, 0].contiguous())),
]


@pytest.mark.parametrize("which", range(len(REFUSED)))
def test_refusals_leave_the_device_usable(dev, ops, which):
    """What the host can see is refused before anything is queued (the checks themselves run without a GPU in
    test_operators_host.py); the next call works."""
    word, call = REFUSED[which]
    z, t = rows_of(4, 100, "f32", 1), torch.zeros(4, device="cuda", dtype=torch.int64)
    with pytest.raises(Exception, match=word):
        call(ops, dev, z, t, lambda *s: torch.empty(*s, device="cuda"))
    check_score(dev, ops, z, t, top=2)
