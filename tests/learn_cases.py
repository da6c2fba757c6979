"""Cases of the language-model training operators at the level of the `fusion` module,
against 64-bit numpy (learn_oracle): tests/test_learn_cpu.py runs them over the host-memory
double of the C ABI, tests/test_learn_gpu.py over the kernels.

Tolerances (u = 2^-24, the largest relative error of one fp32 rounding): a case's values
are chains of at most a few hundred roundings with results of order one, and none cancels
by more than a factor of ~10 below the largest term; TOL = 1e-5 = 168 u relative to the
largest value of the array holds that chain and is what the framework's GEMM, which the
model case runs through, is held to."""
import numpy as np
import pytest

import learn_oracle as O

TOL = 1e-5


def dev(F):
    return F.CppDevice(F.CppDeviceType.CPU, 0)


def T(F, a, grad=False):
    a = np.ascontiguousarray(a, np.float32)
    return F.Tensor(list(a.shape), a.ravel(), F.CppDType.FLOAT32, dev(F), grad)


def near(got, want, what, tol=TOL, scale=None):
    got = got if isinstance(got, np.ndarray) else got.to_numpy()
    assert got.shape == want.shape, f"{what}: {got.shape} != {want.shape}"
    scale = max(np.abs(want).max(initial=0.0) if scale is None else scale, 1e-30)
    err = np.abs(got.astype(np.float64) - want).max(initial=0.0)
    assert err <= tol * scale, f"{what}: off by {err / scale:.3g} of the largest value"


def up(F, y, g):
    """A scalar whose gradient with respect to y is g."""
    return (y * T(F, g)).sum()


def group_norm(F):
    rng = np.random.default_rng(1)
    for shape, groups, act in [((3, 5, 7, 12), 4, "silu"), ((4, 10), 2, "gelu"), ((2, 3, 6), 6, "none"),
                               ((5, 4, 8), 1, "relu")]:
        x, g = rng.standard_normal(shape) * 2 + 1, rng.standard_normal(shape)
        ga, be = 1 + 0.3 * rng.standard_normal(shape[-1]), 0.2 * rng.standard_normal(shape[-1])
        x, g, ga, be = (a.astype(np.float32) for a in (x, g, ga, be))
        flat = (shape[0], int(np.prod(shape[1:-1])), shape[-1])
        y, _, _, dx, dg, db = O.group_norm(x.reshape(flat), ga, be, groups, 1e-5, act, g.reshape(flat))
        tx, tg, tb = T(F, x, True), T(F, ga, True), T(F, be, True)
        with F.grad_tape():
            out = F.group_norm(tx, groups, tg, tb, activation=act)
            up(F, out, g).backward()
        near(out, y.reshape(shape), "y")
        near(tx.get_grad(), dx.reshape(shape), "dx")
        near(tg.get_grad(), dg, "dgamma")
        near(tb.get_grad(), db, "dbeta")
        # without gamma and beta, and untraced
        y, _, _, dx, _, _ = O.group_norm(x.reshape(flat), None, None, groups, 1e-3, act, g.reshape(flat))
        tx = T(F, x, True)
        with F.grad_tape():
            up(F, F.group_norm(tx, groups, eps=1e-3, activation=act), g).backward()
        near(tx.get_grad(), dx.reshape(shape), "dx plain")
        near(F.group_norm(T(F, x), groups, eps=1e-3, activation=act), y.reshape(shape), "y plain")


def group_norm_only_parameters(F):
    """x needs no gradient: gamma's and beta's are still right."""
    rng = np.random.default_rng(2)
    x, g = rng.standard_normal((6, 8)).astype(np.float32), rng.standard_normal((6, 8)).astype(np.float32)
    ga, be = rng.standard_normal(8).astype(np.float32), rng.standard_normal(8).astype(np.float32)
    tg, tb = T(F, ga, True), T(F, be, True)
    with F.grad_tape():
        up(F, F.group_norm(T(F, x), 2, tg, tb), g).backward()
    _, _, _, _, dg, db = O.group_norm(x[:, None], ga, be, 2, 1e-5, "none", g[:, None])
    near(tg.get_grad(), dg, "dgamma")
    near(tb.get_grad(), db, "dbeta")


def saved_values_survive_writes(F):
    """An in-place update between forward and backward leaves the gradient at the values
    that the forward read."""
    rng = np.random.default_rng(3)
    x, g = rng.standard_normal((4, 6)).astype(np.float32), rng.standard_normal((4, 6)).astype(np.float32)
    ga, be = np.ones(6, np.float32) * 2, np.zeros(6, np.float32)
    tx, tg, tb = T(F, x, True), T(F, ga, True), T(F, be, True)
    with F.grad_tape():
        loss = up(F, F.group_norm(tx, 3, tg, tb), g)
        tg -= T(F, np.ones(6))
        tx -= T(F, x)
        loss.backward()
    _, _, rstd, dx, _, _ = O.group_norm(x[:, None], ga, be, 3, 1e-5, "none", g[:, None])
    # Two values a group: xh = +-s with 1 - s^2 = eps / (var + eps), so dx = rstd (a - mean a
    # - xh mean(a xh)) leaves only a (1 - s^2) of terms of size rstd |a|, a = dy gamma. The
    # terms carry the roundings of mean, rstd (stored in fp32: xh is off by u (|mean| + |x|)
    # rstd), of xh, of the products and the differences: fewer than 16 u of rstd |a| (1 +
    # rstd |x|), which is what the gradient can be held to.
    terms = np.repeat(rstd, 2, axis=1) * np.abs(g * ga) * (1 + np.repeat(rstd, 2, axis=1) * np.abs(x))
    near(tx.get_grad(), dx[:, 0], "dx", tol=16 * 2.0 ** -24, scale=terms.max())


def route(F):
    rng = np.random.default_rng(4)
    for shape, k, renorm in [((7, 9), 3, True), ((2, 3, 40), 4, False), ((5, 1), 1, True), ((6,), 6, False)]:
        z = rng.standard_normal(shape).astype(np.float32) * 2
        flat = z.reshape(-1, shape[-1])
        dw = rng.standard_normal((len(flat), k)).astype(np.float32)
        w, ids, dz = O.route(flat, k, renorm, dw)
        tz = T(F, z, True)
        with F.grad_tape():
            tw, ti = F.route(tz, k, renormalize=renorm)
            up(F, tw, dw.reshape(tw.shape)).backward()
        assert ti.to_numpy().shape == tuple(shape[:-1]) + (k,)
        np.testing.assert_array_equal(ti.to_numpy().reshape(-1, k), ids)
        near(tw.to_numpy().reshape(-1, k), w, "weights")
        # each entry of dlogits is a difference of at most two terms of order max |dw|
        err = np.abs(tz.get_grad().to_numpy().reshape(-1, shape[-1]) - dz).max()
        assert err <= TOL * np.abs(dw).max(), err


def route_masked(F):
    z = np.array([[1, 1, 1, 0], [-np.inf] * 4, [-np.inf, 2, -np.inf, 2], [3, -np.inf, -np.inf, -np.inf]], np.float32)
    w, ids = F.route(T(F, z), 2)
    np.testing.assert_array_equal(ids.to_numpy(), [[0, 1], [-1, -1], [1, 3], [0, -1]])
    np.testing.assert_array_equal(w.to_numpy(), np.float32([[0.5, 0.5], [0, 0], [0.5, 0.5], [1, 0]]))


def plan(F):
    rng = np.random.default_rng(5)
    for t, k, e, cap in [(9, 2, 4, 0), (9, 2, 4, 3), (1, 1, 1, 0), (20, 3, 5, 20), (0, 2, 3, 0), (0, 2, 3, 2)]:
        ids = rng.integers(-1, e + 1, (t, k))
        p = F.ExpertPlan(F.Indices(ids), e, cap)
        slot, src, counts, offsets = O.expert_sort(ids, e, cap)
        np.testing.assert_array_equal(p.slot.to_numpy(), slot)
        np.testing.assert_array_equal(p.src.to_numpy(), src)
        np.testing.assert_array_equal(p.counts.to_numpy(), counts)
        np.testing.assert_array_equal(p.offsets.to_numpy(), offsets)
        assert (p.tokens, p.k, p.experts, p.capacity, p.rows) == (t, k, e, cap, len(src))


def dispatch_and_combine(F):
    rng = np.random.default_rng(6)
    for lead, k, e, cap, width in [((9,), 2, 4, 0, 5), ((3, 4), 2, 4, 4, 8), ((6,), 1, 3, 1, 4)]:
        t = int(np.prod(lead))
        ids = rng.integers(-1, e, lead + (k,))
        p = F.ExpertPlan(F.Indices(ids), e, cap)
        slot, src, _, _ = O.expert_sort(ids.reshape(t, k), e, cap)
        x = rng.standard_normal(lead + (width,)).astype(np.float32)
        w = rng.uniform(0.1, 1, lead + (k,)).astype(np.float32)
        g = rng.standard_normal(lead + (width,)).astype(np.float32)
        rows = O.dispatch(x.reshape(t, width), slot, len(src))
        scale = rng.standard_normal(rows.shape).astype(np.float32)
        out, drows, dw = O.combine(rows * scale, w.reshape(t, k), slot, g.reshape(t, width))
        dx = O.combine(drows * scale, None, slot)
        tx, tw = T(F, x, True), T(F, w, True)
        with F.grad_tape():
            r = F.expert_dispatch(tx, p)
            assert r.shape == ([e, cap, width] if cap else [len(src), width])
            y = F.expert_combine(r * T(F, scale.reshape(r.shape)), p, tw)
            assert y.shape == list(lead) + [width]
            up(F, y, g).backward()
        np.testing.assert_array_equal(r.to_numpy().reshape(rows.shape), rows.astype(np.float32))
        near(y, out.reshape(g.shape), "out")
        near(tw.get_grad(), dw.reshape(w.shape), "dw")
        near(tx.get_grad(), dx.reshape(x.shape), "dx")
        # no weights: the gradient of the sum
        tr = T(F, rows, True)
        with F.grad_tape():
            y = F.expert_combine(tr, p)
            up(F, y, g).backward()
        out, drows, _ = O.combine(rows, None, slot, g.reshape(t, width))
        near(y, out.reshape(g.shape), "sum")
        near(tr.get_grad(), drows, "drows of the sum")


def distill(F):
    rng = np.random.default_rng(7)
    for lead, v, k, tau, tail in [((6,), 50, 4, 2.0, False), ((2, 3), 50, 4, 1.0, True), ((), 17, 17, 1.0, False),
                                  ((5,), 300, 9, 0.5, True)]:
        r = int(np.prod(lead))
        z = rng.standard_normal(lead + (v,)).astype(np.float32) * 2
        ids = np.stack([rng.permutation(v)[:k] for _ in range(r)])
        t = -np.sort(-rng.standard_normal((r, k)).astype(np.float32) * 2)
        if r > 1:
            ids[0, k // 2:] = -1  # a short list
            ids[1] = v            # none
        lse = None
        if tail:
            inside = np.where((ids >= 0) & (ids < v), np.exp(t.astype(np.float64) / tau), 0).sum(1)
            lse = np.log(np.maximum(inside, 1e-3) / 0.7).astype(np.float32)
        g = rng.uniform(0.5, 1, max(r, 1)).astype(np.float32)
        loss, dz = O.distill(z.reshape(r, v), ids, t, tau, lse, g)
        tz = T(F, z, True)
        with F.grad_tape():
            out = F.distill(tz, F.Indices(ids.reshape(lead + (k,))), T(F, t.reshape(lead + (k,))), temperature=tau,
                            teacher_lse=None if lse is None else T(F, lse))
            assert out.shape == (list(lead) or [1])
            up(F, out, g.reshape(out.shape)).backward()
        near(out, loss.reshape(out.shape), "loss")
        near(tz.get_grad(), dz.reshape(z.shape), "dz")


def model_step(F, tol=TOL):
    """A training step of a small mixture-of-experts model: norm, router, experts, vocabulary,
    distillation, all gradients against numpy's."""
    rng = np.random.default_rng(8)
    t, d, h, e, k, cap, v, n, groups = 40, 16, 24, 4, 2, 24, 60, 5, 4
    shapes = {"gamma": (d,), "beta": (d,), "wr": (d, e), "w1": (e, d, h), "w2": (e, h, d), "wo": (d, v)}
    W = {a: (rng.standard_normal(s) * (0.4 if len(s) > 1 else 0.2) + (a == "gamma")).astype(np.float32)
         for a, s in shapes.items()}
    x = rng.standard_normal((t, d)).astype(np.float32)
    ids = np.stack([rng.permutation(v)[:n] for _ in range(t)])
    teach = -np.sort(-rng.standard_normal((t, n)).astype(np.float32))
    tau, g = 2.0, np.full(t, 1.0 / t, np.float32)

    P = {a: T(F, w, True) for a, w in W.items()}
    with F.grad_tape():
        xn = F.group_norm(T(F, x), groups, P["gamma"], P["beta"], activation="silu")
        w, chosen = F.route(xn @ P["wr"], k)
        p = F.ExpertPlan(chosen, e, cap)
        rows = F.expert_dispatch(xn, p)
        hidden = rows @ P["w1"]
        hidden = hidden * hidden
        y = F.expert_combine(hidden @ P["w2"], p, w)
        loss = F.distill(y @ P["wo"], F.Indices(ids), T(F, teach), temperature=tau)
        up(F, loss, g).backward()

    f = {a: b.astype(np.float64) for a, b in W.items()}
    xn64 = O.group_norm(x[:, None], W["gamma"], W["beta"], groups, 1e-5, "silu")[0][:, 0]
    zr = xn64 @ f["wr"]
    w64, cho = O.route(zr, k, True)
    # the routing is decided by margins far above the errors of the logits
    srt = -np.sort(-zr, axis=1)
    assert (srt[:, k - 1] - srt[:, k]).min() > 1e-3
    np.testing.assert_array_equal(chosen.to_numpy(), cho)
    slot, src, counts, _ = O.expert_sort(cho, e, cap)
    assert counts.max() > cap - 8  # the capacity is nearly used up
    rows64 = O.dispatch(xn64, slot, e * cap).reshape(e, cap, d)
    h64 = rows64 @ f["w1"]
    o64 = (h64 ** 2) @ f["w2"]
    y64 = O.combine(o64.reshape(-1, d), w64, slot)
    loss64, dlog = O.distill(y64 @ f["wo"], ids, teach, tau, None, g)
    G = {"wo": y64.T @ dlog}
    dy = dlog @ f["wo"].T
    _, do, dw = O.combine(o64.reshape(-1, d), w64, slot, dy)
    do = do.reshape(e, cap, d)
    G["w2"] = (h64 ** 2).transpose(0, 2, 1) @ do
    dh = (do @ f["w2"].transpose(0, 2, 1)) * 2 * h64
    G["w1"] = rows64.transpose(0, 2, 1) @ dh
    drows = dh @ f["w1"].transpose(0, 2, 1)
    dxn = O.combine(drows.reshape(-1, d), None, slot)
    dzr = O.route(zr, k, True, dw)[2]
    G["wr"] = xn64.T @ dzr
    dxn = dxn + dzr @ f["wr"].T
    _, _, _, _, G["gamma"], G["beta"] = O.group_norm(x[:, None], W["gamma"], W["beta"], groups, 1e-5, "silu",
                                                     dxn[:, None])
    near(loss, loss64, "loss", tol)
    for a in P:
        near(P[a].get_grad(), G[a], "d" + a, tol)


API_CASES = [group_norm, group_norm_only_parameters, saved_values_survive_writes, route, route_masked, plan,
             dispatch_and_combine, distill, model_step]


def refusals(F):
    x = T(F, np.ones((4, 6)))
    one = T(F, np.ones(6))
    ids = F.Indices(np.zeros((4, 2), np.int64))
    p = F.ExpertPlan(ids, 3, 4)
    bad = [
        lambda: F.group_norm(x, 4),                                   # channels not a multiple
        lambda: F.group_norm(x, 0),
        lambda: F.group_norm(T(F, np.ones(6)), 2),                    # no batch axis
        lambda: F.group_norm(x, 2, one),                              # gamma without beta
        lambda: F.group_norm(x, 2, one, T(F, np.ones(5))),
        lambda: F.group_norm(x, 2, activation="tanh"),
        lambda: F.group_norm(x, 2, eps=-1.0),
        lambda: F.route(x, 7),                                        # k > experts
        lambda: F.route(x, 0),
        lambda: F.route(T(F, np.ones((1, 1025))), 2),
        lambda: F.Indices(np.zeros((2, 2))),                          # not whole numbers
        lambda: F.Indices(np.array([1 << 31])),
        lambda: F.Indices(np.array([2 ** 64 - 1], np.uint64)),
        lambda: F.Indices([[1, 2], [3]]),
        lambda: F.Indices(np.int64(3)),                               # no axis
        lambda: F.ExpertPlan(ids, 0, 4),
        lambda: F.ExpertPlan(ids, 1025, 4),
        lambda: F.ExpertPlan(ids, 3, -1),
        lambda: F.ExpertPlan(ids, 3, 1 << 31),
        lambda: F.ExpertPlan(F.Indices(np.zeros((4, 0), np.int64)), 3),
        lambda: F.expert_dispatch(T(F, np.ones((5, 6))), p),          # another number of tokens
        lambda: F.expert_combine(T(F, np.ones((3, 5, 6))), p),        # another number of rows
        lambda: F.expert_combine(T(F, np.ones((3, 4, 6))), p, T(F, np.ones((4, 3)))),
        lambda: F.distill(x, ids, T(F, np.ones((4, 3)))),             # shapes differ
        lambda: F.distill(T(F, np.ones((5, 6))), ids, T(F, np.ones((4, 2)))),
        lambda: F.distill(x, ids, T(F, np.ones((4, 2))), temperature=0.0),
        lambda: F.distill(x, ids, T(F, np.ones((4, 2))), temperature=float("inf")),
        lambda: F.distill(x, ids, T(F, np.ones((4, 2))), teacher_lse=T(F, np.ones(3))),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was not refused")
