"""The language-model training operators' kernels through the C ABI, against the 64-bit
implementations of learn_oracle, at the sizes, alignments and masks where they can go
wrong; the same operators through the `fusion` module (learn_cases).

Bounds: u = 2^-24 is the largest relative error of one fp32 rounding, and every bound below
counts the roundings of the operator's formula to first order, with D sequential additions
for a sum of m values spread over at least 32 lanes (D = m / 32 + 32). CUDA's expf, erff
and logf and the hardware's 2^x are within 2 ulp = 4 u of their result.
"""
import ctypes as C

import numpy as np
import pytest

import learn_cases
import learn_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GUARD = 64
SENTINEL = np.float32(-12345.678)


class Out:
    """A device array of `shape` between two guard zones, `off` floats off 16-byte alignment;
    get() checks that the zones were left alone."""

    def __init__(self, capi, shape, off=0, dtype=np.float32):
        self.shape, self.n, self.off, self.dtype = tuple(shape), int(np.prod(shape)), off, dtype
        self.host = np.full(self.n + 2 * GUARD, SENTINEL, np.float32)
        self.d = capi.DeviceArray.from_numpy(self.host)
        self.ptr = self.d.ptr + 4 * (GUARD + off)

    def get(self):
        a = self.d.numpy()
        lo, hi = GUARD + self.off, GUARD + self.off + self.n
        assert np.all(a[:lo] == SENTINEL) and np.all(a[hi:] == SENTINEL), "wrote outside its output"
        return a[lo:hi].view(self.dtype).reshape(self.shape).copy()


class In:
    def __init__(self, capi, a, off=0):
        a = np.ascontiguousarray(a)
        a = a.astype(np.int32).view(np.float32) if a.dtype.kind in "iu" else a.astype(np.float32)
        self.d = capi.DeviceArray.from_numpy(np.concatenate([np.zeros(off, np.float32), a.ravel()]))
        self.ptr = self.d.ptr + 4 * off


def ptr(x):
    return None if x is None else x.ptr


def close(got, want, bound, what):
    got = got.astype(np.float64)
    same_nan = np.isnan(got) & np.isnan(want)
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= bound) | same_nan | (got == want)
    if not ok.all():
        i = np.unravel_index(int(np.argmin(ok)), ok.shape)
        raise AssertionError(f"{what}: {int((~ok).sum())} values off; at {i}: {got[i]!r} for {want[i]!r}, "
                             f"bound {np.broadcast_to(bound, ok.shape)[i]!r}")


# ---------------------------------------------------------------- group norm


def norm_bounds(x, gamma, beta, groups, eps, act, dy=None):
    """First-order bounds of y, mean, rstd (and dx, dgamma, dbeta)."""
    x = x.astype(np.float64)
    b, n, c = x.shape
    cg, m = c // groups, n * c // groups
    D = m / 32 + 32
    ga = np.ones(c) if gamma is None else gamma.astype(np.float64)
    be = np.zeros(c) if beta is None else beta.astype(np.float64)
    spread = lambda s: np.repeat(s, cg, axis=-1)[:, None, :]  # noqa: E731  [b, groups] -> [b, 1, c]
    over = lambda v: v.reshape(b, n, groups, cg).mean(axis=(1, 3))  # noqa: E731
    mean, var = over(x), None
    d = x - spread(mean)
    var = over(d * d)
    e_mean = (D + 3) * U * over(np.abs(x))
    e_d = spread(e_mean) + U * np.abs(d)
    with np.errstate(divide="ignore", invalid="ignore"):
        rstd = 1 / np.sqrt(var + eps)
        r_rstd = 0.5 * (over(2 * np.abs(d) * e_d + e_d * e_d) + (D + 3) * U * var) / (var + eps) + 4 * U
    xh = d * spread(rstd)
    e_xh = spread(rstd) * e_d + np.abs(xh) * (spread(r_rstd) + 2 * U)
    v = xh * ga + be
    e_v = np.abs(ga) * e_xh + 3 * U * (np.abs(ga * xh) + np.abs(be))
    res = [1.13 * e_v + 16 * U * np.abs(v), e_mean, rstd * r_rstd]
    if dy is None:
        return res, e_v, v
    dy = dy.astype(np.float64)
    slope = O.act_slope(v, act)
    e_slope = 0.0 if act in ("none", "relu") else 1.2 * e_v + 24 * U
    dv, a = dy * slope, dy * slope * ga
    e_dv = np.abs(dy) * e_slope + 2 * U * np.abs(dv)
    e_a = e_dv * np.abs(ga) + 2 * U * np.abs(a)
    k1, k2 = np.abs(over(a)), np.abs(over(a * xh))
    e_k1 = over(e_a) + (D + 3) * U * over(np.abs(a))
    e_k2 = over(e_a * np.abs(xh) + np.abs(a) * e_xh) + (D + 3) * U * over(np.abs(a * xh))
    parts = np.abs(a) + spread(k1) + np.abs(xh) * spread(k2)
    e_dx = spread(rstd) * (e_a + spread(e_k1) + e_xh * spread(k2) + np.abs(xh) * spread(e_k2) + 4 * U * parts) \
        + spread(rstd) * parts * (spread(r_rstd) + 2 * U)
    chain = b * n / 8 + 64
    e_dg = (e_dv * np.abs(xh) + np.abs(dv) * e_xh).sum(axis=(0, 1)) + chain * U * np.abs(dv * xh).sum(axis=(0, 1))
    e_db = e_dv.sum(axis=(0, 1)) + chain * U * np.abs(dv).sum(axis=(0, 1))
    return res + [e_dx, e_dg, e_db], e_v, v


def run_norm(capi, x, gamma, beta, groups, eps, act, dy=None, off=0, params=True):
    L = capi.lib()
    b, n, c = x.shape
    a = capi.ACTIVATIONS[act]
    dx_, dg, db = In(capi, x, off), gamma is not None and In(capi, gamma, off), beta is not None and In(capi, beta, off)
    pg, pb = (ptr(dg) if dg else None), (ptr(db) if db else None)
    y, mean, rstd = Out(capi, x.shape, off), Out(capi, (b, groups)), Out(capi, (b, groups))
    size = capi.group_norm_workspace(b, n, c, groups)
    work = Out(capi, ((size + 3) // 4,))
    capi.check(L.fz_group_norm(y.ptr, mean.ptr, rstd.ptr, dx_.ptr, pg, pb, b, n, c, groups, eps, a, work.ptr, size, None))
    res = [y.get(), mean.get(), rstd.get()]
    work.get()
    if dy is None:
        return res
    size = capi.group_norm_workspace(b, n, c, groups, True)
    work = Out(capi, ((size + 3) // 4,))
    dd = In(capi, dy, off)
    gx, gg, gb = Out(capi, x.shape, off), Out(capi, (c,), off), Out(capi, (c,), off)
    capi.check(L.fz_group_norm_backward(gx.ptr, gg.ptr if params else None, gb.ptr if params else None, dd.ptr,
                                        dx_.ptr, mean.ptr, rstd.ptr, pg, pb, b, n, c, groups, a, work.ptr, size, None))
    work.get()
    return res + [gx.get()] + ([gg.get(), gb.get()] if params else [])


# (batch, len, channels, groups): one value; odd groups; the MLP's rows; 10, 3, 2 and 1 channels a
# group; groups of 4 and more than one CTA holds; one group of many channels; many small samples;
# more samples than CTAs; a long sample with few channels, and a large one
NORM_SHAPES = [(1, 1, 1, 1), (3, 1, 8, 2), (2, 5, 12, 4), (4, 1, 4096, 32), (2, 37, 320, 32), (1, 1, 3, 1),
               (3, 100, 6, 6), (2, 4096, 64, 8), (1, 16384, 8, 2), (65, 1, 100, 1), (5, 7, 36, 9), (2, 130, 1000, 1),
               (1, 3, 20000, 2), (1000, 3, 8, 1), (4000, 1, 64, 4), (1, 30011, 16, 4), (2, 1024, 256, 32),
               (1, 65536, 32, 1), (3, 257, 68, 17), (9, 33, 1024, 64), (1, 2, 40000, 1), (300, 2, 2048, 1)]


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("act,affine,off", [("silu", True, 0), ("gelu", True, 1), ("none", False, 0)])
def test_group_norm(capi, shape, act, affine, off):
    b, n, c, groups = shape
    rng = np.random.default_rng(b * 7 + n * 3 + c)
    x = (rng.standard_normal((b, n, c)) * 1.5 + 0.7).astype(np.float32)
    dy = rng.standard_normal((b, n, c)).astype(np.float32)
    gamma = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32) if affine else None
    beta = (0.2 * rng.standard_normal(c)).astype(np.float32) if affine else None
    got = run_norm(capi, x, gamma, beta, groups, 1e-5, act, dy, off)
    want = O.group_norm(x, gamma, beta, groups, 1e-5, act, dy)
    bounds, _, _ = norm_bounds(x, gamma, beta, groups, 1e-5, act, dy)
    for name, g, w, e in zip(("y", "mean", "rstd", "dx", "dgamma", "dbeta"), got, want, bounds):
        close(g, w, e, name)
    again = run_norm(capi, x, gamma, beta, groups, 1e-5, act, dy, off)
    for g, h in zip(got, again):
        np.testing.assert_array_equal(g.view(np.uint32), h.view(np.uint32))


# channels a group that no vector of 4 divides while a row of them is whole vectors, up to a
# tile of 1020 channels; one tile a sample, a cluster's, and two launches
MIXED_SHAPES = [(3, 64, 12, 4), (2, 100, 20, 4), (2, 300, 12, 2), (1, 33, 1020, 4), (2, 50, 1020, 2), (1, 9000, 40, 8),
                (1, 40000, 28, 4), (3, 1369, 264, 8), (2, 65, 500, 20), (1, 20000, 140, 4), (5, 70, 104, 8),
                (3, 90, 12, 4), (2, 500, 64, 32), (1, 3000, 8, 4), (3, 9, 140, 4), (2, 70, 1000, 4)]


@pytest.mark.parametrize("shape", MIXED_SHAPES, ids=str)
@pytest.mark.parametrize("act,affine,off", [("silu", True, 0), ("gelu", True, 1), ("none", False, 0)])
def test_group_norm_vectors_across_groups(capi, shape, act, affine, off):
    test_group_norm(capi, shape, act, affine, off)


# a backward in vectors across groups after a forward by rows, beside sizes of the rows' own
@pytest.mark.parametrize("shape", [(5, 8, 1048, 8), (3, 5, 1020, 4), (7, 8, 1020, 4), (6, 48, 40, 4), (4, 24, 680, 4), (5, 48, 40, 8),
                                   (3, 11, 888, 4), (3, 9, 1048, 8), (3, 8, 2040, 4), (300, 48, 40, 4), (4, 80, 48, 8)], ids=str)
@pytest.mark.parametrize("act,affine,off", [("silu", True, 0), ("gelu", True, 1), ("none", False, 0)])
def test_group_norm_backward_in_other_tiles(capi, shape, act, affine, off):
    test_group_norm(capi, shape, act, affine, off)


# thread columns that are no power of two; groups in pieces; many tiles of a few rows
@pytest.mark.parametrize("shape", [(2, 300, 300, 5), (3, 500, 150, 1), (2, 51, 271, 1), (1, 90, 1031, 1), (2, 40, 9000, 2),
                                   (1, 700, 777, 1), (3, 2000, 80, 4), (2, 12, 1100, 2), (1, 5000, 1036, 1), (40, 64, 640, 32),
                                   (37, 18, 264, 4), (700, 7, 148, 2), (5, 232, 4, 2), (30, 30, 1040, 8)], ids=str)
@pytest.mark.parametrize("act,affine,off", [("silu", True, 0), ("gelu", True, 1), ("none", False, 0)])
def test_group_norm_tiles_of_each_width(capi, shape, act, affine, off):
    test_group_norm(capi, shape, act, affine, off)


@pytest.mark.parametrize("shape,at", [((3, 64, 12, 4), 1), ((2, 100, 20, 4), 2), ((1, 9000, 40, 8), 3), ((2, 1369, 320, 32), 13),
                                      ((1, 40000, 28, 4), 1), ((3, 130, 264, 8), 5)], ids=str)
def test_group_norm_neighbours_in_a_vector_stay_apart(capi, shape, at):
    """NaN in one group's last channel and 1e18 in the next one's first: the groups around them,
    whose values share vectors with theirs, come out bit for bit as without them."""
    b, n, c, groups = shape
    per = c // groups
    rng = np.random.default_rng(16)
    x, dy = rng.standard_normal(shape[:3]).astype(np.float32), rng.standard_normal(shape[:3]).astype(np.float32)
    clean = run_norm(capi, x, None, None, groups, 1e-5, "silu", dy)
    bad = x.copy()
    bad[0, n // 2, at * per - 1] = np.nan
    bad[0, n - 1, at * per] = 1e18
    got = run_norm(capi, bad, None, None, groups, 1e-5, "silu", dy)
    hit = np.zeros((b, n, c), bool)
    hit[0, :, (at - 1) * per:(at + 1) * per] = True
    for which in (0, 3):
        np.testing.assert_array_equal(got[which][~hit], clean[which][~hit])
    assert np.isnan(got[0][0, :, (at - 1) * per:at * per]).all()
    assert np.isfinite(got[0][0, :, at * per:(at + 1) * per]).all()


@pytest.mark.parametrize("shape", [(4, 1, 4096, 32), (2, 37, 320, 32), (1, 16384, 8, 2)], ids=str)
def test_group_norm_relu(capi, shape):
    """ReLU's slope jumps at zero: the inputs keep away from it by more than v's error."""
    b, n, c, groups = shape
    rng = np.random.default_rng(11)
    x = rng.standard_normal((b, n, c)).astype(np.float32)
    dy = rng.standard_normal((b, n, c)).astype(np.float32)
    gamma, beta = np.ones(c, np.float32), np.zeros(c, np.float32)
    for _ in range(4):  # move values near zero away from it
        bounds, e_v, v = norm_bounds(x, gamma, beta, groups, 1e-5, "relu", dy)
        x = np.where(np.abs(v) < 1e-2, x + np.float32(0.05), x)
    bounds, e_v, v = norm_bounds(x, gamma, beta, groups, 1e-5, "relu", dy)
    assert np.all(np.abs(v) > 2 * e_v)
    got = run_norm(capi, x, gamma, beta, groups, 1e-5, "relu", dy)
    want = O.group_norm(x, gamma, beta, groups, 1e-5, "relu", dy)
    for name, g, w, e in zip(("y", "mean", "rstd", "dx", "dgamma", "dbeta"), got, want, bounds):
        close(g, w, e, name)


@pytest.mark.parametrize("shape", [(4, 1, 256, 4), (3, 600, 64, 2), (1, 40000, 8, 1)], ids=str)
def test_group_norm_offset_and_constant(capi, shape):
    """A large common offset costs no more digits than x lost by it; a constant group has
    variance 0, and its result is beta."""
    b, n, c, groups = shape
    rng = np.random.default_rng(12)
    x = (rng.standard_normal((b, n, c)) + 1000).astype(np.float32)
    x[0, :, : c // groups] = 3.25
    beta = rng.standard_normal(c).astype(np.float32)
    gamma = np.ones(c, np.float32)
    got = run_norm(capi, x, gamma, beta, groups, 1e-5, "none")
    want = O.group_norm(x, gamma, beta, groups, 1e-5, "none")
    bounds, _, _ = norm_bounds(x, gamma, beta, groups, 1e-5, "none")
    for name, g, w, e in zip(("y", "mean", "rstd"), got, want, bounds):
        close(g, w, e, name)
    # variance 3.25 is exact in every order of summation, so is the group's mean
    np.testing.assert_array_equal(got[0][0, :, : c // groups], np.broadcast_to(beta[: c // groups], (n, c // groups)))


@pytest.mark.parametrize("shape", [(6, 1, 64, 4), (3, 50, 40, 4), (2, 9000, 16, 2)], ids=str)
def test_group_norm_nan_stays_in_its_group(capi, shape):
    b, n, c, groups = shape
    rng = np.random.default_rng(13)
    x = rng.standard_normal((b, n, c)).astype(np.float32)
    clean = run_norm(capi, x, None, None, groups, 1e-5, "silu")[0]
    x[1, n // 2, 0] = np.nan
    x[0, 0, c - 1] = np.inf
    y = run_norm(capi, x, None, None, groups, 1e-5, "silu")[0]
    hit = np.zeros((b, n, c), bool)
    hit[1, :, : c // groups] = True
    hit[0, :, c - c // groups:] = True
    assert np.isnan(y[1, :, : c // groups]).all() and np.isnan(y[0, :, c - c // groups:]).any()
    np.testing.assert_array_equal(y[~hit], clean[~hit])


# the last of a sample's tiles, in a cluster and in two launches, has fewer rows than a CTA's threads
@pytest.mark.parametrize("shape", [(1, 181, 260, 4), (1, 961, 260, 4), (2, 181, 260, 4), (3, 64, 1020, 4), (2, 300, 300, 5),
                                   (1, 40000, 28, 4)], ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("off", [0, 1])
def test_group_norm_gradients_of_a_bad_group_stay_in_it(capi, shape, act, off):
    """NaN in each of the groups in turn: dx, dgamma and dbeta of the others are bit for bit what they
    are without it."""
    b, n, c, groups = shape
    per = c // groups
    rng = np.random.default_rng(17)
    x, dy = rng.standard_normal(shape[:3]).astype(np.float32), rng.standard_normal(shape[:3]).astype(np.float32)
    clean = run_norm(capi, x, None, None, groups, 1e-5, act, dy, off)
    for g in range(groups):
        bad = x.copy()
        bad[b - 1, n // 2, g * per] = np.nan
        got = run_norm(capi, bad, None, None, groups, 1e-5, act, dy, off)
        hit = np.zeros((b, n, c), bool)
        hit[b - 1, :, g * per:(g + 1) * per] = True
        np.testing.assert_array_equal(got[3][~hit], clean[3][~hit])
        assert np.isnan(got[3][hit]).all()
        for which in (4, 5):
            np.testing.assert_array_equal(np.delete(got[which], np.s_[g * per:(g + 1) * per]),
                                          np.delete(clean[which], np.s_[g * per:(g + 1) * per]))


@pytest.mark.parametrize("shape,value", [((2, 300, 1, 1), 1e36), ((3, 181, 260, 4), 2e34), ((2, 2000, 12, 2), 3e33)], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_group_norm_gradients_of_a_large_constant(capi, shape, value, act):
    """Equal values so large that value * rstd overflows: x - mean is 0, and the gradients are finite.
    (eps is chosen so that it does, while no sum of the values does.)"""
    b, n, c, groups = shape
    rng = np.random.default_rng(18)
    x = np.full(shape[:3], value, np.float32)
    x = np.float32(2.0 ** np.floor(np.log2(x)))  # a power of two: its sums and mean are exact
    eps = np.float32((float(x.flat[0]) / 1e39) ** 2)
    dy = rng.standard_normal(shape[:3]).astype(np.float32)
    got = run_norm(capi, x, None, None, groups, eps, act, dy)
    rstd = 1 / np.sqrt(np.float64(eps))
    # xh = 0 and v = 0: dv = dy / 2, dx = rstd (dv - mean dv), dgamma = 0, dbeta = sum dv
    dv = dy.astype(np.float64) / 2
    g4 = dv.reshape(b, n, groups, c // groups)
    mean, size = g4.mean(axis=(1, 3), keepdims=True), np.abs(g4).mean(axis=(1, 3), keepdims=True)
    m = n * c // groups
    want = rstd * (g4 - mean).reshape(x.shape)
    close(got[3], want, rstd * U * (16 * np.abs(g4) + (m / 32 + 48) * size).reshape(x.shape), "dx")
    assert not got[4].any()
    close(got[5], dv.sum(axis=(0, 1)), (b * n / 8 + 64) * U * np.abs(dv).sum(axis=(0, 1)), "dbeta")


# 1, 2, 4 and 8 vectors a lane of a warp, 2 a thread of a CTA, so that each thread adds up some 250
# steps; how many teams of a group are in flight on 148 SMs, how many of them a step takes, and the
# steps of a block
@pytest.mark.parametrize("shape,parts,at_once,block", [((65536, 1, 4096, 32), 74, 4, 16), ((40000, 1, 8192, 32), 74, 2, 16),
                                                       ((20000, 1, 16384, 32), 74, 1, 64), ((10000, 1, 32768, 32), 37, 1, 64),
                                                       ((40000, 1, 4096, 2), 148, 1, 16), ((300000, 1, 512, 64), 296, 4, 16)], ids=str)
def test_group_norm_parameter_sums_keep_their_digits(capi, shape, parts, at_once, block):
    """One large dy before many ones: a chain of additions to it loses each of them, blocks of
    steps do not. x is +-1, so xh is too (eps = 0) and every product is exact. The bound: the
    teams of a step, the steps of a block, a thread's blocks, and the fold over the teams in flight:
    16 rows a block, their blocks, 16 warps, 8 CTAs."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    b, n, c, groups = shape
    x = torch.ones(b, n, c, device="cuda")
    x[:, :, 1::2] = -1
    dy = torch.ones_like(x)
    big = 2.0 ** 24 * at_once
    dy[0] = big
    dy[0, :, c // 2:] = 1
    dy[b - 1, :, c // 2:] = big
    y, dx = torch.empty_like(x), torch.empty_like(x)
    stats, gb = torch.empty(2, b, groups, device="cuda"), torch.empty(2, c, device="cuda")
    size = capi.group_norm_workspace(b, n, c, groups, True)
    work = torch.empty(size // 4 + 4, device="cuda")
    at = lambda t: t.data_ptr()  # noqa: E731
    capi.check(L.fz_group_norm(at(y), at(stats[0]), at(stats[1]), at(x), None, None, b, n, c, groups, 0.0, 0, at(work), size, 1))
    capi.check(L.fz_group_norm_backward(at(dx), at(gb[0]), at(gb[1]), at(dy), at(x), at(stats[0]), at(stats[1]), None, None, b, n, c,
                                        groups, 0, at(work), size, 1))
    torch.cuda.synchronize()
    assert torch.equal(y, x)
    sign = x[0, 0].double().cpu().numpy()
    got = gb.double().cpu().numpy()
    want = big + b * n - 1
    bound = (at_once + block + b / parts / at_once / block + 1 + 16 + 16 + 16 + 8) * U * want
    close(got[0], sign * want, bound, "dgamma")
    close(got[1], np.full(c, want), bound, "dbeta")
    del x, y, dx, dy, work
    torch.cuda.empty_cache()


SPIKE_SHAPES = [(65, 1, 100, 1), (4, 1, 4096, 32), (2, 4096, 64, 8), (1, 16384, 8, 2), (1, 65536, 32, 1), (1, 30011, 16, 4),
                (1, 40000, 28, 4), (1, 9000, 40, 8), (1, 20000, 140, 4), (1, 5000, 1036, 1), (2, 1024, 256, 32), (1, 2, 40000, 1),
                (700, 7, 148, 2), (1, 181, 260, 4), (1, 961, 260, 4), (5, 7, 2368, 32), (3, 257, 68, 17), (2, 40, 9000, 2),
                (1, 300001, 32, 1), (300, 2, 2048, 1), (5, 8, 1048, 8)]


@pytest.mark.parametrize("shape", SPIKE_SHAPES, ids=str)
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("where", ["first", "last", "inside"])
def test_group_norm_counts_each_value_once(capi, shape, off, where):
    """One value other than 0: it alone makes mean and rstd, which show it left out, counted twice or
    counted for another group. dy of small whole numbers: dbeta is exact. (The sums' zeros are exact, so
    the bounds are a few dozen roundings of divisions and joins, whatever the length.)"""
    b, n, c, groups = shape
    per, m = c // groups, n * c // groups
    rng = np.random.default_rng(b + n + c)
    at = {"first": (0, 0, 0), "last": (b - 1, n - 1, c - 1), "inside": tuple(int(rng.integers(s)) for s in (b, n, c))}[where]
    x = np.zeros((b, n, c), np.float32)
    x[at] = 1000.0
    dy = rng.integers(-8, 9, (b, n, c)).astype(np.float32)
    eps = 2.0 ** -20
    y, mean, rstd, dx, dg, db = run_norm(capi, x, None, None, groups, eps, "none", dy, off)
    want_mean, want_rstd = np.zeros((b, groups)), np.full((b, groups), 1 / np.sqrt(eps))
    want_mean[at[0], at[2] // per] = 1000.0 / m
    var = 1e6 / m * (1 - 1 / m)
    want_rstd[at[0], at[2] // per] = 1 / np.sqrt(var + eps)
    close(mean, want_mean, 64 * U * np.abs(want_mean), "mean")
    close(rstd, want_rstd, 64 * U * want_rstd, "rstd")
    np.testing.assert_array_equal(db, dy.sum(axis=(0, 1), dtype=np.float64))
    xh = (x - np.repeat(want_mean, per, axis=1)[:, None]) * np.repeat(want_rstd, per, axis=1)[:, None]
    # xh = s (x - mean) of a group of zeros and one 1000: the roundings of mean and rstd (64 each), and
    # sums of equal magnitudes: at most 32 rows, 16 levels, a run of 16 and the fold's 56
    close(dg, (dy * xh).sum(axis=(0, 1)), (2 * 64 + 4 + 32 + 16 + 16 + 56) * U * (np.abs(dy * xh)).sum(axis=(0, 1)), "dgamma")


def test_group_norm_workspace_stays_below_the_input(capi):
    """Samples of one row whose groups need several CTAs: the parameters' partial sums are an eighth
    of x, not twice x, once there are many; beside them two launches leave 2 floats a tile. Narrow
    groups: two thirds at most."""
    for shape in ((65536, 1, 16384, 1), (100000, 1, 4097, 1), (65536, 1, 131072, 8), (200000, 2, 5000, 1), (1000000, 1, 2100, 1)):
        b, n, c, _ = shape
        assert capi.group_norm_workspace(*shape, True) <= 4 * b * n * c * (1 / 8 + 1 / 64), shape
    for shape in ((100000, 3, 508, 4), (100000, 5, 504, 4), (50000, 11, 400, 4), (30000, 3, 2368, 32), (70000, 5, 1020, 4),
                  (400000, 2, 255, 1), (300000, 3, 127, 1)):
        b, n, c, _ = shape
        assert capi.group_norm_workspace(*shape, True) <= 4 * b * n * c * 2 / 3, shape


# runs of samples at one place of a sample: clusters (vectors of 4 and single floats), two launches,
# vectors across groups, several bundles; a last run that is shorter
@pytest.mark.parametrize("shape,off", [((2503, 1, 8200, 1), 0), ((5003, 1, 2100, 1), 1), ((3001, 1, 20000, 1), 0),
                                       ((40011, 5, 508, 4), 0), ((9001, 9, 516, 12), 0), ((6007, 1, 4097, 1), 0),
                                       ((2000, 3, 5000, 1), 2)], ids=str)
def test_group_norm_parameter_sums_of_many_samples(capi, shape, off):
    """dbeta of small whole numbers is exact in every order of summation: no row is left out or counted
    twice. dgamma within the roundings of a thread's rows (32), the tile's tree (8), a run (16), the
    fold (56), and of xh (64)."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    b, n, c, groups = shape
    gen = torch.Generator("cuda").manual_seed(3)
    flat = torch.empty(b * n * c + 4, device="cuda")
    x = flat[off:off + b * n * c].view(b, n, c).normal_(generator=gen)
    dy = torch.randint(-8, 9, (b, n, c), generator=gen, device="cuda").float()
    y, dx = torch.empty_like(flat), torch.full((b * n * c + 8,), 7.0, device="cuda")
    stats, gb = torch.empty(2, b, groups, device="cuda"), torch.empty(2, c, device="cuda")
    size = capi.group_norm_workspace(b, n, c, groups, True)
    work = torch.empty(size // 4 + 4, device="cuda")
    work.fill_(float("nan"))
    at = lambda t: t.data_ptr()  # noqa: E731
    capi.check(L.fz_group_norm(at(y[off:]), at(stats[0]), at(stats[1]), at(x), None, None, b, n, c, groups, 1e-5, 0, at(work), size, 1))
    work.fill_(float("nan"))
    capi.check(L.fz_group_norm_backward(at(dx[off:]), at(gb[0]), at(gb[1]), at(dy), at(x), at(stats[0]), at(stats[1]), None, None, b, n,
                                        c, groups, 0, at(work), size, 1))
    torch.cuda.synchronize()
    assert torch.equal(gb[1].double(), dy.double().sum((0, 1)))
    total, size_of = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")
    for lo in range(0, b, 500):
        part = x[lo:lo + 500].double()
        grouped = part.view(-1, n, groups, c // groups)
        var, mean = torch.var_mean(grouped, dim=(1, 3), keepdim=True, correction=0)
        xh = ((grouped - mean) / torch.sqrt(var + 1e-5)).view(part.shape)
        d = dy[lo:lo + 500].double()
        total += (d * xh).sum((0, 1))
        size_of += (d.abs() * (xh.abs() + 1)).sum((0, 1))
        if lo == 0 or lo + 500 >= b:
            a = d.view(grouped.shape)
            h = xh.view(grouped.shape)
            r = 1 / torch.sqrt(var + 1e-5)
            want = r * (a - a.mean((1, 3), keepdim=True) - h * (a * h).mean((1, 3), keepdim=True))
            got = dx[off + lo * n * c:off + (lo + part.shape[0]) * n * c].view(grouped.shape).double()
            # sums of up to 32 rows, 8 levels and 16 tiles; values of at most 8
            bound = 100 * U * r * (a.abs() + 8 * (1 + h.abs()))
            assert ((got - want).abs() <= bound).all()
    assert ((gb[0].double() - total).abs() <= (32 + 8 + 16 + 56 + 64) * U * size_of).all()
    assert (dx[:off] == 7).all() and (dx[off + b * n * c:] == 7).all()
    del flat, x, dy, y, dx, work
    torch.cuda.empty_cache()


# more than 256 tiles a group: vectors of 4, across groups, single floats
@pytest.mark.parametrize("shape,off", [((1, 1 << 20, 8, 2), 0), ((2, 500001, 12, 4), 0), ((1, 200003, 31, 1), 0), ((1, 400000, 32, 4), 1),
                                       ((3, 300000, 32, 1), 0)], ids=str)
def test_group_norm_of_long_samples(capi, shape, off):
    """Bounds: sums of at most 32 rows, 8 levels and a tile's 16 columns in fp32 (the tiles' are joined in
    64 bits), so D = 64 with what is rounded beside them; a common offset of 50 costs x's own digits."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    b, n, c, groups = shape
    gen = torch.Generator("cuda").manual_seed(5)
    flat = torch.empty(b * n * c + 4, device="cuda")
    x = flat[off:off + b * n * c].view(b, n, c).normal_(generator=gen)
    x += 50
    x[:, -1, -1] += 1000  # the last value of each sample counts
    dy = torch.randint(-8, 9, (b, n, c), generator=gen, device="cuda").float()
    y, dx = torch.empty_like(flat), torch.empty_like(flat)
    stats, gb = torch.empty(2, b, groups, device="cuda"), torch.empty(2, c, device="cuda")
    size = capi.group_norm_workspace(b, n, c, groups)
    assert size > 8 * b * groups * 257  # a pair a tile and one of the group
    size = capi.group_norm_workspace(b, n, c, groups, True)
    work = torch.full((size // 4 + 4,), float("nan"), device="cuda")
    at = lambda t: t.data_ptr()  # noqa: E731
    capi.check(L.fz_group_norm(at(y[off:]), at(stats[0]), at(stats[1]), at(x), None, None, b, n, c, groups, 1e-5, 0, at(work), size, 1))
    work.fill_(float("nan"))
    capi.check(L.fz_group_norm_backward(at(dx[off:]), at(gb[0]), at(gb[1]), at(dy), at(x), at(stats[0]), at(stats[1]), None, None, b, n,
                                        c, groups, 0, at(work), size, 1))
    torch.cuda.synchronize()
    g4 = lambda t: t.view(b, n, groups, c // groups).double()  # noqa: E731
    X, A, Y, DX = g4(x), g4(dy), g4(y[off:off + b * n * c]), g4(dx[off:off + b * n * c])
    E = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mean = E(X)
    var = E((X - mean) ** 2)
    rstd = 1 / torch.sqrt(var + 1e-5)
    H = (X - mean) * rstd
    D = 64 * U
    e_mean = D * E(X.abs())
    e_rstd = D + e_mean * rstd  # relative
    assert ((stats[0].view_as(mean).double() - mean).abs() <= e_mean).all()
    assert ((stats[1].view_as(mean).double() - rstd).abs() <= rstd * e_rstd).all()
    e_h = rstd * e_mean + H.abs() * (e_rstd + 4 * U)
    assert ((Y - H).abs() <= e_h).all()
    k1, k2 = E(A), E(A * H)
    e_k1, e_k2 = D * E(A.abs()), D * E((A * H).abs()) + E(A.abs() * e_h)
    want = rstd * (A - k1 - H * k2)
    size_of = A.abs() + k1.abs() + H.abs() * k2.abs()
    assert ((DX - want).abs() <= rstd * (e_k1 + H.abs() * e_k2 + e_h * k2.abs() + size_of * (e_rstd + 6 * U))).all()
    assert torch.equal(gb[1].double(), dy.double().sum((0, 1)))
    e_g = (A.abs() * e_h + (A * H).abs() * (D + 56 * U)).sum((0, 1)).view(c)
    assert ((gb[0].double() - (A * H).sum((0, 1)).view(c)).abs() <= e_g).all()
    del flat, x, dy, y, dx, work, X, A, Y, DX, H
    torch.cuda.empty_cache()


def test_group_norm_of_a_long_sample_takes_no_longer(capi):
    """One sample of 2^23 rows of 32 channels (up to 32768 tiles) against 16 of 2^19, the same bytes. Each
    tile's joining all tiles' statistics took 6 times as long; 3 times is the most allowed here."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    n = 1 << 28
    x, y, dx = (torch.ones(n, device="cuda") for _ in range(3))
    at = lambda t: t.data_ptr()  # noqa: E731
    times = []
    for b in (16, 1):
        s = (b, n // 32 // b, 32, 1)
        stats, gb = torch.empty(2, b, device="cuda"), torch.empty(2, 32, device="cuda")
        size = capi.group_norm_workspace(*s, True)
        work = torch.empty(size // 4 + 4, device="cuda")

        def call():
            capi.check(L.fz_group_norm(at(y), at(stats[0]), at(stats[1]), at(x), None, None, *s, 1e-5, 0, at(work), size, 1))
            capi.check(L.fz_group_norm_backward(at(dx), at(gb[0]), at(gb[1]), at(x), at(x), at(stats[0]), at(stats[1]), None, None, *s, 0,
                                                at(work), size, 1))

        best = float("inf")
        for i in range(4):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            call()
            end.record()
            torch.cuda.synchronize()
            best = min(best, begin.elapsed_time(end)) if i else best
        times.append(best)
    del x, y, dx
    torch.cuda.empty_cache()
    assert times[1] <= 3 * times[0], times


def test_group_norm_partial_results(capi):
    """mean and rstd, and the parameters' gradients, are optional; an empty batch has zero
    gradients."""
    L = capi.lib()
    rng = np.random.default_rng(14)
    x, dy = rng.standard_normal((2, 3, 8)).astype(np.float32), rng.standard_normal((2, 3, 8)).astype(np.float32)
    y, d = Out(capi, x.shape), In(capi, x)
    size = capi.group_norm_workspace(2, 3, 8, 2)
    work = Out(capi, ((size + 3) // 4,))
    capi.check(L.fz_group_norm(y.ptr, None, None, d.ptr, None, None, 2, 3, 8, 2, 1e-5, 0, work.ptr, size, None))
    full = run_norm(capi, x, None, None, 2, 1e-5, "none", dy)
    np.testing.assert_array_equal(y.get(), full[0])
    np.testing.assert_array_equal(run_norm(capi, x, None, None, 2, 1e-5, "none", dy, params=False)[3], full[3])
    dg, db = Out(capi, (8,)), Out(capi, (8,))
    size = capi.group_norm_workspace(0, 3, 8, 2, True)
    work = Out(capi, ((size + 3) // 4,))
    capi.check(L.fz_group_norm_backward(None, dg.ptr, db.ptr, None, None, None, None, None, None, 0, 3, 8, 2, 0,
                                        work.ptr, size, None))
    assert not dg.get().any() and not db.get().any()


def test_group_norm_gradient_by_differences(capi):
    """<dx, h> against the central difference of the kernel's own forward along h."""
    rng = np.random.default_rng(15)
    shape, groups, eps = (3, 20, 24), 4, 1e-3
    x, dy, h = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    gamma, beta = rng.standard_normal(24).astype(np.float32), rng.standard_normal(24).astype(np.float32)
    step = np.float32(2.0 ** -6)
    dx = run_norm(capi, x, gamma, beta, groups, eps, "gelu", dy)[3].astype(np.float64)
    hi, lo = x + step * h, x - step * h
    f = lambda z: (run_norm(capi, z, gamma, beta, groups, eps, "gelu")[0].astype(np.float64) * dy).sum()  # noqa: E731
    slope = (f(hi) - f(lo)) / (2 * float(step))
    # the difference's own error: its third-order term, measured at a doubled step in 64 bits,
    # and the forward's roundings over the step
    g = lambda s: ((O.group_norm(x + s * h, gamma, beta, groups, eps, "gelu")[0] - O.group_norm(  # noqa: E731
        x - s * h, gamma, beta, groups, eps, "gelu")[0]) * dy).sum() / (2 * s)
    curve = abs(g(2 * float(step)) - g(float(step)))
    e_y = norm_bounds(x, gamma, beta, groups, eps, "gelu")[0][0]
    bound = curve + 1.2 * (e_y * np.abs(dy)).sum() / float(step)
    assert abs(slope - (dx * h).sum()) <= bound


# ---------------------------------------------------------------- router


def run_route(capi, z, k, renorm, dw=None):
    L = capi.lib()
    t, e = z.shape
    d, w, ids = In(capi, z), Out(capi, (t, k)), Out(capi, (t, k), dtype=np.int32)
    capi.check(L.fz_route(w.ptr, ids.ptr, d.ptr, t, e, k, renorm, None))
    if dw is None:
        return w.get(), ids.get()
    g, dz = In(capi, dw), Out(capi, (t, e))
    capi.check(L.fz_route_backward(dz.ptr, g.ptr, w.ptr, ids.ptr, d.ptr, t, e, k, renorm, None))
    return w.get(), ids.get(), dz.get()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (5, 3, 3), (33, 32, 4), (7, 33, 2), (1000, 64, 8), (17, 100, 1),
                                   (9, 256, 32), (4, 300, 5), (3, 513, 8), (2, 1024, 32), (70001, 8, 2)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route(capi, t, e, k, renorm):
    rng = np.random.default_rng(t + e)
    z = (rng.standard_normal((t, e)) * 3).astype(np.float32)
    z[: t // 2] = np.round(z[: t // 2])  # ties
    z[rng.random((t, e)) < 0.1] = -np.inf
    z[rng.random((t, e)) < 0.05] = -0.0
    z[0] = -np.inf if t > 4 else z[0]
    dw = rng.standard_normal((t, k)).astype(np.float32)
    sample = slice(None) if t < 2000 else np.r_[0:500, t - 500:t]
    w, ids, dz = (a[sample] for a in run_route(capi, z, k, renorm, dw))
    w64, i64, dz64 = O.route(z[sample], k, renorm, dw[sample])
    np.testing.assert_array_equal(ids, i64)
    # exp's argument (exact to u |d|, |d| the distance below the largest), exp, a sum of at
    # most E / 32 + 5 additions of such terms, the quotient
    far = np.where(np.isfinite(z), np.nanmax(np.where(np.isfinite(z), z, -1e9), axis=1, keepdims=True) - z, 0)[sample].max()
    rel = U * (2 * far + e / 32 + k + 24)
    close(w, w64, rel * w64, "weights")
    terms = (np.abs(w64) * np.abs(dw[sample])).sum(1, keepdims=True)
    close(dz, dz64, (rel + (k + 8) * U) * (np.abs(dw[sample]).max(1, keepdims=True) + terms), "dlogits")
    if renorm:
        assert not dz[dz64 == 0].any()


# more experts than eight lanes hold: half the tokens with ties, one without experts
@pytest.mark.parametrize("t,e,k", [(61, 300, 8), (64, 512, 4), (33, 512, 8), (31, 700, 3), (40, 1024, 8), (5, 257, 1), (1500, 384, 6)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_many_experts(capi, t, e, k, renorm):
    test_route(capi, t, e, k, renorm)


@pytest.mark.parametrize("e", [40, 300, 1000])
def test_route_nan_stays_with_its_token(capi, e):
    """A NaN, or a tie, among the tokens that share a warp."""
    rng = np.random.default_rng(31)
    z = rng.standard_normal((50, e)).astype(np.float32)
    clean, clean_ids = run_route(capi, z, 4, False)
    z[7, e - 1], z[20, 3], z[21] = np.nan, np.nan, 0.5
    w, ids = run_route(capi, z, 4, False)
    others = np.delete(np.arange(50), [7, 20, 21])
    np.testing.assert_array_equal(ids[others], clean_ids[others])
    np.testing.assert_array_equal(w[others], clean[others])
    assert ids[7, 0] == e - 1 and ids[20, 0] == 3 and np.isnan(w[[7, 20]]).all()
    np.testing.assert_array_equal(ids[21], np.arange(4))
    close(w[21], np.full(4, 1 / e), (e / 32 + 30) * U / e, "uniform")


def test_route_specials(capi):
    """NaN ranks first and makes its token's weights NaN, other tokens keep theirs; the
    type's lowest value is a number like others; equal logits go to the lowest experts."""
    low = np.finfo(np.float32).min
    z = np.array([[0, np.nan, 1, 2], [low, low, low, low], [-np.inf, low, -np.inf, -np.inf], [5, 5, 5, 5],
                  [-np.inf] * 4, [0.0, -0.0, 0.0, -0.0]], np.float32)
    w, ids = run_route(capi, z, 2, True)
    np.testing.assert_array_equal(ids, [[1, 3], [0, 1], [1, -1], [0, 1], [-1, -1], [0, 1]])
    assert np.isnan(w[0]).all()
    np.testing.assert_array_equal(w[1:], np.float32([[.5, .5], [1, 0], [.5, .5], [0, 0], [.5, .5]]))
    w, ids, dz = run_route(capi, z, 2, False, np.ones((6, 2), np.float32))
    assert np.isnan(dz[0]).all() and not np.isnan(dz[1:]).any() and not dz[4].any()


def test_route_backward_ignores_foreign_ids(capi):
    """Ids that name no expert take no part (and touch no memory outside the row)."""
    L = capi.lib()
    z, w = np.zeros((2, 4), np.float32), np.full((2, 2), 0.5, np.float32)
    ids = np.array([[1, 1000000], [-7, 4]])
    a = [In(capi, v) for v in (np.ones((2, 2)), w, ids, z)]
    dz = Out(capi, (2, 4))
    capi.check(L.fz_route_backward(dz.ptr, *[v.ptr for v in a], 2, 4, 2, 1, None))
    np.testing.assert_array_equal(dz.get(), [[0, 0.25, 0, 0], [0, 0, 0, 0]])


# ---------------------------------------------------------------- experts


def run_sort(capi, ids, e, cap):
    t, k = ids.shape
    rows = e * cap if cap else t * k
    d = In(capi, ids)
    outs = [Out(capi, s, dtype=np.int32) for s in ((t, k), (rows,), (e,), (e + 1,))]
    capi.check(capi.lib().fz_expert_sort(*[o.ptr for o in outs], d.ptr, t, k, e, cap, None))
    return [o.get() for o in outs]


@pytest.mark.parametrize("t,k,e,cap", [(1, 1, 1, 0), (1, 2, 4, 1), (16, 2, 64, 0), (31, 3, 7, 0), (1000, 4, 8, 300),
                                       (1000, 4, 8, 700), (4097, 2, 5, 0), (9000, 8, 256, 250), (20000, 2, 1024, 0),
                                       (5000, 1, 1024, 6), (300, 7, 1000, 0), (65536, 8, 64, 0), (64, 1, 3, 40000)])
def test_expert_sort(capi, t, k, e, cap):
    rng = np.random.default_rng(t + e)
    ids = np.minimum((rng.random((t, k)) ** 2 * (e + 1)).astype(np.int64), e) - (rng.random((t, k)) < 0.1) * (e + 3)
    for got, want, name in zip(run_sort(capi, ids, e, cap), O.expert_sort(ids, e, cap), ("slot", "src", "counts", "offsets")):
        np.testing.assert_array_equal(got, want, err_msg=name)


@pytest.mark.parametrize("ids", [np.full((70, 3), -1), np.full((70, 3), 2), np.full((5000, 2), 2 ** 31 - 1),
                                 np.zeros((20000, 1), np.int64)], ids=["none", "one", "foreign", "first"])
@pytest.mark.parametrize("cap", [0, 50])
def test_expert_sort_one_sided(capi, ids, cap):
    for got, want in zip(run_sort(capi, ids, 4, cap), O.expert_sort(ids, 4, cap)):
        np.testing.assert_array_equal(got, want)


def test_expert_sort_without_tokens(capi):
    L = capi.lib()
    for cap in (0, 5):
        src, counts, offsets = (Out(capi, (n,), dtype=np.int32) for n in (15 if cap else 0, 3, 4))
        capi.check(L.fz_expert_sort(None, src.ptr, counts.ptr, offsets.ptr, None, 0, 2, 3, cap, None))
        assert (src.get() == -1).all() and not counts.get().any()
        np.testing.assert_array_equal(offsets.get(), np.arange(4) * cap)


EXPERT_SHAPES = [(1, 1, 1, 0, 1, 0), (16, 2, 8, 0, 4096, 0), (37, 3, 5, 11, 1001, 0), (100, 8, 16, 40, 64, 0),
                 (5, 4, 4, 0, 516, 1), (300, 2, 3, 300, 8, 0), (64, 1, 4, 0, 2048, 0), (9, 2, 3, 2, 7, 3), (700, 5, 9, 0, 132, 0),
                 (3, 40, 64, 2, 260, 0)]


@pytest.mark.parametrize("t,k,e,cap,width,off", EXPERT_SHAPES)
def test_dispatch_and_combine(capi, t, k, e, cap, width, off):
    L = capi.lib()
    rng = np.random.default_rng(t * 5 + width)
    ids = rng.integers(-1, e, (t, k))
    slot, src, _, _ = O.expert_sort(ids, e, cap)
    n = len(src)
    x, g = (rng.standard_normal((t, width)).astype(np.float32) for _ in range(2))
    y = rng.standard_normal((n, width)).astype(np.float32)
    y[src < 0] = np.nan  # rows that no choice has are never read into a result
    w = rng.uniform(-1, 1, (t, k)).astype(np.float32)
    dslot, dsrc = In(capi, slot), In(capi, src)
    dx, dy, dg, dw = In(capi, x, off), In(capi, y, off), In(capi, g, off), In(capi, w)
    rows = Out(capi, (n, width), off)
    capi.check(L.fz_expert_dispatch(rows.ptr, dx.ptr, dslot.ptr, dsrc.ptr, t, k, n, width, None))
    np.testing.assert_array_equal(rows.get(), O.dispatch(x, slot, n).astype(np.float32))

    clean = np.where(np.isnan(y), 0, y)
    out64, drows64, dw64 = O.combine(clean, w, slot, g)
    held = (slot >= 0)[..., None]
    terms = (np.abs(w)[..., None] * np.abs(clean)[np.maximum(slot, 0)] * held).sum(1)
    out = Out(capi, (t, width), off)
    capi.check(L.fz_expert_combine(out.ptr, dy.ptr, dw.ptr, dslot.ptr, t, k, n, width, None))
    close(out.get(), out64, (k + 1) * U * terms, "out")
    plain = Out(capi, (t, width), off)
    capi.check(L.fz_expert_combine(plain.ptr, dy.ptr, None, dslot.ptr, t, k, n, width, None))
    close(plain.get(), O.combine(clean, None, slot), (k + 1) * U * (np.abs(clean)[np.maximum(slot, 0)] * held).sum(1), "sum")

    drows, dweights = Out(capi, (n, width), off), Out(capi, (t, k))
    capi.check(L.fz_expert_combine_backward(drows.ptr, dweights.ptr, dg.ptr, dy.ptr, dw.ptr, dslot.ptr, dsrc.ptr, t, k, n,
                                            width, None))
    # one product, rounded once (a zero's sign aside)
    want = np.zeros((n, width), np.float32)
    for i, j in zip(*np.nonzero(slot >= 0)):
        want[slot[i, j]] = w[i, j] * g[i]
    np.testing.assert_array_equal(drows.get(), want)
    prods = (np.abs(g)[:, None] * np.abs(clean)[np.maximum(slot, 0)] * held).sum(2)
    close(dweights.get(), dw64, (width / 32 + 40) * U * prods, "dweights")
    only = Out(capi, (n, width), off)
    capi.check(L.fz_expert_combine_backward(only.ptr, None, dg.ptr, None, None, dslot.ptr, dsrc.ptr, t, k, n, width, None))
    np.testing.assert_array_equal(only.get(), O.dispatch(g, slot, n).astype(np.float32))


# rows of several passes of a warp, and of a CTA; empty rows beside them
@pytest.mark.parametrize("t,k,e,cap,width,off", [(1300, 4, 6, 0, 301, 0), (40, 2, 3, 35, 2500, 1), (3, 2, 4, 5, 9000, 0),
                                                 (700, 2, 5, 0, 770, 2), (20, 1, 4, 8, 1030, 0)])
def test_dispatch_and_combine_of_wide_rows(capi, t, k, e, cap, width, off):
    test_dispatch_and_combine(capi, t, k, e, cap, width, off)


def test_combine_passes_over_foreign_slots(capi):
    """A slot outside the rows is no choice: nothing is read or written for it."""
    L = capi.lib()
    slot, src = np.array([[0, 99], [-5, 1], [2 ** 31 - 1, 2]]), np.array([0, 3, 5])
    x = np.arange(24, dtype=np.float32).reshape(3, 8)
    a = {n: In(capi, v) for n, v in (("slot", slot), ("src", src), ("x", x), ("w", np.ones((3, 2))))}
    rows, out, dw = Out(capi, (3, 8)), Out(capi, (3, 8)), Out(capi, (3, 2))
    capi.check(L.fz_expert_dispatch(rows.ptr, a["x"].ptr, a["slot"].ptr, a["src"].ptr, 3, 2, 3, 8, None))
    np.testing.assert_array_equal(rows.get(), x)
    capi.check(L.fz_expert_combine(out.ptr, rows.ptr, a["w"].ptr, a["slot"].ptr, 3, 2, 3, 8, None))
    np.testing.assert_array_equal(out.get(), x)
    back = Out(capi, (3, 8))
    capi.check(L.fz_expert_combine_backward(back.ptr, dw.ptr, a["x"].ptr, rows.ptr, a["w"].ptr, a["slot"].ptr, a["src"].ptr, 3, 2,
                                            3, 8, None))
    np.testing.assert_array_equal(back.get(), x)
    np.testing.assert_array_equal(dw.get() != 0, [[True, False], [False, True], [False, True]])


def test_rows_past_32_bit_offsets(capi):
    """Rows whose element offsets pass 2^31 (2.2e9 floats, 8.6 GB each way)."""
    L = capi.lib()
    t, width, n = 64, 8192, 263000
    rng = np.random.default_rng(3)
    at = np.sort(rng.choice(n, t, replace=False))
    at[-1] = n - 1
    src = np.full(n, -1)
    src[at] = np.arange(t)
    x = rng.standard_normal((t, width)).astype(np.float32)
    rows = capi.DeviceArray((n, width))
    dx, dslot, dsrc = In(capi, x), In(capi, at[:, None]), In(capi, src)
    out = Out(capi, (t, width))
    capi.check(L.fz_expert_dispatch(rows.ptr, dx.ptr, dslot.ptr, dsrc.ptr, t, 1, n, width, None))
    capi.check(L.fz_expert_combine(out.ptr, rows.ptr, None, dslot.ptr, t, 1, n, width, None))
    np.testing.assert_array_equal(out.get(), x)
    most = capi.DeviceArray((n,))
    capi.check(L.fz_reduce(capi.REDOPS["max"], most.ptr, rows.ptr, n, width, 1, None))
    m = most.numpy()
    assert not m[src < 0].any()
    np.testing.assert_array_equal(m[at], x.max(1))
    rows.free()
    capi.check(L.fz_pool_release())


# ---------------------------------------------------------------- distillation


def distill_bounds(z, ids, teacher, tau, lse, dloss):
    """First-order bounds of the loss and dz, row by row; chains of at most V / 512 additions
    and as many rescalings (6 u each) a thread."""
    r, v = z.shape
    k = ids.shape[1]
    e_loss, e_dz = np.zeros(r), np.zeros((r, v))
    for i in range(r):
        held = (ids[i] >= 0) & (ids[i] < v)
        at, t = ids[i][held], teacher[i][held].astype(np.float64)
        if not held.any() or (lse is None and np.all(t == -np.inf)):
            continue
        z64 = z[i].astype(np.float64)

        def log_sum(x):
            m = x.max(initial=-np.inf)
            arg = np.where(np.isfinite(x), (x - m) / tau, 0)
            ex = np.where(np.isfinite(x), np.exp(arg), 0)
            s = ex.sum()
            err = U * ((ex * (4 * np.abs(arg) + 5)).sum() / s + v / 512 * 3 + 64) + 4 * U * abs(np.log(s))
            return m, np.log(s), err

        with np.errstate(all="ignore"):
            m, ls, e_ls = log_sum(z64)
            arg = np.where(np.isfinite(z64), (z64 - m) / tau, 0)
            q, e_q = np.where(np.isfinite(z64), np.exp(arg - ls), 0), 4 * U * np.abs(arg) + e_ls + 8 * U
            if lse is None:
                tm, tls, e_tls = log_sum(t)
                e_tls += k * U
                logp = (t - tm) / tau - tls
                e_p = np.where(np.isfinite(t), 4 * U * np.abs((t - tm) / tau) + e_tls + 4 * U, 0)
            else:
                logp = t / tau - np.float64(lse[i])
                e_p = np.where(np.isfinite(t), 3 * U * (np.abs(t / tau) + abs(float(lse[i]))) + 4 * U, 0)
            p = np.exp(logp)
            logq = arg[at] - ls
            gap = np.where(p > 0, np.abs(logp - logq), 0)
            e = (p * ((e_p + 6 * U) * gap + e_p + e_q[at])).sum() + k * U * (p * gap).sum()
            pt = 0.0
            e_pt = (p * e_p).sum() + (k / 32 + 16) * U * p.sum()
            g, e_g = np.zeros(v), np.zeros(v)
            if lse is not None:
                pt = max(0.0, 1 - p.sum())
                out = np.ones(v, bool)
                out[at] = False
                if pt > 0:
                    om, ol, e_ol = log_sum(z64[out])
                    lqt = (om - m) / tau + ol - ls
                    e += e_pt * (abs(np.log(pt) - lqt) + 1) + pt * (e_ol + e_ls + 8 * U * (abs(lqt) + abs(np.log(pt)) + 1))
                    qt = np.exp(np.where(np.isfinite(z64), (z64 - om) / tau - ol, -np.inf))
                    e_qt = 4 * U * np.abs(np.where(np.isfinite(z64), (z64 - om) / tau, 0)) + e_ol + 8 * U
                    e_g[out] += (pt * qt * (e_qt + 4 * U) + e_pt * qt)[out]
            mass = p.sum() + pt
            e_g += mass * q * (e_q + 4 * U) + (e_pt + 2 * U) * q + (k / 32 + 16) * U * q
            np.add.at(e_g, at, p * (e_p + (k + 4) * U))
            g = mass * q
            e_loss[i] = tau * tau * (e + 8 * U * (p * gap).sum())
            e_dz[i] = tau * abs(float(dloss[i])) * (e_g + 4 * U * g)
    return e_loss, e_dz


def run_distill(capi, z, ids, teacher, tau, lse, dloss, off=0, pitch=0):
    L = capi.lib()
    r, v = z.shape
    k = ids.shape[1]
    ld = v + pitch
    wide = np.full((r, ld), np.nan, np.float32)  # columns behind the vocabulary are never read
    wide[:, :v] = z
    a = [In(capi, wide, off), In(capi, ids), In(capi, teacher), In(capi, dloss)]
    dl = None if lse is None else In(capi, lse)
    loss, stats = Out(capi, (r,)), Out(capi, (r, 4))
    capi.check(L.fz_distill(loss.ptr, stats.ptr, a[0].ptr, ld, a[1].ptr, a[2].ptr, ptr(dl), r, v, k, tau, None))
    ldd = v + (pitch + 1 if pitch else 0)
    dz = Out(capi, (r, ldd), off)
    capi.check(L.fz_distill_backward(dz.ptr, ldd, a[3].ptr, stats.ptr, a[0].ptr, ld, a[1].ptr, a[2].ptr, ptr(dl), r, v, k,
                                     tau, None))
    got = dz.get()
    assert np.all(got[:, v:] == SENTINEL), "columns behind the vocabulary were written"
    return loss.get(), got[:, :v]


def distill_inputs(rng, r, v, k, tau, tail):
    z = (rng.standard_normal((r, v)) * 2).astype(np.float32)
    ids = np.stack([rng.permutation(v)[:k] for _ in range(r)])
    t = -np.sort(-(rng.standard_normal((r, k)) * 2 + 3).astype(np.float32))
    ids[rng.random((r, k)) < 0.1] = -1
    if r > 2:
        ids[1] = -1
        ids[2] = v + 5
    lse = None
    if tail:
        inside = np.where((ids >= 0) & (ids < v), np.exp(t.astype(np.float64) / tau), 0).sum(1)
        lse = np.log(np.maximum(inside, 1e-3) / rng.uniform(0.3, 0.99, r)).astype(np.float32)
    return z, ids, t, lse, (rng.standard_normal(r)).astype(np.float32)


# (rows, vocab, k, tau, alignment offset, extra pitch)
DISTILL_SHAPES = [(1, 1, 1, 1.0, 0, 0), (4, 5, 5, 2.0, 0, 0), (3, 130, 7, 1.0, 1, 0), (5, 1000, 64, 0.5, 0, 3), (2, 50001, 33, 4.0, 2, 0),
                  (1, 131072, 8, 1.0, 0, 0), (400, 515, 20, 2.0, 3, 2), (7, 32768, 256, 1.0, 0, 0), (3, 9000, 1024, 1.0, 0, 0),
                  (320, 4099, 3, 1.0, 0, 0), (2, 262144, 100, 2.0, 1, 1)]


@pytest.mark.parametrize("r,v,k,tau,off,pitch", DISTILL_SHAPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill(capi, r, v, k, tau, off, pitch, tail):
    z, ids, t, lse, g = distill_inputs(np.random.default_rng(v + k), r, v, k, tau, tail)
    loss, dz = run_distill(capi, z, ids, t, tau, lse, g, off, pitch)
    loss64, dz64 = O.distill(z, ids, t, tau, lse, g)
    e_loss, e_dz = distill_bounds(z, ids, t, tau, lse, g)
    close(loss, loss64, e_loss, "loss")
    close(dz, dz64, e_dz, "dz")
    again = run_distill(capi, z, ids, t, tau, lse, g, off, pitch)
    np.testing.assert_array_equal(loss.view(np.uint32), again[0].view(np.uint32))
    np.testing.assert_array_equal(dz.view(np.uint32), again[1].view(np.uint32))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_repeated_ids(capi, tail):
    """An id named twice counts its p twice, and its logit once; results do not vary."""
    rng = np.random.default_rng(21)
    z, ids, t, lse, g = distill_inputs(rng, 6, 3000, 40, 1.0, tail)
    ids = rng.integers(0, 12, ids.shape) * 250
    if tail:
        lse = np.log(np.exp(t.astype(np.float64)).sum(1) / 0.8).astype(np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    loss64, dz64 = O.distill(z, ids, t, 1.0, lse, g)
    e_loss, e_dz = distill_bounds(z, ids, t, 1.0, lse, g)
    close(loss, loss64, e_loss, "loss")
    close(dz, dz64, e_dz, "dz")
    for _ in range(3):
        again = run_distill(capi, z, ids, t, 1.0, lse, g)
        np.testing.assert_array_equal(dz.view(np.uint32), again[1].view(np.uint32))


# enough rows for a warp a row (short rows), 128 threads (medium ones), and for a backward that
# splits long rows
@pytest.mark.parametrize("r,v,k,tau,off,pitch", [(1300, 515, 20, 2.0, 3, 2), (1250, 90, 64, 1.0, 0, 0), (1190, 4096, 9, 1.0, 1, 0),
                                                 (460, 9000, 33, 0.5, 1, 1), (300, 131100, 9, 1.0, 0, 0)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_many_rows(capi, r, v, k, tau, off, pitch, tail):
    test_distill(capi, r, v, k, tau, off, pitch, tail)


# rows whose backward is cut into 1, 2, 4 and 8 pieces
@pytest.mark.parametrize("r,v,k,tau,off,pitch", [(300, 79999, 9, 1.0, 1, 0), (300, 80000, 9, 1.0, 0, 0), (300, 160001, 5, 2.0, 3, 2),
                                                 (297, 320003, 40, 1.0, 1, 1)])
def test_distill_pieces_of_many_rows(capi, r, v, k, tau, off, pitch):
    """Every 40th row against 64 bits; the columns behind a row stay as they were."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    gen = torch.Generator("cuda").manual_seed(9)
    ld, at = v + pitch, lambda t: t.data_ptr()  # noqa: E731
    flat = torch.randn(r * ld + off, generator=gen, device="cuda") * 2
    z = flat[off:].view(r, ld)
    ids = torch.stack([torch.randperm(v, generator=gen, device="cuda")[:k] for _ in range(r)]).to(torch.int32)
    ids[:, 0] = v - 1
    t = torch.randn(r, k, generator=gen, device="cuda")
    lse = (t / tau).logsumexp(1) + 0.4
    loss, stats, one = torch.empty(r, device="cuda"), torch.empty(r, 4, device="cuda"), torch.ones(r, device="cuda")
    out = torch.full((r * ld + off,), 7.0, device="cuda")
    dz = out[off:].view(r, ld)
    capi.check(L.fz_distill(at(loss), at(stats), at(z), ld, at(ids), at(t), at(lse), r, v, k, tau, 1))
    capi.check(L.fz_distill_backward(at(dz), ld, at(one), at(stats), at(z), ld, at(ids), at(t), at(lse), r, v, k, tau, 1))
    torch.cuda.synchronize()
    for i in range(0, r, 40):
        q = torch.log_softmax(z[i, :v].double() / tau, 0)
        p = torch.exp(t[i].double() / tau - lse[i].double())
        rest = 1 - p.sum()
        inside = torch.zeros(v, dtype=torch.bool, device="cuda")
        inside[ids[i].long()] = True
        tail = torch.logsumexp(q.masked_fill(inside, -torch.inf), 0)
        want = torch.where(inside, q.exp(), q.exp() * (1 - rest / tail.exp()))
        want[ids[i].long()] -= p
        # exp's argument (up to 20, twice rounded), a sum of up to v / 512 additions a thread, p and its rest
        bound = U * (4 * 20 + 3 * v / 512 + 100) * (want.abs() + q.exp() + p.sum() * inside)
        assert ((dz[i, :v].double() - want * tau).abs() <= tau * bound).all()
    if pitch:
        assert (dz[:, v:] == 7).all()
    assert (out[:off] == 7).all()
    del flat, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("r,v,k", [(1200, 300, 40), (1200, 300, 256), (450, 5000, 40), (9, 40000, 1000), (1, 20000, 1024)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_repeated_ids_of_each_team(capi, r, v, k, tail):
    """One id named by all of a row, by half of it, by two entries at its ends; none."""
    rng = np.random.default_rng(23)
    z, ids, t, lse, g = distill_inputs(rng, r, v, k, 1.0, False)
    ids = np.stack([rng.permutation(v) for _ in range(r)])[:, :k]
    ids[::4] = v - 1
    ids[1::4, ::2] = 0
    ids[2::4, 0] = ids[2::4, -1]
    if tail:
        lse = np.log(np.exp(t.astype(np.float64)).sum(1) / 0.8).astype(np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    loss64, dz64 = O.distill(z, ids, t, 1.0, lse, g)
    e_loss, e_dz = distill_bounds(z, ids, t, 1.0, lse, g)
    close(loss, loss64, e_loss, "loss")
    close(dz, dz64, e_dz, "dz")
    again = run_distill(capi, z, ids, t, 1.0, lse, g)
    np.testing.assert_array_equal(dz.view(np.uint32), again[1].view(np.uint32))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_masks(capi, tail):
    """Masked columns at -inf and at the type's lowest value; a row of nothing but the lowest
    value (a uniform student); a common offset of 10^4; rows whose logits are NaN but have no
    teacher; an entry of the teacher at -inf; a NaN in one row stays in it."""
    rng = np.random.default_rng(22)
    low = np.finfo(np.float32).min
    r, v, k = 8, 5000, 16
    z, ids, t, lse, g = distill_inputs(rng, r, v, k, 1.0, tail)
    ids = np.stack([rng.permutation(v)[:k] for _ in range(r)])
    keep = np.ones(v, bool)
    keep[rng.choice(v, 500, replace=False)] = False
    keep[ids[0]] = keep[ids[1]] = True
    z[0, ~keep] = -np.inf
    z[1, ~keep] = low
    z[2] = low
    z[3] += 10000
    z[4] = np.nan
    ids[4] = -1
    t[5, 3:] = -np.inf
    z[6, 17] = np.nan
    ids[7, 1:] = -1
    t[7] = -np.inf
    if tail:
        inside = np.where(ids >= 0, np.exp(t.astype(np.float64)), 0).sum(1)
        lse = np.log(np.maximum(inside, 1e-3) / 0.7).astype(np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    ok = np.array([0, 1, 2, 3, 4, 5, 7])
    loss64, dz64 = O.distill(z[ok], ids[ok], t[ok], 1.0, None if lse is None else lse[ok], g[ok])
    e_loss, e_dz = distill_bounds(z[ok], ids[ok], t[ok], 1.0, None if lse is None else lse[ok], g[ok])
    close(loss[ok], loss64, e_loss, "loss")
    close(dz[ok], dz64, e_dz, "dz")
    assert loss[4] == 0 and not dz[4].any()
    assert np.isnan(loss[6]) and np.isnan(dz[6]).all()
    if not tail:
        assert loss[7] == 0 and not dz[7].any()


# a warp, 128 threads, a CTA and a cluster a row; every column named, or the others masked
@pytest.mark.parametrize("r,v,k", [(1200, 64, 64), (1200, 256, 256), (300, 64, 64), (300, 1000, 1000), (3, 2000, 1024), (460, 6000, 100),
                                   (150, 6000, 64), (3, 40000, 64), (2, 40000, 1024)])
@pytest.mark.parametrize("mask", [-np.inf, np.finfo(np.float32).min, -1e6])
def test_distill_list_with_the_whole_mass(capi, r, v, k, mask):
    """The teacher's list holds its whole mass, and the student has none outside it: what rounding
    leaves of 1 - sum p is no mass. The result is that of the list alone; masked columns have no
    gradient."""
    rng = np.random.default_rng(r + v + k)
    z = (rng.standard_normal((r, v)) * 2).astype(np.float32)
    ids = np.stack([rng.permutation(v)[:k] for _ in range(r)])
    t = (rng.standard_normal((r, k)) * 2 + rng.uniform(-20, 20, (r, 1))).astype(np.float32)
    g = rng.standard_normal(r).astype(np.float32)
    outside = np.ones((r, v), bool)
    np.put_along_axis(outside, ids, False, 1)
    z[outside] = mask
    t64 = t.astype(np.float64)
    lse = (np.log(np.exp(t64 - t64.max(1, keepdims=True)).sum(1)) + t64.max(1)).astype(np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    loss64, dz64 = O.distill(z, ids, t, 1.0, None, g)
    e_loss, e_dz = distill_bounds(z, ids, t, 1.0, None, g)
    # p from lse in place of the list's own sum: lse is rounded, and so is the argument
    m = z.max(1, keepdims=True).astype(np.float64)
    logq = z - m - np.log(np.exp(z - m).sum(1, keepdims=True))
    logp = t64 - lse[:, None].astype(np.float64)
    p, at = np.exp(logp), np.take_along_axis(logq, ids, 1)
    e_p = p * (3 * U * (np.abs(t64) + np.abs(lse[:, None])) + 4 * U)
    e_loss = e_loss + (e_p * (np.abs(logp - at) + 1)).sum(1)
    more = np.exp(logq) * e_p.sum(1, keepdims=True)
    np.put_along_axis(more, ids, np.take_along_axis(more, ids, 1) + e_p, 1)
    close(loss, loss64, e_loss, "loss")
    close(dz, dz64, e_dz + np.abs(g[:, None]) * more, "dz")
    assert not dz[outside].any()


@pytest.mark.parametrize("r,v,k", [(1200, 300, 20), (5, 300, 20), (150, 6000, 20), (3, 40000, 64)])
def test_distill_mass_outside_that_the_student_lacks(capi, r, v, k):
    """A tail of the teacher where the student's columns are all at -inf: the loss is infinite, the
    entries' gradient is q - p, and the masked columns have none."""
    rng = np.random.default_rng(v + k)
    z = np.full((r, v), -np.inf, np.float32)
    ids = np.stack([rng.permutation(v)[:k] for _ in range(r)])
    np.put_along_axis(z, ids, (rng.standard_normal((r, k)) * 2).astype(np.float32), 1)
    t = rng.standard_normal((r, k)).astype(np.float32)
    lse = np.log(np.exp(t.astype(np.float64)).sum(1) / 0.7).astype(np.float32)
    g = rng.standard_normal(r).astype(np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    assert (loss == np.inf).all()
    z64 = np.take_along_axis(z, ids, 1).astype(np.float64)
    q, p = np.exp(z64) / np.exp(z64).sum(1, keepdims=True), np.exp(t.astype(np.float64) - lse[:, None])
    want = np.zeros((r, v))
    np.put_along_axis(want, ids, (q - p) * g[:, None], 1)
    # q: its argument |z - max| + log sum <= 20, 2^x, the sum; P and p as in distill_bounds
    close(dz, want, 200 * U * np.abs(g[:, None]) * (want != 0), "dz")


def test_distill_student_without_mass(capi):
    """The student gives a teacher's entry no probability: the loss is infinite, the gradient
    q - p is not."""
    z = np.zeros((1, 6), np.float32)
    z[0, 2] = -np.inf
    loss, dz = run_distill(capi, z, np.array([[2, 3]]), np.zeros((1, 2), np.float32), 1.0, None, np.ones(1, np.float32))
    assert loss[0] == np.inf
    close(dz, np.array([[.2, .2, -.5, -.3, .2, .2]]), 8 * U, "dz")


def test_distill_sure_student(capi):
    """The tail's mass far below one rounding of the whole: its log and gradient keep their
    digits."""
    rng = np.random.default_rng(23)
    z = (rng.standard_normal((3, 4000)) - 40).astype(np.float32)
    ids = np.stack([rng.permutation(4000)[:4] for _ in range(3)])
    np.put_along_axis(z, ids, np.float32(10), 1)
    t = np.zeros((3, 4), np.float32)
    lse = np.full(3, np.log(4 / 0.9), np.float32)
    g = np.ones(3, np.float32)
    loss, dz = run_distill(capi, z, ids, t, 1.0, lse, g)
    loss64, dz64 = O.distill(z, ids, t, 1.0, lse, g)
    e_loss, e_dz = distill_bounds(z, ids, t, 1.0, lse, g)
    close(loss, loss64, e_loss, "loss")
    close(dz, dz64, e_dz, "dz")
    # the tail's part: qT = 4000 e^(-40 + 1/2) / (4 e^10), 0.1 (log 0.1 - log qT) = 4.03; the
    # entries': 0.9 log(0.225 / 0.25) = -0.09
    assert np.all(loss64 > 3.9)


def test_distill_gradient_by_differences(capi):
    rng = np.random.default_rng(24)
    z, ids, t, lse, g = distill_inputs(rng, 4, 200, 6, 2.0, True)
    h = rng.standard_normal(z.shape).astype(np.float32)
    step = np.float32(2.0 ** -5)
    dz = run_distill(capi, z, ids, t, 2.0, lse, g)[1].astype(np.float64)
    f = lambda s: (run_distill(capi, z + s * h, ids, t, 2.0, lse, g)[0].astype(np.float64) * g).sum()  # noqa: E731
    slope = (f(step) - f(-step)) / (2 * float(step))
    f64 = lambda s: (O.distill(z + s * h.astype(np.float64), ids, t, 2.0, lse) * g).sum()  # noqa: E731
    d = lambda s: (f64(s) - f64(-s)) / (2 * s)  # noqa: E731
    s = float(step)
    e_loss, _ = distill_bounds(z, ids, t, 2.0, lse, g)
    # third-order term, the forward's roundings over the step, and the rounding of z + s h
    # (u |z| a value, through the gradient)
    bound = abs(d(2 * s) - d(s)) + 1.2 * (e_loss * np.abs(g)).sum() / s + U * (np.abs(dz) * (np.abs(z) + 1)).sum() / s
    assert abs(slope - (dz * h).sum()) <= bound


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("case", learn_cases.API_CASES, ids=lambda c: c.__name__)
def test_api(capi, case):
    import nova_b200

    # the model case runs through the framework's 3xTF32 products, held to 1e-5 norm-wise each;
    # four of them in a row, forward and back, add up
    if case is learn_cases.model_step:
        case(nova_b200.fusion, tol=4e-5)
    else:
        case(nova_b200.fusion)


def test_api_refusals(capi):
    import nova_b200

    learn_cases.refusals(nova_b200.fusion)


def test_two_streams_and_graph_replay(capi):
    """The same calls on a stream of the caller's, and captured into a CUDA graph that is
    replayed on new inputs, give the same bits as on the library's stream. Group norm in each
    of its forms: rows, a cluster a sample, two launches."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    gen = torch.Generator("cuda").manual_seed(1)
    norms = [(4, 70, 64, 8), (2, 4096, 64, 8), (1, 40000, 32, 2)]
    t, e, k, v, kt = 200, 16, 2, 5000, 12
    xs = [torch.randn(b, n, c, generator=gen, device="cuda") for b, n, c, _ in norms]
    z = torch.randn(t, e, generator=gen, device="cuda")
    lg = torch.randn(t, v, generator=gen, device="cuda")
    ids = torch.randint(0, v, (t, kt), generator=gen, device="cuda", dtype=torch.int32)
    teach = torch.randn(t, kt, generator=gen, device="cuda")
    sizes = [capi.group_norm_workspace(*s, True) for s in norms]

    def buffers():
        f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        i = lambda *s: torch.zeros(s, device="cuda", dtype=torch.int32)  # noqa: E731
        o = dict(w=f(t, k), ids=i(t, k), slot=i(t, k), src=i(t * k), counts=i(e), offs=i(e + 1), rows=f(t * k, e),
                 out=f(t, e), loss=f(t), stats=f(t, 4), dz=f(t, v), one=torch.ones(t, device="cuda"), dl=f(t, e))
        for q, (b, n, c, g) in enumerate(norms):
            o.update({f"y{q}": f(b, n, c), f"mean{q}": f(b, g), f"rstd{q}": f(b, g), f"dx{q}": f(b, n, c),
                      f"dg{q}": f(c), f"db{q}": f(c), f"work{q}": f(sizes[q] // 4 + 4)})
        return o

    def work(o, s):
        p = {a: q.data_ptr() for a, q in o.items()}
        for q, (b, n, c, g) in enumerate(norms):
            x = xs[q].data_ptr()
            capi.check(L.fz_group_norm(p[f"y{q}"], p[f"mean{q}"], p[f"rstd{q}"], x, None, None, b, n, c, g, 1e-5, 2,
                                       p[f"work{q}"], sizes[q], s))
            capi.check(L.fz_group_norm_backward(p[f"dx{q}"], p[f"dg{q}"], p[f"db{q}"], p[f"y{q}"], x, p[f"mean{q}"],
                                                p[f"rstd{q}"], None, None, b, n, c, g, 2, p[f"work{q}"], sizes[q], s))
        capi.check(L.fz_route(p["w"], p["ids"], z.data_ptr(), t, e, k, 1, s))
        capi.check(L.fz_route_backward(p["dl"], p["w"], p["w"], p["ids"], z.data_ptr(), t, e, k, 1, s))
        capi.check(L.fz_expert_sort(p["slot"], p["src"], p["counts"], p["offs"], p["ids"], t, k, e, 0, s))
        capi.check(L.fz_expert_dispatch(p["rows"], z.data_ptr(), p["slot"], p["src"], t, k, t * k, e, s))
        capi.check(L.fz_expert_combine(p["out"], p["rows"], p["w"], p["slot"], t, k, t * k, e, s))
        capi.check(L.fz_distill(p["loss"], p["stats"], lg.data_ptr(), v, ids.data_ptr(), teach.data_ptr(), None, t, v, kt, 1.5, s))
        capi.check(L.fz_distill_backward(p["dz"], v, p["one"], p["stats"], lg.data_ptr(), v, ids.data_ptr(), teach.data_ptr(), None,
                                         t, v, kt, 1.5, s))

    ref, side, cap = buffers(), buffers(), buffers()
    torch.cuda.synchronize()
    work(ref, None)
    stream = torch.cuda.Stream()
    work(side, stream.cuda_stream)
    capi.check(L.fz_stream_sync(None))
    torch.cuda.synchronize()
    same = lambda p, q: [a for a in p if not a.startswith("work")  # noqa: E731
                         and not torch.equal(p[a].view(torch.int32), q[a].view(torch.int32))]
    assert not same(ref, side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        work(cap, torch.cuda.current_stream().cuda_stream)
    for seed in (5, 6):
        for a in (*xs, z, lg, teach):
            a.normal_(generator=gen)
        torch.cuda.synchronize()
        graph.replay()
        work(ref, None)
        capi.check(L.fz_stream_sync(None))
        torch.cuda.synchronize()
        assert not same(ref, cap), seed
    del graph  # nothing captured outlives its buffers


FIRST_CALLS = """
import sys
import torch
from nova_b200 import capi
L = capi.lib()
b, n, c, g = 2, 4096, 64, 8  # a cluster a sample
x = torch.randn(b, n, c, device="cuda")
size = capi.group_norm_workspace(b, n, c, g, True)
work, stats, gb = torch.empty(size // 4 + 4, device="cuda"), torch.empty(2, b, g, device="cuda"), torch.empty(2, c, device="cuda")
y, dx, other = torch.empty_like(x), torch.empty_like(x), torch.zeros(4, device="cuda")
p = lambda t: t.data_ptr()
def call(s):
    capi.check(L.fz_group_norm(p(y), p(stats[0]), p(stats[1]), p(x), None, None, b, n, c, g, 1e-5, 2, p(work), size, s))
    capi.check(L.fz_group_norm_backward(p(dx), p(gb[0]), p(gb[1]), p(x), p(x), p(stats[0]), p(stats[1]), None, None, b, n, c, g, 2,
                                        p(work), size, s))
side, cap = torch.cuda.Stream(), torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=cap, capture_error_mode="global"):
    other += 1
    if sys.argv[1] == "beside":
        call(side.cuda_stream)
    else:
        call(cap.cuda_stream)
torch.cuda.synchronize()
graph.replay()
torch.cuda.synchronize()
assert (other == 1).all()
first = [t.clone() for t in (y, dx, gb)]
for t in (y, dx, gb):
    t.zero_()
torch.cuda.synchronize()
call(side.cuda_stream)
torch.cuda.synchronize()
assert all(torch.equal(u, v) for u, v in zip(first, (y, dx, gb)))
want = torch.nn.functional.silu(torch.nn.functional.group_norm(x.double().transpose(1, 2), g, eps=1e-5)).transpose(1, 2)
assert (y - want).abs().max() < 1e-4  # values up to 5: some 300 roundings, of sums at most 100 deep
capi.check(L.fz_kernel_status())
del graph
"""


@pytest.mark.parametrize("where", ["beside", "captured"])
def test_first_norm_of_a_process_during_a_capture(capi, where):
    """The first group norm of a process, while another stream is captured in the global mode
    (which forbids allocations in the whole process), and captured itself."""
    import os
    import pathlib
    import subprocess
    import sys

    pytest.importorskip("torch")
    root = pathlib.Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, where], cwd=root, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": str(root)})
    assert r.returncode == 0, r.stderr[-2000:]


def test_norm_and_distill_past_32_bit_offsets(capi):
    """More than 2^31 values: the last rows and samples come out as they do in a small call."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    s = 1  # the legacy default stream, torch's
    at = lambda t: t.data_ptr()  # noqa: E731
    new = lambda *n: torch.empty(n, device="cuda")  # noqa: E731

    def norm(x, dy, g, act):
        b, n, c = x.shape
        y, dx, mean, rstd, dg, db = torch.empty_like(x), torch.empty_like(x), new(b, g), new(b, g), new(c), new(c)
        size = capi.group_norm_workspace(b, n, c, g, True)
        work = new(size // 4 + 4)
        capi.check(L.fz_group_norm(at(y), at(mean), at(rstd), at(x), None, None, b, n, c, g, 1e-5, act, at(work), size, s))
        capi.check(L.fz_group_norm_backward(at(dx), at(dg), at(db), at(dy), at(x), at(mean), at(rstd), None, None, b, n, c, g, act,
                                            at(work), size, s))
        torch.cuda.synchronize()
        return y, dx

    gen = torch.Generator("cuda").manual_seed(2)
    for shape, g in (((530000, 1, 4096), 32), ((36, 250000, 256), 8)):
        x = torch.randn(shape, generator=gen, device="cuda")
        y, dx = norm(x, x, g, 2)
        few = x[-2:].clone()
        y_few, dx_few = norm(few, few, g, 2)
        assert torch.equal(y[-2:], y_few) and torch.equal(dx[-2:], dx_few)
        del x, y, dx
        torch.cuda.empty_cache()
    r, v, k = 17000, 131072, 8
    z = torch.randn(r, v, generator=gen, device="cuda")
    ids = torch.randint(0, v, (r, k), generator=gen, device="cuda", dtype=torch.int32)
    teach = torch.randn(r, k, generator=gen, device="cuda")
    one = torch.ones(r, device="cuda")

    def distill(a, b):
        n = b - a
        loss, stats, dz = new(n), new(n, 4), new(n, v)
        capi.check(L.fz_distill(at(loss), at(stats), at(z[a:]), v, at(ids[a:]), at(teach[a:]), None, n, v, k, 1.0, s))
        capi.check(L.fz_distill_backward(at(dz), v, at(one), at(stats), at(z[a:]), v, at(ids[a:]), at(teach[a:]), None, n, v, k, 1.0, s))
        torch.cuda.synchronize()
        return loss, dz

    loss, dz = distill(0, r)
    few, dz_few = distill(r - 600, r)
    # another number of rows may cut them otherwise: equal but for the order of the sums
    assert torch.allclose(loss[-600:], few, rtol=1e-5, atol=0)
    assert torch.allclose(dz[-600:], dz_few, rtol=1e-4, atol=1e-9)
    del z, dz, dz_few
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(530000, 1, 4096, 32), (36, 250000, 256, 8), (131073, 1, 16400, 2)], ids=str)
def test_norm_parameter_sums_past_32_bit_offsets(capi, shape):
    """More than 2^31 values: dbeta of ones is the number of rows, exactly; dgamma against 64 bits, within
    xh's roundings (sums of at most 32 rows, 16 levels and 16 joins, and its own) and the sum's
    (16 steps a block, at most 128 blocks, the fold's 56)."""
    torch = pytest.importorskip("torch")
    L = capi.lib()
    b, n, c, g = shape
    at = lambda t: t.data_ptr()  # noqa: E731
    x = torch.randn(b, n, c, generator=torch.Generator("cuda").manual_seed(4), device="cuda")
    dy, y = torch.ones_like(x), torch.empty_like(x)
    stats, gb = torch.empty(2, b, g, device="cuda"), torch.empty(2, c, device="cuda")
    size = capi.group_norm_workspace(b, n, c, g, True)
    work = torch.empty(size // 4 + 4, device="cuda")
    capi.check(L.fz_group_norm(at(y), at(stats[0]), at(stats[1]), at(x), None, None, b, n, c, g, 1e-5, 0, at(work), size, 1))
    # dx goes where y was
    capi.check(L.fz_group_norm_backward(at(y), at(gb[0]), at(gb[1]), at(dy), at(x), at(stats[0]), at(stats[1]), None, None, b, n, c, g, 0,
                                        at(work), size, 1))
    torch.cuda.synchronize()
    assert (gb[1] == b * n).all()
    del dy, y, work
    torch.cuda.empty_cache()
    total, size_of = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // (n * c))
    for lo in range(0, b, step):
        part = x[lo:lo + step].double().view(-1, n, g, c // g)
        var, mean = torch.var_mean(part, dim=(1, 3), keepdim=True, correction=0)
        xh = (part - mean) / torch.sqrt(var + 1e-5)
        total += xh.sum((0, 1)).view(c)
        size_of += xh.abs().sum((0, 1)).view(c)
    rows = b * n
    bound = (64 + 64 + 16 + 128 + 56) * U * (size_of + rows)  # rows: xh's error from the mean's
    assert ((gb[0].double() - total).abs() <= bound).all()
    del x
    torch.cuda.empty_cache()


def test_norms_from_two_threads(capi):
    """Two host threads, each on its own stream, whose first calls of several of the norm's kernels meet
    in the table of resident clusters."""
    import threading

    rng = np.random.default_rng(32)
    jobs = [[(rng.standard_normal(s[:3]).astype(np.float32), s[3]) for s in shapes] for shapes in
            ([(3, 1100, 36, 3), (2, 333, 72, 6), (1, 9001, 52, 4), (4, 77, 1000, 1), (2, 2, 9000, 1)],
             [(2, 2, 9004, 1), (4, 79, 1000, 1), (1, 9003, 52, 4), (2, 331, 72, 6), (3, 1102, 36, 3)])]
    got, errors = [[], []], []

    def work(q):
        try:
            capi.check(capi.lib().fz_set_device(0))
            for _ in range(5):
                got[q] = [run_norm(capi, x, None, None, g, 1e-5, "silu", x) for x, g in jobs[q]]
        except Exception as err:  # pragma: no cover
            errors.append(err)

    threads = [threading.Thread(target=work, args=(q,)) for q in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for q in range(2):
        for (x, g), res in zip(jobs[q], got[q]):
            for a, e in zip(res, run_norm(capi, x, None, None, g, 1e-5, "silu", x)):
                np.testing.assert_array_equal(a, e)


def test_calls_from_two_threads(capi):
    """Two host threads, each on its own stream, with their own buffers."""
    import threading

    rng = np.random.default_rng(30)
    jobs = [distill_inputs(rng, 20, 3000, 10, 1.0, True) for _ in range(2)]
    want = [run_distill(capi, z, i, t, 1.0, lse, g) for z, i, t, lse, g in jobs]
    got, errors = [None, None], []

    def work(q):
        try:
            capi.check(capi.lib().fz_set_device(0))
            z, i, t, lse, g = jobs[q]
            for _ in range(20):
                got[q] = run_distill(capi, z, i, t, 1.0, lse, g)
        except Exception as err:  # pragma: no cover
            errors.append(err)

    threads = [threading.Thread(target=work, args=(q,)) for q in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a[0], b[0])
        np.testing.assert_array_equal(a[1], b[1])
