"""Group norm with an activation on channels-last data, forward and backward, against the formulas in float64.

Bounds (u = 2^-24, uh half a step of the type), for n values in a group:
* mean: its sum adds n values of size |x - k| in at most n roundings, (n + 4) u mean|x - k| + 2 u |mean|, with k one of
  the values: mean|x - k| <= 2 max|x - mean|. It is taken relative to the standard deviation: em = mean's error * inv.
* var: relative (2 n + 8) u of its sums where the pairwise joins lose nothing; inv half of it. The n of both is the
  longest run of additions, not the whole group: a thread's rows plus the joins, at most rows / 4 + chunks + 20 here;
  the tests use n itself, which is larger, capped at 4096 (a thread adds at most that many rows of these cases).
* xhat is off by em + |xhat| (ev + 3 u) with ev inv's relative error; z by |gamma| times that and 2 u |z|; the
  activations have slopes of at most 1.1 and the sigmoid's exp and division 8 u; the result rounds to the type.
* backward takes mean and inv as saved: xhat 3 u |xhat| (and 2 u |mean inv|: x - mean rounds), slopes 20 u, dz (n + 8) u of the sums' magnitudes; dx sums
  three terms and rounds.
"""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_dropout import HALF_STEP, TINY, store, value
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)

U = 2.0 ** -24
EPS = 1e-5


def act(z, a):
    return np.maximum(z, 0) if a == 1 else z / (1 + np.exp(-z)) if a == 2 else z


def slope(z, y, a):
    s = 1 / (1 + np.exp(-z))
    return (y > 0).astype(np.float64) if a == 1 else s * (1 + z * (1 - s)) if a == 2 else np.ones_like(z)


class Case:
    def __init__(self, hip, N, P, C, G, dt=2, a=0, affine=True, mean=0.5, std=1.5, seed=1, shift=0):
        print(f"case {N}x{P}x{C}/{G} dtype {dt} act {a}", flush=True)
        self.hip, self.dt, self.a, self.dims = hip, dt, a, (N, P, C, G)
        self.x = store(O.randn((N, P, C), seed, std) + np.float32(mean), dt)
        self.g = store(O.randn((N, P, C), seed + 1, 0.3), dt)
        self.gamma = O.randn((C,), seed + 2, 0.3) + np.float32(1) if affine else None
        self.beta = O.randn((C,), seed + 3, 0.3) if affine else None
        size = 4 if dt == 2 else 2
        self.off = shift * size   # elements by which x, y and the gradients lie off an allocation's start
        pad = lambda t: to_dev(hip, np.concatenate([np.zeros(shift, t.dtype), t.reshape(-1)]))  # noqa: E731
        self.shift = shift
        self.dx, self.dg = pad(self.x), pad(self.g)
        self.dgamma, self.dbeta = (None if t is None else to_dev(hip, t) for t in (self.gamma, self.beta))
        self.y, self.gx = (to_dev(hip, np.full(self.x.size + shift, 7, self.x.dtype)) for _ in range(2))
        self.mean, self.inv = empty_dev(hip, (N, G)), empty_dev(hip, (N, G))
        self.ggamma, self.gbeta = empty_dev(hip, (C,)), empty_dev(hip, (C,))

    def forward(self):
        self.hip.HIPBackend.groupNormNhwc(self.dx.ptr + self.off, self.dgamma, self.dbeta, self.y.ptr + self.off, self.mean, self.inv,
                                          *self.dims, EPS, self.a, self.dt)

    def backward(self):
        self.hip.HIPBackend.groupNormNhwcBackward(self.dg.ptr + self.off, self.dx.ptr + self.off, self.y.ptr + self.off if self.a == 1 else None,
                                                  self.mean, self.inv, self.dgamma, self.dbeta, self.gx.ptr + self.off, self.ggamma,
                                                  self.gbeta, *self.dims, self.a, self.dt)

    def results(self):
        return [t.numpy() for t in (self.y, self.mean, self.inv, self.gx, self.ggamma, self.gbeta)]

    def check(self):
        N, P, C, G = self.dims
        per, dt = C // G, self.dt
        uh = HALF_STEP[dt]
        x = value(self.x, dt).astype(np.float64).reshape(N, P, G, per)
        gamma = np.ones((G, per)) if self.gamma is None else self.gamma.astype(np.float64).reshape(G, per)
        beta = np.zeros((G, per)) if self.beta is None else self.beta.astype(np.float64).reshape(G, per)
        n = min(P * per, 4096)
        mu = x.mean((1, 3), keepdims=True)
        var = ((x - mu) ** 2).mean((1, 3), keepdims=True)
        inv = 1 / np.sqrt(var + EPS)
        spread = np.abs(x - mu).max((1, 3), keepdims=True)
        lim_mean = (n + 4) * U * 2 * spread + 2 * U * np.abs(mu)
        mean_k, inv_k = (t.numpy().astype(np.float64).reshape(N, 1, G, 1) for t in (self.mean, self.inv))
        assert np.all(np.abs(mean_k - mu) <= lim_mean)
        ev = (n + 8) * U + U + (lim_mean * inv) ** 2   # a wrong mean adds its square to the variance
        assert np.all(np.abs(inv_k - inv) <= ev * inv)
        xhat = (x - mu) * inv
        z = xhat * gamma + beta
        want = act(z, self.a)
        got = value(self.y.numpy()[self.shift:], dt).reshape(N, P, G, per)
        lim = 1.1 * (np.abs(gamma) * (lim_mean * inv + np.abs(xhat) * (ev + 3 * U) + U * np.abs(mu * inv)) + 2 * U * (np.abs(z) + np.abs(beta)))
        lim += 8 * U * np.abs(want) + uh * np.abs(want) * 1.01 + TINY[dt]
        assert np.all(np.abs(got - want) <= 1.01 * lim), float((np.abs(got - want) / lim).max())
        # backward, from the saved statistics and output
        xhat = (x - mean_k) * inv_k
        z = xhat * gamma + beta
        g = value(self.g, dt).astype(np.float64).reshape(N, P, G, per)
        dz = g * slope(z, got, self.a)
        exh = 3 * U * np.abs(xhat) + U * (np.abs(mean_k) + np.abs(x)) * inv_k
        edz = 20 * U * np.abs(g) + (0.6 * np.abs(g) * (np.abs(gamma) * exh + 2 * U * (np.abs(z) + np.abs(beta))) if self.a == 2 else 0.0)
        m = min(N * P, 4096)
        want = [(dz * xhat).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1)]
        lims = [((m + 8) * U * np.abs(dz * xhat) + edz * np.abs(xhat) + np.abs(dz) * exh).sum((0, 1)).reshape(-1),
                ((m + 8) * U * np.abs(dz) + edz).sum((0, 1)).reshape(-1)]
        for name, t, w, li in zip(("gamma", "beta"), (self.ggamma, self.gbeta), want, lims):
            assert np.all(np.abs(t.numpy() - w) <= 1.01 * li + 1e-30), name
        d = dz * gamma
        avg = lambda t: t.mean((1, 3), keepdims=True)  # noqa: E731
        s1, s2 = avg(d), avg(d * xhat)
        want = inv_k * (d - s1 - xhat * s2)
        e1 = avg((n + 8) * U * np.abs(d) + edz * np.abs(gamma))
        e2 = avg((n + 8) * U * np.abs(d * xhat) + edz * np.abs(gamma * xhat) + np.abs(d) * exh)
        lim = inv_k * (edz * np.abs(gamma) + e1 + np.abs(xhat) * e2 + exh * np.abs(s2) + 4 * U * (np.abs(d) + np.abs(s1) + np.abs(xhat * s2)))
        got = value(self.gx.numpy()[self.shift:], dt).reshape(N, P, G, per)
        lim = 1.01 * (lim + uh * np.abs(want) * 1.01) + TINY[dt]
        assert np.all(np.abs(got - want) <= lim), float((np.abs(got - want) / lim).max())


def run(hip, *dims, **kw):
    c = Case(hip, *dims, **kw)
    c.forward()
    c.backward()
    c.check()
    return c


# one pixel, one channel, groups of one to all channels, widths around the 8 channels of a thread and the 64, 256 and
# 512 of a workgroup, images of one row to many chunks
SIZES = [(1, 1, 1, 1), (2, 1, 16, 2), (1, 5, 7, 7), (3, 49, 15, 5), (2, 64, 8, 1), (1, 130, 24, 3), (2, 33, 64, 8), (1, 200, 72, 9),
         (2, 49, 480, 32), (1, 300, 257, 1), (4, 31, 512, 32), (1, 70, 520, 2), (2, 7, 2056, 4), (1, 5000, 16, 4), (3, 1000, 96, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(hip, size, dt):
    run(hip, *size, dt=dt, a=(sum(size) + dt) % 3, seed=sum(size))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("a", [0, 1, 2], ids=["none", "relu", "silu"])
def test_activations_and_no_affine(hip, a, dt):
    run(hip, 2, 100, 64, 8, dt=dt, a=a)
    run(hip, 2, 100, 64, 8, dt=dt, a=a, affine=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
def test_addresses_off_the_vector(hip, dt):
    run(hip, 2, 40, 64, 8, dt=dt, a=2, shift=1)
    run(hip, 2, 40, 33, 3, dt=dt, a=1, shift=3)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [128, 125], ids=str)
def test_large_output(hip, C):
    """Over 24 MB: streaming stores."""
    run(hip, 2, 26000, C, 1, dt=2, a=2)


@pytest.mark.gpu
def test_mean_far_above_the_spread(hip):
    """A mean of 1000 spreads: sums of squares alone would leave nothing of the variance."""
    run(hip, 2, 3000, 32, 4, dt=2, mean=1000.0, std=1.0)
    run(hip, 1, 20, 64, 2, dt=2, mean=-3000.0, std=0.5, a=2)


@pytest.mark.gpu
def test_constant_image_and_first_pixel_apart(hip):
    """No spread at all (inv is 1 / sqrt(eps)), and an image whose first pixel is far from the others."""
    c = Case(hip, 1, 200, 16, 2, seed=3)
    c.x[...] = 2.5
    c.dx.upload(c.x)
    c.forward()
    assert np.allclose(c.inv.numpy(), EPS ** -0.5, rtol=4 * U) and np.all(c.mean.numpy() == 2.5)
    assert np.array_equal(c.y.numpy().reshape(200, 16), np.broadcast_to(c.beta, (200, 16)))
    c = Case(hip, 1, 2000, 16, 2, seed=4, mean=100.0, std=1.0)
    c.x[0, 0] = 0.0
    c.dx.upload(c.x)
    c.forward()
    c.backward()
    c.check()


@pytest.mark.gpu
def test_nan_stays_in_its_group(hip):
    c = Case(hip, 2, 90, 32, 4, a=2)
    c.x[1, 17, 9] = np.nan
    c.dx.upload(c.x)
    c.forward()
    bad = np.isnan(c.y.numpy().reshape(2, 90, 4, 8))
    assert bad[1, :, 1].all() and bad.sum() == 90 * 8


@pytest.mark.gpu
def test_in_place_and_without_saved_statistics(hip):
    c = run(hip, 2, 150, 48, 6, dt=1, a=2)
    y, gx = c.y.numpy(), c.gx.numpy()
    place = to_dev(hip, c.x)
    hip.HIPBackend.groupNormNhwc(place, c.dgamma, c.dbeta, place, None, None, *c.dims, EPS, c.a, c.dt)
    assert np.array_equal(place.numpy().reshape(-1), y)
    place = to_dev(hip, c.g)
    hip.HIPBackend.groupNormNhwcBackward(place, c.dx, None, c.mean, c.inv, c.dgamma, c.dbeta, place, None, None, *c.dims, c.a, c.dt)
    assert np.array_equal(place.numpy().reshape(-1), gx)


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the float64 loss sum(y * g) along random directions; SiLU, whose slope is smooth."""
    c = run(hip, 2, 30, 24, 3, a=2, seed=5)
    N, P, C, G = c.dims
    at = [value(c.x, 2).astype(np.float64), c.gamma.astype(np.float64), c.beta.astype(np.float64)]

    def loss(x, gamma, beta):
        t = x.reshape(N, P, G, C // G)
        t = (t - t.mean((1, 3), keepdims=True)) / np.sqrt(t.var((1, 3), keepdims=True) + EPS)
        return (act(t.reshape(N, P, C) * gamma + beta, 2) * c.g).sum()

    for i, got in enumerate((c.gx.numpy().reshape(N, P, C), c.ggamma.numpy(), c.gbeta.numpy())):
        d = O.randn(at[i].shape, 60 + i, 1.0).astype(np.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * d, at[i] - 1e-5 * d
        fd = (loss(*up) - loss(*down)) / 2e-5
        # what check() allows an element is below 2000 u of the largest one; the difference itself is good to 1e-6
        assert abs((got * d).sum() - fd) <= 2000 * U * np.abs(got).max() * np.abs(d).sum() + 1e-6 * (1 + abs(fd))


@pytest.mark.gpu
def test_repeats_agree_and_graphs_replay(hip, streams):
    cases = [Case(hip, 2, 500, 64, 8, dt=0, a=1, seed=2), Case(hip, 1, 60, 100, 10, dt=2, a=2, seed=3)]
    want = []
    for c in cases:
        c.forward()
        c.backward()
        want.append(c.results())
    graphs = []
    for c in cases:
        s = streams.create()
        hip.set_stream(s)
        c.forward()
        c.backward()
        streams.sync(s)
        graphs.append((s, hip.Graph(lambda c=c: (c.forward(), c.backward()))))
    hip.set_stream(None)
    try:
        for _ in range(3):
            for c in cases:
                for t in (c.y, c.gx):
                    t.upload(np.full(t.shape, 7, t.dtype))
            hip.synchronize()
            for _, g in graphs:
                g.launch()
            run(hip, 1, 333, 40, 5, dt=1, a=1)
            for s, _ in graphs:
                streams.sync(s)
            for c, w in zip(cases, want):
                assert all(np.array_equal(a, b) for a, b in zip(w, c.results()))
    finally:
        for _, g in graphs:
            g.destroy()


@pytest.mark.gpu
def test_nothing_to_do(hip):
    H = hip.HIPBackend
    H.groupNormNhwc(None, None, None, None, None, None, 0, 4, 8, 2, EPS, 0)
    H.groupNormNhwc(None, None, None, None, None, None, 2, 0, 8, 2, EPS, 0)
    gg, gb = (to_dev(hip, np.ones(8, np.float32)) for _ in range(2))
    H.groupNormNhwcBackward(None, None, None, None, None, None, None, None, gg, gb, 0, 4, 8, 2, 0)
    assert np.all(gg.numpy() == 0) and np.all(gb.numpy() == 0)


GOOD = dict(dt=2, x=4096, y=4096, st=4096, n=1, p=4, c=8, g=2, eps=1e-5, a=0)
BAD = [dict(dt=3), dict(dt=-1), dict(x=None), dict(a=3), dict(a=-1), dict(g=0), dict(g=3), dict(n=-1), dict(p=-1), dict(c=-8),
       dict(n=65536), dict(c=2 ** 18 + 2), dict(p=2 ** 30 + 1), dict(x=4098), dict(dt=0, x=4097), dict(st=4098)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **bad}
    sizes = [a["n"], a["p"], a["c"], a["g"]]
    with pytest.raises(om.OmHipError, match="omHipGroupNormNhwc"):
        om.call("omHipGroupNormNhwc", a["dt"], a["x"], a["st"], a["st"], a["y"], a["st"], a["st"], *sizes, a["eps"], a["a"])
    with pytest.raises(om.OmHipError, match="omHipGroupNormNhwcBackward"):
        om.call("omHipGroupNormNhwcBackward", a["dt"], a["x"], a["x"], a["x"], a["st"], a["st"], a["st"], a["st"], a["y"], a["st"],
                a["st"], *sizes, a["a"])


def test_more_refusals():
    import omnimatchdeeplearningtool_amd as om
    with pytest.raises(om.OmHipError, match="eps"):
        om.call("omHipGroupNormNhwc", 2, 4096, None, None, 4096, None, None, 1, 4, 8, 2, -1.0, 0)
    with pytest.raises(om.OmHipError, match="saved output"):
        om.call("omHipGroupNormNhwcBackward", 2, 4096, 4096, None, 4096, 4096, None, None, 4096, None, None, 1, 4, 8, 2, 1)
    with pytest.raises(om.OmHipError, match="null"):
        om.call("omHipGroupNormNhwcBackward", 2, 4096, 4096, None, None, 4096, None, None, 4096, None, None, 1, 4, 8, 2, 0)


def far_case(hip, size, dt, spread):
    """A mean of 1e20: its square has no fp32 value."""
    c = Case(hip, *size, dt=dt, seed=7)
    c.x = store(np.float32(1e20) + O.randn(c.x.shape, 7, 1.0) * np.float32(spread), dt)
    c.dx.upload(c.x)
    c.forward()
    c.backward()
    return c


FAR = [(3, 20, 64, 8), (1, 20, 60, 4), (2, 300, 12, 4), (1, 400, 64, 1),   # one launch, one launch of one image, three launches
       (1, 650, 1000, 1)]                                                      # several waves join a group


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [1, 2], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", FAR, ids=str)
def test_constant_image_far_from_zero(hip, size, dt):
    """1e20 everywhere: mean is the value itself, inv 1 / sqrt(eps), xhat 0, so y is beta, dgamma 0 and dbeta the sums."""
    c = far_case(hip, size, dt, 0.0)
    N, P, C, G = size
    y, mean, inv, gx, ggamma, gbeta = c.results()
    assert np.all(mean == value(c.x, dt)[0, 0, 0]) and np.allclose(inv, EPS ** -0.5, rtol=4 * U, atol=0)
    assert np.array_equal(value(y, dt).reshape(N, P, C), np.broadcast_to(value(store(c.beta, dt), dt), (N, P, C)))
    g = value(c.g, dt).astype(np.float64)
    assert np.all(ggamma == 0)
    assert np.all(np.abs(gbeta - g.sum((0, 1))) <= 1.01 * (N * P + 8) * U * np.abs(g).sum((0, 1)))
    d = (g * c.gamma).reshape(N, P, G, C // G)
    avg = lambda t: t.mean((1, 3), keepdims=True)  # noqa: E731
    want = EPS ** -0.5 * (d - avg(d))
    lim = EPS ** -0.5 * ((P * C // G + 8) * U * avg(np.abs(d)) + 8 * U * (np.abs(d) + np.abs(avg(d)))) + HALF_STEP[dt] * np.abs(want)
    assert np.all(np.abs(value(gx, dt).reshape(want.shape) - want) <= 1.01 * lim)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [1, 2], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", FAR[:3], ids=str)
def test_spread_far_from_zero(hip, size, dt):
    """1e20 +- 3e17. At most 16 joins lie between a value and its group (5 of row threads, one or two of a lane's entries,
    6 of lanes, chunks): each rounds the mean, u |mean|, on top of the sums' (n + 4) u. A mean that is off by e moves a
    join's squared difference by 2 e |mb - ma|; over 16 of them, by Cauchy-Schwarz, 2 sqrt(16) e / std of the variance and
    e^2 / var, half of which is inv's."""
    c = far_case(hip, size, dt, 3e17)
    N, P, C, G = size
    per, n, joins = C // G, P * C // G, 16
    x = value(c.x, dt).astype(np.float64).reshape(N, P, G, per)
    y, mean, inv, gx, ggamma, gbeta = c.results()
    avg = lambda t: t.mean((1, 3), keepdims=True)  # noqa: E731
    mu = avg(x)
    sd = np.sqrt(avg((x - mu) ** 2))
    em = (n + 4) * U * 2 * np.abs(x - mu).max((1, 3), keepdims=True) + (joins + 2) * U * np.abs(mu)
    mean, inv = (t.astype(np.float64).reshape(N, 1, G, 1) for t in (mean, inv))
    ev = (n + 8) * U + joins ** 0.5 * em / sd + (em / sd) ** 2
    assert ev.max() < 2.0 ** -8
    assert np.all(np.abs(mean - mu) <= em)
    assert np.all(np.abs(inv * sd - 1) <= ev)
    gamma, beta = (t.astype(np.float64).reshape(G, per) for t in (c.gamma, c.beta))
    xhat = (x - mu) / sd
    want = xhat * gamma + beta
    lim = np.abs(gamma) * (em / sd + np.abs(xhat) * (ev + 3 * U)) + 3 * U * (np.abs(want) + np.abs(beta)) + HALF_STEP[dt] * np.abs(want)
    assert np.all(np.abs(value(y, dt).reshape(want.shape) - want) <= 1.01 * lim)
    # from the saved statistics: x - mean is exact (neighbours of each other) but for a rounding of the result
    xhat = (x - mean) * inv
    g = value(c.g, dt).astype(np.float64).reshape(x.shape)
    d = g * gamma
    want = inv * (d - avg(d) - xhat * avg(d * xhat))
    e2 = (n + 10) * U * avg(np.abs(d * xhat))
    lim = inv * ((n + 8) * U * avg(np.abs(d)) + np.abs(xhat) * e2 + 5 * U * (np.abs(d) + np.abs(avg(d)) + np.abs(xhat * avg(d * xhat))))
    lim += (HALF_STEP[dt] + 2 * U) * np.abs(want) + 2.0 ** -126   # its size is 1e-18: no subnormals
    assert np.all(np.abs(value(gx, dt).reshape(want.shape) - want) <= 1.01 * lim)
    for got, t in ((ggamma, g * xhat), (gbeta, g)):
        assert np.all(np.abs(got - t.sum((0, 1)).reshape(-1)) <= 1.01 * (N * P + 12) * U * np.abs(t).sum((0, 1)).reshape(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 1, 8, 8), (2, 1, 16, 16), (1, 300, 8, 8)], ids=str)
def test_infinity_is_no_constant(hip, size):
    """Groups that one thread's rows make up: an infinity leaves no deviation, so inv and the group's values are NaN."""
    c = Case(hip, *size)
    N, P, C, G = size
    c.x[0, P - 1, 3] = np.inf
    c.x[0, 0, 5] = -np.inf
    c.dx.upload(c.x)
    c.forward()
    y, inv = c.y.numpy().reshape(N, P, C), c.inv.numpy()
    bad = np.zeros((N, C), bool)
    bad[0, [3, 5]] = True
    assert np.array_equal(np.isnan(inv), bad)
    assert np.array_equal(np.isnan(y), np.broadcast_to(bad[:, None], y.shape))


@pytest.mark.gpu
def test_more_groups_than_one_dimension_of_a_grid(hip):
    """65535 images of 1025 groups: 2^26 pairs and more, 16 of them a workgroup of 1024 threads in the backward's join.
    Images repeat after 61, so 61 of them are the reference."""
    N, P, C, G, dt = 65535, 1, 4100, 1025, 0
    some, per = 61, C // G
    print(f"case {N}x{P}x{C}/{G}", flush=True)
    x, g = (store(O.randn((some, C), k, 1.0), dt) for k in (1, 2))
    every = np.arange(N) % some
    dx, dg = to_dev(hip, x[every]), to_dev(hip, g[every])
    y, gx = empty_dev(hip, (N, C), np.uint16), empty_dev(hip, (N, C), np.uint16)
    mean, inv = empty_dev(hip, (N, G)), empty_dev(hip, (N, G))
    gamma = O.randn((C,), 3, 0.3) + np.float32(1)
    dgamma, ggamma, gbeta = to_dev(hip, gamma), empty_dev(hip, (C,)), empty_dev(hip, (C,))
    hip.HIPBackend.groupNormNhwc(dx, dgamma, None, y, mean, inv, N, P, C, G, EPS, 0, dt)
    hip.HIPBackend.groupNormNhwcBackward(dg, dx, None, mean, inv, dgamma, None, gx, ggamma, gbeta, N, P, C, G, 0, dt)
    got = gx.numpy()
    assert np.array_equal(got, got[every])
    v = value(x, dt).astype(np.float64).reshape(some, G, per)
    mu = v.mean(2, keepdims=True)
    s = 1 / np.sqrt(((v - mu) ** 2).mean(2, keepdims=True) + EPS)
    xhat = (v - mu) * s
    w = value(g, dt).astype(np.float64).reshape(some, G, per)
    d = w * gamma.reshape(G, per)
    avg = lambda t: t.mean(2, keepdims=True)  # noqa: E731
    want = s * (d - avg(d) - xhat * avg(d * xhat))
    # the saved mean and inv are off by (n + 4) u spread and (2 n + 8) u; 64 u of the terms covers four values a group
    size = s * (np.abs(d) + avg(np.abs(d)) + (1 + np.abs(xhat)) * (1 + s * np.abs(v).max(2, keepdims=True)) * avg(np.abs(d) * (1 + np.abs(xhat))))
    off = np.abs(value(got[:some], dt).reshape(want.shape) - want)
    assert np.all(off <= 1.01 * (64 * U * size + HALF_STEP[dt] * np.abs(want)) + TINY[dt])
    times = np.bincount(every, minlength=some)[:, None]
    for name, out, t in (("gamma", ggamma, w * xhat), ("beta", gbeta, w)):
        t, most = t.reshape(some, C), (np.abs(w) * (1 + np.abs(xhat)) * (1 + s * np.abs(v).max(2, keepdims=True))).reshape(some, C)
        # 32 runs of at most N / 32 additions, then 5
        assert np.all(np.abs(out.numpy() - (t * times).sum(0)) <= 1.01 * (N // 32 + 70) * U * (most * times).sum(0)), name


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1], ids=["fp16", "bf16"])
@pytest.mark.parametrize("a,C", [(1, 128), (2, 125), (1, 125)], ids=str)
def test_large_output_in_half_precision(hip, a, C, dt):
    """Over 24 MB of 16-bit values: streaming stores, whole groups of 8 channels and not, ReLU's saved output among the
    inputs."""
    run(hip, 2, 51000, C, 1, dt=dt, a=a)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [1, 2], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [(1, 5000, 256, 1), (1, 701, 2040, 1), (2, 900, 1000, 2), (1, 3001, 1030, 10), (3, 257, 1536, 3)], ids=str)
def test_few_wide_groups(hip, size, dt):
    """Groups whose partial sums several waves join: last chunks of fewer rows, widths that are no multiple of 8."""
    run(hip, *size, dt=dt, a=sum(size) % 3, seed=sum(size))
    run(hip, *size, dt=dt, mean=50.0, affine=False, seed=sum(size) + 1)
