"""Norms of queries and keys with their rotation, forward and backward, against the formulas in float64, element by element.

Bounds, with u = 2^-24 and uh half a step of the data's type (2^-11, 2^-8, 2^-24):
* a sum of D squares carries (D + 1) u, its mean and eps 2 u more; the inverse root halves that and adds 2 u of its own, so
  inv is off by ei = (D / 2 + 4) u of itself;
* z = x inv w: ei + 2 u; a turned value sums two products: 3 u more, in units of |a c| + |b s|; y rounds once more, uh;
* backward: g carries 2 u of G = |ga c| + |gb s|; xhat ei + u; g w xhat summed over D: ei + (D + 6) u; its mean times xhat
  and inv: 3 ei + (D + 12) u in units of inv (G w + |xhat| mean(G w |xhat|)), at most (5 / 2 D + 24) u; dx rounds, uh;
* dw sums n products: (n + 4) u + ei in units of the sum of G |xhat|;
* a binary16 result below 2^-14 is off by 2^-25.
"""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)

U = 2.0 ** -24
EPS = 1e-6
TYPES = ["fp16", "bf16", "fp32"]
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}


def store(x, t):
    """The values in the type's storage."""
    return x.astype(np.float32) if t == "fp32" else O.bf16_bits(x) if t == "bf16" else x.astype(np.float16).view(np.uint16)


def value(s, t):
    return s if t == "fp32" else (s.astype(np.uint32) << 16).view(np.float32) if t == "bf16" else s.view(np.float16).astype(np.float32)


class Case:
    def __init__(self, hip, B, S, H, Hkv, D, R, t="fp16", interleaved=False, positions=None, table=None, weights=True, packed=False,
                 pad=0, seed=1, std=2.0, grad=0.1):
        print(f"case {t} {B}x{S} heads {H}/{Hkv}x{D} rotary {R} interleaved={interleaved}", flush=True)
        self.hip, self.t, self.dims, self.R, self.inter = hip, t, (B, S, H, Hkv, D), R, interleaved
        self.rows = S if table is None else table
        self.size = 4 if t == "fp32" else 2
        rnd = lambda shape, k, s: value(store(O.randn(shape, seed + k, s), t), t)  # noqa: E731
        self.packed, self.pad = packed, pad
        self.widths = [(H + 2 * Hkv) * D + pad] if packed else [H * D + pad, Hkv * D + pad]
        self.first = [0, H * D] if packed else [0, 0]
        self.x = [rnd((B, S, w), i, std) for i, w in enumerate(self.widths)]
        self.g = [rnd((B, S, w), 4 + i, grad) for i, w in enumerate(self.widths)]
        self.w = [1 + O.randn((D,), seed + 8 + i, 0.2) for i in range(2)] if weights else [None, None]
        angle = np.arange(self.rows)[:, None] * 10000.0 ** (-np.arange(R // 2) * 2.0 / max(R, 1))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.positions = None if positions is None else np.asarray(positions, np.int32).reshape(B, S)
        up = lambda a: None if a is None or a.size == 0 else to_dev(hip, a)  # noqa: E731
        self.dx, self.dg = [up(store(a, t)) for a in self.x], [up(store(a, t)) for a in self.g]
        self.dw = [up(a) for a in self.w]
        self.dcos, self.dsin, self.dpos = up(self.cos), up(self.sin), up(self.positions)
        fresh = lambda: [up(np.full(a.shape, 1.5, np.float32) if t == "fp32" else np.full(a.shape, 0x1234, np.uint16)) for a in self.x]  # noqa: E731
        self.dy, self.dgx = fresh(), fresh()
        self.dgw = [to_dev(hip, np.full(D, np.nan, np.float32)) for _ in range(2)]

    def ptrs(self, bufs):
        return [None if bufs[0 if self.packed else i] is None else bufs[0 if self.packed else i].ptr + self.size * self.first[i]
                for i in range(2)]

    def strides(self):
        S = self.dims[1]
        w = self.widths * 2 if self.packed else self.widths
        return [w[0], w[0] * S, w[1], w[1] * S]

    def tables(self):
        return [*self.dw, self.dcos, self.dsin, self.dpos]

    def sizes(self):
        return [*self.dims, self.R, self.rows, EPS, self.inter, TYPES.index(self.t)]

    def forward(self):
        self.hip.HIPBackend.qkNormRotary(*self.ptrs(self.dx), *self.strides(), *self.tables(), *self.ptrs(self.dy), *self.strides(),
                                         *self.sizes())

    def backward(self):
        self.hip.HIPBackend.qkNormRotaryBackward(*self.ptrs(self.dg), *self.strides(), *self.ptrs(self.dx), *self.strides(),
                                                 *self.tables(), *self.ptrs(self.dgx), *self.dgw, *self.sizes())

    def results(self):
        return [b.numpy() for b in (*self.dy, *self.dgx, *self.dgw) if b is not None]

    def part(self, arrays, i):
        B, S, H, Hkv, D = self.dims
        n = (H, Hkv)[i]
        return arrays[0 if self.packed else i][:, :, self.first[i]:self.first[i] + n * D].reshape(B, S, n, D)

    def turned(self, x, sign=1.0):
        """Rotated values, and |a c| + |b s| of each."""
        B, S, H, Hkv, D = self.dims
        at = np.broadcast_to(np.arange(S), (B, S)) if self.positions is None else self.positions
        some = (at >= 0) & (at < self.rows)
        at = np.where(some, at, 0)
        y, size = x.copy(), np.abs(x)
        if self.R and self.rows:
            c = np.where(some[..., None], self.cos[at], 1.0)[:, :, None].astype(np.float64)
            s = np.where(some[..., None], self.sin[at], 0.0)[:, :, None].astype(np.float64) * sign
            i, j = (np.arange(0, self.R, 2), np.arange(1, self.R, 2)) if self.inter else \
                (np.arange(self.R // 2), np.arange(self.R // 2, self.R))
            a, b = x[..., i], x[..., j]
            y[..., i], y[..., j] = a * c - b * s, b * c + a * s
            size[..., i], size[..., j] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
        return y, size

    def check(self):
        B, S, H, Hkv, D = self.dims
        uh, tiny = HALF_STEP[self.t], 2.0 ** -25 if self.t == "fp16" else 1e-37
        ei = (D / 2 + 4) * U
        for i in range(2):
            if (H, Hkv)[i] == 0:
                continue
            x, g = self.part(self.x, i).astype(np.float64), self.part(self.g, i).astype(np.float64)
            w = np.ones(D) if self.w[i] is None else self.w[i].astype(np.float64)
            inv = 1 / np.sqrt((x * x).mean(3, keepdims=True) + np.float64(np.float32(EPS)))
            xhat = x * inv
            y, size = self.turned(xhat * w)
            got = value(np.ascontiguousarray(self.part([None if b is None else b.numpy() for b in self.dy], i)), self.t)
            lim = 1.01 * ((ei + 6 * U) * size + uh * np.abs(y)) + tiny
            off = np.abs(got - y)
            assert np.all(off <= lim), ("y", i, float((off / lim).max()))
            g, size = self.turned(g, -1.0)
            dx = inv * (g * w - xhat * (g * w * xhat).mean(3, keepdims=True))
            mass = inv * (size * np.abs(w) + np.abs(xhat) * (size * np.abs(w * xhat)).mean(3, keepdims=True))
            got = value(np.ascontiguousarray(self.part([None if b is None else b.numpy() for b in self.dgx], i)), self.t)
            lim = 1.01 * ((2.5 * D + 24) * U * mass + uh * np.abs(dx)) + tiny
            off = np.abs(got - dx)
            assert np.all(off <= lim), ("dx", i, float((off / lim).max()))
            dw = (g * xhat).sum((0, 1, 2))
            lim = 1.01 * ((B * S * (H, Hkv)[i] + 4) * U + ei) * (size * np.abs(xhat)).sum((0, 1, 2)) + 1e-37
            off = np.abs(self.dgw[i].numpy() - dw)
            assert np.all(off <= lim), ("dw", i, float((off / lim).max()))
        for bufs in (self.dy, self.dgx):   # nothing outside the heads' columns was touched
            for i, b in enumerate(bufs):
                if b is None:
                    continue
                used = (H + Hkv) * D if self.packed else (H, Hkv)[i] * D
                assert np.all(b.numpy()[:, :, used:] == (1.5 if self.t == "fp32" else 0x1234))


def run(hip, *dims, **kw):
    c = Case(hip, *dims, **kw)
    c.forward()
    c.backward()
    c.check()
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [8, 16, 24, 40, 64, 72, 96, 120, 128, 200, 256])
def test_head_dimensions(hip, D, t):
    """Whole heads turned, half of them, and none."""
    for R in {D, D // 16 * 8, 0}:
        run(hip, 2, 5, 3, 2, D, R, t=t, interleaved=D % 16 == 0, seed=D)
        run(hip, 2, 5, 3, 2, D, R, t=t, interleaved=D % 16 != 0, seed=D + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,Hkv", [(1, 1, 1, 1), (1, 1, 16, 4), (16, 1, 16, 4), (3, 7, 5, 1), (1, 333, 12, 12), (64, 20, 9, 3)],
                         ids=str)
def test_tokens_and_heads(hip, B, S, H, Hkv):
    for t in TYPES:
        run(hip, B, S, H, Hkv, 64, 64, t=t, seed=S)
        run(hip, B, S, H, Hkv, 64, 32, t=t, packed=True, pad=8, interleaved=True, seed=S)


@pytest.mark.gpu
def test_more_rows_than_a_grid(hip):
    """Every workgroup takes several rows; results large enough for streaming stores."""
    run(hip, 20, 2001, 12, 4, 64, 64, t="bf16", seed=2)
    run(hip, 2, 1500, 40, 8, 256, 256, t="fp32", seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions(hip, interleaved):
    """Far ones, the same twice, and ones outside the table, which leave a token unrotated."""
    p = [[-1, 0, 999, 1000, 5, 5], [2 ** 31 - 1, -2 ** 31, 1, 500, 998, 0]]
    c = run(hip, 2, 6, 3, 2, 64, 64, t="fp32", interleaved=interleaved, positions=p, table=1000, seed=4)
    y = c.part([b.numpy() for b in c.dy], 0)
    x = c.part(c.x, 0).astype(np.float64)
    z = x / np.sqrt((x * x).mean(3, keepdims=True) + EPS) * c.w[0]
    for b, s in ((0, 0), (0, 3), (1, 0), (1, 1)):
        assert np.allclose(y[b, s], z[b, s], rtol=1e-5, atol=1e-6)
    run(hip, 2, 6, 3, 2, 64, 64, table=0, seed=4)   # no table: nothing is turned
    run(hip, 2, 6, 3, 2, 64, 64, table=3, seed=4)   # a table shorter than the sequence


@pytest.mark.gpu
def test_queries_or_keys_alone_and_no_weights(hip):
    run(hip, 2, 9, 4, 0, 64, 64, seed=5)
    run(hip, 2, 9, 0, 4, 64, 64, seed=5)
    run(hip, 2, 9, 4, 2, 64, 64, weights=False, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_rows_of_zeros_small_and_large_values(hip, t):
    """inv is 1 / sqrt(eps) for a row of zeros; squares of 2^-60 and, but for binary16, of 1e15."""
    c = Case(hip, 1, 6, 2, 2, 64, 32, t=t, seed=6)
    for i in range(2):
        c.x[i][:, 0] = 0
        c.x[i][:, 1] *= 1e-3
        c.x[i][:, 2] *= 1e3 if t == "fp16" else 1e15
        c.x[i] = value(store(c.x[i], t), t)
        c.dx[i].upload(store(c.x[i], t))
    c.forward()
    c.backward()
    c.check()


@pytest.mark.gpu
def test_results_in_place(hip):
    for t in TYPES:
        c = run(hip, 3, 50, 6, 2, 64, 64, t=t, packed=True, seed=7)
        H = hip.HIPBackend
        H.qkNormRotaryBackward(*c.ptrs(c.dg), *c.strides(), *c.ptrs(c.dx), *c.strides(), *c.tables(), *c.ptrs(c.dg), None, None,
                               *c.sizes())
        H.qkNormRotary(*c.ptrs(c.dx), *c.strides(), *c.tables(), *c.ptrs(c.dx), *c.strides(), *c.sizes())
        for i in range(2):
            assert np.array_equal(c.part([b.numpy() for b in c.dx], i), c.part([b.numpy() for b in c.dy], i))
            assert np.array_equal(c.part([b.numpy() for b in c.dg], i), c.part([b.numpy() for b in c.dgx], i))


@pytest.mark.gpu
def test_outputs_with_strides_of_their_own(hip):
    """Tokens of all images in turn in the output, and rows past 32 bits of offset."""
    B, S, H, D = 3, 40, 4, 64
    c = run(hip, B, S, H, H, D, D, seed=8)
    w = H * D
    out = [empty_dev(hip, (S, B, w), np.uint16) for _ in range(2)]
    hip.HIPBackend.qkNormRotary(*c.ptrs(c.dx), *c.strides(), *c.tables(), *out, B * w, w, B * w, w, *c.sizes())
    far = 2 ** 31 + 64
    big = empty_dev(hip, (2 * far + S * w,), np.uint16)
    hip.HIPBackend.qkNormRotary(*c.ptrs(c.dx), *c.strides(), *c.tables(), big, out[1].ptr, w, far, B * w, w, *c.sizes())
    for i in range(2):
        assert np.array_equal(out[i].numpy().transpose(1, 0, 2), c.dy[i].numpy())
    row = empty_dev(hip, (S * w,), np.uint16)
    for b in range(B):
        hip.call("omHipCopyD2D", row.ptr, big.ptr + 2 * b * far, 2 * S * w)
        assert np.array_equal(row.numpy(), c.dy[0].numpy()[b].reshape(-1))


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the float64 loss sum(y * g) along random directions of x and w."""
    for inter in (False, True):
        c = run(hip, 2, 7, 3, 2, 32, 24 if inter else 32, t="fp32", interleaved=inter, seed=9)
        D = 32
        for i in range(2):
            x, w, g = (a.astype(np.float64) for a in (c.part(c.x, i), c.w[i], c.part(c.g, i)))

            def loss(x, w):
                z = x / np.sqrt((x * x).mean(3, keepdims=True) + np.float64(np.float32(EPS))) * w
                return (c.turned(z)[0] * g).sum()
            gx, gw = c.part([b.numpy() for b in c.dgx], i).astype(np.float64), c.dgw[i].numpy().astype(np.float64)
            e = 1e-5
            for k, at in enumerate((x, w)):
                d = O.randn(at.shape, 60 + k, 1.0).astype(np.float64)
                slope = (loss(x + e * d, w) - loss(x - e * d, w) if k == 0 else loss(x, w + e * d) - loss(x, w - e * d)) / (2 * e)
                mine = ((gx, gw)[k] * d).sum()
                size = (np.abs((gx, gw)[k]) * np.abs(d)).sum()
                # the gradient's own bound, 3 D u of it and of what it cancels (a few times its size); e^2 of a third
                # derivative and 1e-16 / e of rounding
                assert abs(mine - slope) <= 20 * D * U * size + 1e-7 * size + 1e-8


@pytest.mark.gpu
def test_repeats_agree_and_graphs_replay(hip, streams):
    c = Case(hip, 4, 197, 12, 4, 64, 64, seed=10)
    c.forward()
    c.backward()
    want = c.results()
    c.forward()
    c.backward()
    assert all(np.array_equal(a, b) for a, b in zip(want, c.results()))
    s = streams.create()
    hip.set_stream(s)
    c.forward()
    c.backward()
    streams.sync(s)
    graph = hip.Graph(lambda: (c.forward(), c.backward()))
    hip.set_stream(None)
    other = Case(hip, 2, 300, 4, 4, 128, 128, t="bf16", seed=11)
    try:
        for _ in range(3):
            for b in (*c.dy, *c.dgx):
                b.upload(np.full(b.shape, 0x1234, np.uint16))
            for b in c.dgw:
                b.upload(np.full(b.shape, np.nan, np.float32))
            hip.synchronize()
            graph.launch()
            other.forward()
            other.backward()
            streams.sync(s)
            hip.synchronize()
            assert all(np.array_equal(a, b) for a, b in zip(want, c.results()))
        other.check()
    finally:
        graph.destroy()


@pytest.mark.gpu
def test_nothing_to_do(hip):
    """No tokens: nothing is read, the weights' gradients are zeros."""
    gw = [to_dev(hip, np.full(64, np.nan, np.float32)) for _ in range(2)]
    s = [64, 64, 64, 64]
    for B, S in ((0, 5), (5, 0)):
        hip.HIPBackend.qkNormRotary(None, None, *s, *[None] * 5, None, None, *s, B, S, 1, 1, 64, 64, 0, EPS)
        hip.HIPBackend.qkNormRotaryBackward(None, None, *s, None, None, *s, *[None] * 5, None, None, *gw, B, S, 1, 1, 64, 64, 0, EPS)
        for g in gw:
            assert np.all(g.numpy() == 0)
            g.upload(np.full(64, np.nan, np.float32))


# ---------------------------------------------------------------- refusals: checked before anything touches a device
GOOD = dict(dtype=0, x=4096, g=4096, out=4096, ld=128, stride=1280, ldo=128, strideo=1280, w=4096, cos=4096, pos=4096, gw=4096,
            batch=2, seq=10, heads=2, kv=2, dim=64, rotary=64, table=10, eps=1e-6)
BAD = [dict(dtype=3), dict(dtype=-1), dict(x=None), dict(x=4104), dict(out=None), dict(out=4100), dict(ld=120), dict(ld=132),
       dict(stride=-8), dict(stride=1284), dict(w=4098), dict(cos=None), dict(cos=4097), dict(pos=4097), dict(batch=-1), dict(seq=-1),
       dict(heads=-1), dict(dim=4), dict(dim=60), dict(dim=264), dict(rotary=-8), dict(rotary=4), dict(rotary=72), dict(table=-1),
       dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(batch=2 ** 15, seq=2 ** 16)]


def call(om, a, back):
    x, strides = [a["x"]] * 2, [a["ld"], a["stride"]] * 2
    so = [a["ldo"], a["strideo"]] * 2
    tables = [a["w"], a["w"], a["cos"], a["cos"], a["pos"]]
    sizes = [a[k] for k in ("batch", "seq", "heads", "kv", "dim", "rotary", "table", "eps")] + [0]
    if back:
        om.call("omHipQkNormRotaryBackward", a["dtype"], a["g"], a["g"], *so, *x, *strides, *tables, a["out"], a["out"], a["gw"],
                a["gw"], *sizes)
    else:
        om.call("omHipQkNormRotary", a["dtype"], *x, *strides, *tables, a["out"], a["out"], *so, *sizes)


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    for back, name in ((False, "omHipQkNormRotary:"), (True, "omHipQkNormRotaryBackward:")):
        with pytest.raises(om.OmHipError, match=name):
            call(om, {**GOOD, **bad}, back)


@pytest.mark.parametrize("bad", [dict(g=None), dict(g=4104), dict(gw=4098), dict(ldo=120), dict(strideo=4)], ids=str)
def test_refusals_of_the_backward_pass(bad):
    import omnimatchdeeplearningtool_amd as om
    with pytest.raises(om.OmHipError, match="omHipQkNormRotaryBackward"):
        call(om, {**GOOD, **bad}, True)


def test_overlapping_results_are_refused():
    import omnimatchdeeplearningtool_amd as om
    for bad in (0, 64, 1272):
        with pytest.raises(om.OmHipError, match="overlap"):
            call(om, {**GOOD, "strideo": bad}, False)
        with pytest.raises(om.OmHipError, match="overlap"):
            call(om, {**GOOD, "stride": bad}, True)


def test_results_in_place_with_other_strides_are_refused():
    import omnimatchdeeplearningtool_amd as om
    with pytest.raises(om.OmHipError, match="in place"):
        call(om, {**GOOD, "ldo": 136, "strideo": 1360}, False)
    with pytest.raises(om.OmHipError, match="in place"):
        call(om, {**GOOD, "x": 8192, "ldo": 136, "strideo": 1360}, True)
