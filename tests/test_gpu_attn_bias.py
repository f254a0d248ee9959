"""Attention with a learned bias by relative position, forward and backward, against the formulas in float64, element by
element (attn_views says how far off a result may be)."""
import numpy as np
import pytest

import oracle as O
from attn_views import F, Viewed
from conftest import empty_dev, to_dev
from test_gpu_attn_train import Case, U, bits, value
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)


class Bias(Viewed):
    """where: "line" (positions None), or arrays of the queries' and the keys' positions. buckets: the map; zero: its entry of
    the difference 0."""

    def __init__(self, hip, *dims, buckets, zero, n_buckets=None, where="line", table_std=0.7, **kw):
        super().__init__(hip, *dims, **kw)
        B, Sq, Sk, H, Hkv, D = dims
        self.buckets, self.zero = np.asarray(buckets, np.int32), zero
        self.n = int(self.buckets.max()) + 1 if n_buckets is None else n_buckets
        self.table = O.randn((self.n, H), self.seed + 31, table_std)
        self.where = None if isinstance(where, str) else [np.asarray(x, np.int32) for x in where]
        self.dtable, self.dbuckets = to_dev(hip, self.table), to_dev(hip, self.buckets)
        self.dwhere = [None, None] if self.where is None else [to_dev(hip, x) for x in self.where]
        self.dgtable = to_dev(hip, np.full((self.n, H), np.nan, np.float32))

    def bias_args(self):
        return [self.dtable, self.dbuckets, *self.dwhere, self.n, len(self.buckets), self.zero]

    def forward(self):
        self.hip.HIPBackend.attentionBiasForwardHalf(*self.args(), *self.bias_args(), self.dout, self.dlse, *self.dims, self.scale,
                                                     bf16=self.bf16)

    def backward(self):
        self.hip.HIPBackend.attentionBiasBackwardHalf(*self.args(), *self.bias_args(), self.dout, self.dlse, self.dgrad,
                                                      *self.ptrs(self.dgrads), self.dgtable, *self.dims, self.scale,
                                                      bf16=self.bf16)

    def results(self):
        return super().results() + [self.dgtable.numpy()]

    def bucket_of(self, b):
        """Each pair's bucket, -1 where it has none."""
        B, Sq, Sk, *_ = self.dims
        nq, nk = self.sizes(b)
        qa, ka = (np.arange(Sq) + nk - nq, np.arange(Sk)) if self.where is None else [x.astype(np.int64) for x in self.where]
        which = self.buckets[np.clip(qa[:, None] - ka[None] + self.zero, 0, len(self.buckets) - 1)]
        return np.where((which >= 0) & (which < self.n), which, -1)

    def bias(self, b, h):
        which = self.bucket_of(b)
        return np.where(which < 0, 0.0, self.table[which, h].astype(np.float64))

    def seen(self, b):
        return self.standing(b)[0]

    def table_sums(self, b, h, dS, e, see):
        which = self.bucket_of(b)
        some = which >= 0
        for a, x in zip(self.sums, (dS, e, see, np.abs(dS))):
            np.add.at(a[:, h], which[some], np.asarray(x, np.float64)[some])

    def check(self):
        """Also the table's gradient and its bound."""
        self.sums = [np.zeros((self.n, self.dims[3])) for _ in range(4)]
        got, bound = super().check()
        want, e, n, mass = self.sums
        gt, lim = self.dgtable.numpy(), 1.01 * (e + (n + 4) * U * mass) + F
        assert np.all(np.abs(gt - want) <= lim), ("dtable", float((np.abs(gt - want) / lim).max()))
        return got, bound, gt, lim


def run(hip, *dims, **kw):
    c = Bias(hip, *dims, **kw)
    c.forward()
    c.backward()
    return c, c.check()


def line(far, n):
    """Differences -far .. far in n buckets: one each around 0, then wider ones."""
    d = np.arange(-far, far + 1)
    return dict(buckets=np.minimum(np.sign(d) * np.sqrt(np.abs(d)).astype(int) + n // 2, n - 1).clip(0), zero=far, n_buckets=n)


def grid(side, class_token=False):
    wide = 2 * side - 1
    at = (np.arange(side)[:, None] * wide + np.arange(side)).reshape(-1)
    if class_token:
        at = np.concatenate([[1 << 20], at])
    n = wide * wide + 2
    return dict(buckets=np.arange(n), zero=(side - 1) * wide + side, where=(at, at))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 8), (1, 200), (31, 33), (32, 32), (63, 65), (64, 64), (65, 129), (129, 127), (200, 1),
                                   (257, 300)], ids=str)
def test_lengths(hip, Sq, Sk, bf16):
    run(hip, 1, Sq, Sk, 2, 2, 64, bf16=bf16, seed=10 * Sq + Sk, **line(40, 13))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 70), (40, 40), (130, 130), (200, 90), (90, 200), (300, 300)], ids=str)
def test_causal(hip, Sq, Sk):
    """Sq > Sk leaves the first rows without a key."""
    run(hip, 2, Sq, Sk, 2, 1, 64, bf16=Sq % 4 == 0, causal=True, seed=Sq + Sk, **line(33, 9))


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0, 1, 5, 31, 32, 63, 64, 100, 250, 400])
def test_reach_of_the_map(hip, far):
    """From one offset to more than the sequence has: differences past the map take its ends, tile after tile."""
    run(hip, 1, 270, 330, 2, 1, 32, bf16=far % 2 == 0, seed=far, **line(far, 11))


@pytest.mark.gpu
@pytest.mark.parametrize("class_token", [False, True])
@pytest.mark.parametrize("side,D", [(1, 16), (2, 32), (7, 32), (9, 64), (14, 64), (11, 128)], ids=str)
def test_grids(hip, side, D, class_token):
    n = side * side + class_token
    run(hip, 3, n, n, 3, 3, D, packed=True, bf16=D == 128, seed=side, **grid(side, class_token))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 64, 72, 96, 104, 128])
def test_head_dimensions(hip, D, bf16):
    run(hip, 2, 70, 150, 4, 2, D, bf16=bf16, causal=D % 16 == 0, seed=D, **line(60, 15))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (6, 1), (9, 3)], ids=str)
def test_shared_heads_packed_and_padded_rows(hip, H, Hkv):
    """Query heads that share a key head have biases of their own."""
    run(hip, 3, 77, 77, H, Hkv, 40, packed=True, pad=16, causal=True, seed=H, **line(30, 9))
    run(hip, 2, 50, 141, H, Hkv, 128, bf16=True, pad=8, seed=H + 1, **line(90, 21))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk,H,Hkv,D", [(1, 2000, 2, 1, 64), (5, 1500, 4, 4, 128), (1500, 5, 3, 1, 64), (700, 700, 4, 1, 96)],
                         ids=str)
def test_walks_shared_by_workgroups(hip, Sq, Sk, H, Hkv, D, causal):
    run(hip, 3, Sq, Sk, H, Hkv, D, bf16=D > 64, causal=causal, klens=[Sk, 0, Sk // 3], qlens=[Sq, Sq, (Sq + 1) // 2],
        seed=Sq + D, **line(100, 25))


@pytest.mark.gpu
def test_many_images_share_workgroups(hip):
    """More images than a head's workgroups of dQ: each adds several images' dS."""
    lens = [(5 * i) % 27 for i in range(1000)]
    run(hip, 1000, 25, 25, 3, 3, 16, packed=True, seed=5, qlens=lens, klens=lens, **grid(5))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_per_image(hip, causal):
    """Each image's last query stands at its last key."""
    run(hip, 8, 150, 250, 2, 1, 64, bf16=causal, causal=causal, qlens=[0, 1, 150, 64, 33, -5, 400, 100],
        klens=[150, 1, 0, 165, 250, 20, 400, 20], seed=3, **line(50, 9))


@pytest.mark.gpu
def test_what_lies_past_a_length_is_not_read(hip):
    c = Bias(hip, 2, 100, 140, 2, 2, 64, qlens=[37, 100], klens=[70, 129], seed=5, **line(20, 9))
    for i, lens in ((0, c.qlens), (1, c.klens), (2, c.klens)):
        t = bits(c.store[i], False)
        for b in range(2):
            t[b, lens[b]:] = 0x7fff
        c.dev[i].upload(t)
    g = bits(c.grad, False)
    g[0, 37:] = 0x7fff
    c.dgrad.upload(g)
    c.forward()
    c.backward()
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(hip, scale):
    run(hip, 1, 70, 200, 2, 2, 64, scale=scale, seed=9, **line(30, 9))
    run(hip, 1, 70, 200, 2, 2, 64, scale=scale, bf16=True, table_std=20.0, seed=9, **line(30, 9))


@pytest.mark.gpu
def test_biases_that_hide_keys(hip):
    """-inf, the type's lowest value and -1e30 hide a bucket's keys; rows of them alone are empty. Large finite ones do not."""
    for hide in (-np.inf, np.finfo(np.float32).min, -1e30):
        c = Bias(hip, 1, 150, 150, 2, 1, 64, causal=True, seed=8, **line(40, 9))
        c.table[[0, 2, 4, 5], 0] = hide   # head 0: the own position, some behind
        c.table[:, 1] = hide              # head 1: everything
        c.table[3, 0] = -1e4
        c.dtable.upload(c.table)
        c.forward()
        c.backward()
        c.check()
        assert np.isneginf(c.dlse.numpy()[0, 1]).all() and np.isneginf(c.dlse.numpy()[0, 0, 0])


@pytest.mark.gpu
def test_offsets_without_a_bucket_add_nothing(hip):
    b = line(30, 9)
    b["buckets"] = b["buckets"].copy()
    b["buckets"][::3] = -1
    b["buckets"][1::7] = 9
    c, (_, _, got, _) = run(hip, 2, 90, 90, 2, 2, 32, seed=3, **b)
    assert np.isfinite(got).all()


@pytest.mark.gpu
def test_positions_of_any_value(hip):
    """Differences past 32 bits, all tokens in one place, and maps whose zero lies outside."""
    top = 2 ** 31 - 1
    where = (np.array([top, -top - 1, 0, 5] * 20), np.array([-top - 1, top, 3, 0, top] * 14))
    run(hip, 1, 80, 70, 2, 2, 32, seed=1, buckets=np.arange(9), zero=4, where=where)
    run(hip, 1, 80, 70, 2, 2, 32, seed=2, buckets=np.arange(9), zero=4, where=(np.full(80, 7), np.full(70, 9)))
    run(hip, 1, 80, 70, 2, 2, 32, seed=3, buckets=np.arange(200), zero=-50, where=(np.arange(80) * 3, np.arange(70)))
    run(hip, 1, 80, 70, 2, 2, 32, seed=4, buckets=np.arange(9), zero=2 ** 30)
    run(hip, 1, 80, 70, 2, 2, 32, seed=5, buckets=np.arange(9), zero=-2 ** 30)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [2560, 2561])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_maps_around_the_sums_in_doubles(hip, D, offsets):
    """Sums by offset are doubles up to 2560 offsets, where they fill a CU's LDS beside the tiles of 128, and floats beyond;
    sequences of up to 64 tokens have half the waves."""
    for S in (60, 200):
        at = np.arange(S) * 9
        run(hip, 2, S, S, 2, 2, D, seed=7, bf16=S == 60, buckets=np.arange(offsets) // 3, zero=offsets // 2, where=(at, at))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_map(hip, D):
    """4096 offsets, the last ones used, in 16384 buckets; key heads shared by two."""
    at = np.arange(60) * 70
    c, (_, _, got, _) = run(hip, 1, 60, 60, 2, 1, D, seed=6, buckets=(np.arange(4096) * 5) % 16384, zero=2000, n_buckets=16384,
                            where=(at, at))
    assert (got != 0).any(1).sum() == 60   # differences 70 i: i = -28 .. 29 in the map's reach, and its two ends


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the float64 loss sum(out * grad) along random directions of Q, K, V and the table; delta takes
    the rounded out, which adds sum_d |dO| uh |O| times P to each dS."""
    for bf16 in (False, True):
        c, (got, bound, gt, lt) = run(hip, 1, 40, 60, 4, 2, 32, bf16=bf16, causal=True, klens=[55], seed=21, **line(12, 7))
        B, Sq, Sk, H, Hkv, D = c.dims
        uh = 2.0 ** -8 if bf16 else 2.0 ** -11
        which, see = c.bucket_of(0), c.seen(0)

        def loss(parts):
            total = 0.0
            for h in range(H):
                q, k, v = parts[0][0, :, h], parts[1][0, :, h * Hkv // H], parts[2][0, :, h * Hkv // H]
                S = np.where(see, c.scale * q @ k.T + parts[3][which, h], -np.inf)
                P = np.exp(S - S.max(1, keepdims=True))
                total += ((P / P.sum(1, keepdims=True)) @ v * c.grad[0, :, h]).sum()
            return total

        at = [c.part(c.store, i).astype(np.float64) for i in range(3)] + [c.table.astype(np.float64)]
        more = sum((uh * np.abs(c.grad[0, :, h] * value(c.dout.numpy(), bf16)[0, :, h]).sum(1)).sum() for h in range(H))
        for i in range(4):
            d = O.randn(at[i].shape, 50 + i, 1.0).astype(np.float64)
            eps = 1e-4
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + eps * d, at[i] - eps * d
            slope = (loss(up) - loss(down)) / (2 * eps)
            # the difference itself: eps^2 / 6 of a third derivative below 1e3 here, and 1e-16 / eps of rounding
            if i < 3:
                lim = (bound[i] * 1.01 + uh * np.abs(got[i]) * 1.02 + 2.0 ** -25) * np.abs(d)
                factor = abs(c.scale) * max(np.abs(at[0]).max(), np.abs(at[1]).max()) * np.abs(d).max() * D if i < 2 else 0.0
                assert abs((got[i] * d).sum() - slope) <= lim.sum() + more * factor + 1e-5
            else:
                assert abs((gt * d).sum() - slope) <= (lt * np.abs(d)).sum() + more * np.abs(d).max() + 1e-5


@pytest.mark.gpu
def test_without_a_bias_it_is_plain_attention(hip):
    """A table of zeros: within the bounds of both, the plain operator's results."""
    c, p = Bias(hip, 2, 200, 200, 4, 2, 64, seed=4, table_std=0.0, **line(20, 5)), Case(hip, 2, 200, 200, 4, 2, 64, seed=4)
    for x in (c, p):
        x.forward()
        x.backward()
        x.check()


@pytest.mark.gpu
def test_repeats_agree_and_graphs_replay(hip, streams):
    """Calls agree bit for bit, the table's gradient too; graphs captured on two streams replay beside eager work."""
    cases = [Bias(hip, 4, 150, 150, 4, 2, 64, causal=True, seed=2, **line(50, 9)),
             Bias(hip, 300, 50, 50, 2, 2, 32, bf16=True, packed=True, seed=3, **grid(7, True))]
    want = []
    for c in cases:
        c.forward()
        c.backward()
        want.append(c.results())
        for _ in range(3):
            c.forward()
            c.backward()
            assert all(np.array_equal(a, b, equal_nan=a.dtype == np.float32) for a, b in zip(want[-1], c.results()))
    graphs = []
    for c in cases:
        s = streams.create()
        hip.set_stream(s)
        c.forward()
        c.backward()
        streams.sync(s)
        graphs.append((s, hip.Graph(lambda c=c: (c.forward(), c.backward()))))
    hip.set_stream(None)
    other = Bias(hip, 1, 100, 100, 2, 1, 64, seed=13, **line(10, 5))
    try:
        for _ in range(3):
            for c in cases:
                for g in c.dgrads:
                    g.upload(np.full(g.shape, 0x1234, np.uint16))
                c.dgtable.upload(np.full(c.dgtable.shape, np.nan, np.float32))
            hip.synchronize()
            for _, g in graphs:
                g.launch()
            other.forward()
            other.backward()
            for s, _ in graphs:
                streams.sync(s)
            hip.synchronize()
            for c, w in zip(cases, want):
                assert all(np.array_equal(a, b, equal_nan=a.dtype == np.float32) for a, b in zip(w, c.results()))
        other.check()
    finally:
        for _, g in graphs:
            g.destroy()


@pytest.mark.gpu
def test_empty_sequences(hip):
    """No keys, no queries, no images: zeros where there is something to write, and a table gradient of zeros."""
    H = hip.HIPBackend
    q, out, lse, dq = (empty_dev(hip, (2 * 5 * 64,), t) for t in (np.uint16, np.uint16, np.float32, np.uint16))
    for b, fill in ((q, 0x3c00), (out, 0x1234), (dq, 0x1234)):
        b.upload(np.full(640, fill, np.uint16))
    table, buckets = to_dev(hip, np.ones((3, 1), np.float32)), to_dev(hip, np.arange(3, dtype=np.int32))
    bias = [table, buckets, None, None, 3, 3, 1]
    fresh = lambda: to_dev(hip, np.full((3, 1), np.nan, np.float32))  # noqa: E731
    gt = fresh()
    H.attentionBiasForwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, *bias, out, lse, 2, 5, 0, 1, 1, 64, 1.0)
    assert np.all(out.numpy() == 0) and np.all(np.isneginf(lse.numpy()[:10]))
    H.attentionBiasBackwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, *bias, out, lse, q, dq, None, None, gt, 2, 5, 0, 1, 1,
                                64, 1.0)
    assert np.all(dq.numpy() == 0) and np.all(gt.numpy() == 0)
    dk, dv = (to_dev(hip, np.full(640, 0x1234, np.uint16)) for _ in range(2))
    gt = fresh()
    H.attentionBiasForwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, *bias, None, None, 2, 0, 5, 1, 1, 64, 1.0)
    H.attentionBiasBackwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, *bias, None, None, None, None, dk, dv, gt, 2, 0, 5, 1, 1,
                                64, 1.0)
    assert np.all(dk.numpy() == 0) and np.all(dv.numpy() == 0) and np.all(gt.numpy() == 0)
    gt = fresh()
    H.attentionBiasBackwardHalf(*[None] * 3, 64, 0, 64, 0, None, None, False, *bias, *[None] * 6, gt, 0, 5, 5, 1, 1, 64, 1.0)
    assert np.all(gt.numpy() == 0)


# ---------------------------------------------------------------- refusals: checked before anything touches a device
GOOD = dict(dtype=0, ldq=128, sq=1280, ldkv=64, skv=640, batch=1, seq_q=10, seq_k=10, heads=2, kv=1, dim=64, scale=0.125,
            ptr=4096, q=4096, lens=None, table=4096, buckets=4096, qpos=None, kpos=None, n=5, offsets=9, zero=4)
BAD = [dict(table=None), dict(buckets=None), dict(table=4098), dict(buckets=4097), dict(qpos=4096), dict(kpos=4096),
       dict(qpos=4098, kpos=4096), dict(qpos=4096, kpos=4098), dict(n=0), dict(n=-1), dict(n=16385), dict(offsets=0),
       dict(offsets=4097), dict(zero=-2 ** 30 - 1), dict(zero=-2 ** 31), dict(zero=2 ** 30 + 1), dict(zero=2 ** 31 - 1), dict(seq_q=2 ** 29 + 1), dict(seq_k=2 ** 29 + 1), dict(dtype=2), dict(batch=-1), dict(heads=3, kv=2),
       dict(dim=12), dict(dim=136), dict(scale=float("inf")), dict(ldq=120), dict(ldkv=56), dict(sq=1284), dict(q=None),
       dict(q=4098), dict(ptr=None), dict(ptr=4104), dict(lens=4098), dict(heads=65536, kv=1, ldq=65536 * 64)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **bad}
    p = a["ptr"]
    front = [a["dtype"], a["q"], p, p, a["ldq"], a["sq"], a["ldkv"], a["skv"], a["lens"], a["lens"], 0, a["table"], a["buckets"],
             a["qpos"], a["kpos"], a["n"], a["offsets"], a["zero"]]
    back = [a["batch"], a["seq_q"], a["seq_k"], a["heads"], a["kv"], a["dim"], a["scale"]]
    for name, middle in (("omHipAttentionBiasForwardHalf", [p, p]), ("omHipAttentionBiasBackwardHalf", [p] * 7)):
        with pytest.raises(om.OmHipError, match=name):
            om.call(name, *front, *middle, *back)


@pytest.mark.parametrize("grad", [None, 4098])
def test_a_table_gradient_is_asked_for(grad):
    import omnimatchdeeplearningtool_amd as om
    with pytest.raises(om.OmHipError, match="null|aligned"):
        om.call("omHipAttentionBiasBackwardHalf", 0, *[4096] * 3, 128, 1280, 64, 640, None, None, 0, 4096, 4096, None, None, 5, 9, 4,
                *[4096] * 6, grad, 1, 10, 10, 2, 1, 64, 0.125)
