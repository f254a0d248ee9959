"""Attention for training (forward with log-sum-exp, backward) against the formulas in float64, element by element.

Bounds, with u = 2^-24 (fp32) and uh = 2^-11 / 2^-8 (half a step of binary16 / bfloat16):
* a score carries (D + 3) u sum_d |scale q k|, and exp's argument two more roundings of its size, so a probability
  is off by a factor 1 +- ep, ep = 2 (D + 3) u max sum |scale q k| + 4 u (|S| + |lse|) + 8 u;
* forward: P and the result are rounded to the type: 2 uh + ep + (Sk + 4) u, in units of sum_j P |V|; binary16 weights
  below 2^-20 of the largest are subnormal, 2^-31 of it each;
* backward, from the saved out and lse: dV as the forward, in units of sum_i P |dO|. dS is off by
  P (ep (|dP| + |delta|) + (D + 2) u (sum |dO V| + sum |dO O|)) + 2 u |dS| and by uh |dS| of its rounding
  (binary16: 2^-33 of its column's largest at least); dQ and dK sum that with |K|, |Q|, add (n + 2) u, and round;
* a binary16 result below 2^-14 is off by 2^-25.
"""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)

U = 2.0 ** -24


def bits(x, bf16):
    return O.bf16_bits(x) if bf16 else x.astype(np.float16).view(np.uint16)


def value(b, bf16):
    return (b.astype(np.uint32) << 16).view(np.float32) if bf16 else b.view(np.float16).astype(np.float32)


class Case:
    """One call's sizes, inputs on the host (rounded to the type) and on the device, and its results."""

    def __init__(self, hip, B, Sq, Sk, H, Hkv, D, bf16=False, causal=False, qlens=None, klens=None, packed=False, scale=None,
                 seed=1, pad=0, std=1.0, grad=0.1):
        print(f"case {B}x{Sq}x{Sk} heads {H}/{Hkv}x{D} bf16={bf16} causal={causal} q={qlens} k={klens}", flush=True)
        self.hip, self.bf16, self.causal, self.seed = hip, bf16, causal, seed
        self.dims = (B, Sq, Sk, H, Hkv, D)
        self.scale = float(np.float32(D ** -0.5 if scale is None else scale))
        rnd = lambda shape, k, s: value(bits(O.randn(shape, seed + k, s), bf16), bf16)  # noqa: E731
        wq, wk = H * D, Hkv * D
        # storage: one packed tensor, or three, rows `pad` elements longer than they need be
        self.widths = [wq + 2 * wk + pad] if packed else [wq + pad, wk + pad, wk + pad]
        seqs = [Sq] if packed else [Sq, Sk, Sk]
        self.store = [rnd((B, s, w), i, std) for i, (s, w) in enumerate(zip(seqs, self.widths))]
        self.packed = packed
        self.first = [0, wq, wq + wk] if packed else [0, 0, 0]
        self.grad = rnd((B, Sq, H, D), 7, grad)
        self.qlens = None if qlens is None else np.asarray(qlens, np.int32)
        self.klens = None if klens is None else np.asarray(klens, np.int32)
        self.dev = [to_dev(hip, bits(t, bf16)) for t in self.store]
        self.dgrad = to_dev(hip, bits(self.grad, bf16))
        self.dlens = [None if x is None else to_dev(hip, x) for x in (self.qlens, self.klens)]
        self.dout, self.dlse = empty_dev(hip, (B, Sq, H, D), np.uint16), empty_dev(hip, (B, H, Sq))
        # gradients start as a value that must not survive inside the heads' columns and must outside of them
        self.dgrads = [to_dev(hip, np.full(t.shape, 0x1234, np.uint16)) for t in self.store]

    def part(self, arrays, i):
        B, Sq, Sk, H, Hkv, D = self.dims
        n = (H, Hkv, Hkv)[i]
        t = arrays[0 if self.packed else i]
        return t[:, :, self.first[i]:self.first[i] + n * D].reshape(t.shape[0], t.shape[1], n, D)

    def ptrs(self, bufs):
        return [bufs[0 if self.packed else i].ptr + 2 * self.first[i] for i in range(3)]

    def args(self):
        _, Sq, Sk, *_ = self.dims
        wq, wk = (self.widths[0],) * 2 if self.packed else self.widths[:2]
        return [*self.ptrs(self.dev), wq, wq * Sq, wk, wk * Sk, *self.dlens, self.causal]

    def forward(self):
        self.hip.HIPBackend.attentionTrainForwardHalf(*self.args(), self.dout, self.dlse, *self.dims, self.scale, bf16=self.bf16)

    def backward(self):
        self.hip.HIPBackend.attentionBackwardHalf(*self.args(), self.dout, self.dlse, self.dgrad, *self.ptrs(self.dgrads),
                                                  *self.dims, self.scale, bf16=self.bf16)

    def results(self):
        return [self.dout.numpy(), self.dlse.numpy()] + [g.numpy() for g in self.dgrads]

    def seen(self, b):
        B, Sq, Sk, *_ = self.dims
        nq = Sq if self.qlens is None else int(np.clip(self.qlens[b], 0, Sq))
        nk = Sk if self.klens is None else int(np.clip(self.klens[b], 0, Sk))
        i, j = np.arange(Sq)[:, None], np.arange(Sk)[None]
        return (i < nq) & (j < nk) & ((j <= i + Sk - Sq) if self.causal else True)

    def head(self, b, h):
        """Q, K, V of a query head in float64, zeros past the lengths, and what it sees."""
        B, Sq, Sk, H, Hkv, D = self.dims
        see = self.seen(b)
        q, k, v = (self.part(self.store, i)[b, :, x].astype(np.float64) for i, x in ((0, h), (1, h * Hkv // H), (2, h * Hkv // H)))
        return np.where(see.any(1)[:, None], q, 0), np.where(see.any(0)[:, None], k, 0), np.where(see.any(0)[:, None], v, 0), see

    def check(self):
        B, Sq, Sk, H, Hkv, D = self.dims
        uh, tiny = (2.0 ** -8, 0.0) if self.bf16 else (2.0 ** -11, 2.0 ** -25)
        out, lse = value(self.dout.numpy(), self.bf16), self.dlse.numpy()
        raw = [g.numpy() for g in self.dgrads]
        got = [value(np.ascontiguousarray(self.part(raw, i)), self.bf16) for i in range(3)]
        want = [np.zeros(g.shape) for g in got]
        bound = [np.zeros(g.shape) for g in got]
        for b in range(B):
            for h in range(H):
                q, k, v, see = self.head(b, h)
                some = see.any(1)
                kv = h * Hkv // H
                S = np.where(see, self.scale * q @ k.T, -np.inf)
                top = np.where(some, S.max(1, initial=-np.inf), 0.0)
                e = np.exp(S - top[:, None])
                L = np.where(some, np.log(np.maximum(e.sum(1), 1e-300)) + top, -np.inf)
                assert np.array_equal(np.isneginf(lse[b, h]), ~some)
                big = abs(self.scale) * (np.abs(q) @ np.abs(k).T).max(initial=0.0)
                size = np.abs(S[see]).max(initial=0.0) + np.abs(L[some]).max(initial=0.0)
                ep = 2 * (D + 3) * U * big + 4 * U * size + 8 * U
                assert np.all(np.abs(lse[b, h][some] - L[some]) <= ep + 4 * U * np.abs(L[some]) + (Sk + 4) * U)
                P = np.where(see, np.exp(S - np.where(some, L, 0.0)[:, None]), 0.0)
                ref = P @ v
                lim = (2 * uh + ep + (Sk + 4) * U) * 1.01 * (P @ np.abs(v)) + tiny
                lim += (0 if self.bf16 else 2.0 ** -31 * Sk) * np.abs(v).max(initial=0.0) * P.max(1, initial=0.0)[:, None]
                off = np.abs(out[b, :, h] - ref)
                assert np.all(off <= lim), (b, h, float((off / lim).max()))
                assert np.all(out[b, ~some, h] == 0)
                # gradients, from the saved out and lse
                g, o = self.grad[b, :, h].astype(np.float64), out[b, :, h].astype(np.float64)
                g = np.where(some[:, None], g, 0.0)
                P = np.where(see, np.exp(S - np.where(some, lse[b, h].astype(np.float64), 0.0)[:, None]), 0.0)
                dP, delta = g @ v.T, (g * o).sum(1, keepdims=True)
                dS = P * (dP - delta)
                e = P * (ep * (np.abs(dP) + np.abs(delta)) + (D + 2) * U * (np.abs(g) @ np.abs(v).T + (np.abs(g) * np.abs(o)).sum(1, keepdims=True)))
                e += (uh + 2 * U) * np.abs(dS)
                least = 0.0 if self.bf16 else 2.0 ** -33
                c = abs(self.scale)
                want[0][b, :, h] = self.scale * dS @ k
                eq = e + least * np.abs(dS).max(1, initial=0.0)[:, None]
                bound[0][b, :, h] = c * (eq @ np.abs(k) + (Sk + 2) * U * np.abs(dS) @ np.abs(k))
                want[1][b, :, kv] += self.scale * dS.T @ q
                ek = e + least * np.abs(dS).max(0, initial=0.0)[None]
                bound[1][b, :, kv] += c * (ek.T @ np.abs(q) + (Sq + 2) * (H // Hkv) * U * np.abs(dS).T @ np.abs(q))
                want[2][b, :, kv] += P.T @ g
                bound[2][b, :, kv] += (uh + ep + (Sq + 4) * (H // Hkv) * U) * (P.T @ np.abs(g)) + least * np.abs(g).sum(0)
        for name, g, w, lim in zip("qkv", got, want, bound):
            off = np.abs(g - w)
            lim = 1.01 * lim + uh * np.abs(w) * 1.01 + tiny
            assert np.all(off <= lim), ("d" + name, float((off / np.maximum(lim, 1e-300)).max()))
        # nothing outside the heads' columns was touched
        for i, (t, w) in enumerate(zip(raw, self.widths)):
            used = sum(self.dims[k] * self.dims[5] for k in ((3, 4, 4) if self.packed else ((3,), (4,), (4,))[i]))
            assert np.all(t[:, :, used:] == 0x1234)
        return got, bound


def run(hip, *dims, **kw):
    c = Case(hip, *dims, **kw)
    c.forward()
    c.backward()
    return c, c.check()


# one token to several tiles, around the 32, 64 and 128 rows of a wave, a tile and a workgroup
LENGTHS = [(1, 1), (1, 8), (1, 200), (31, 33), (32, 32), (33, 31), (63, 65), (64, 64), (65, 129), (127, 128), (129, 127),
           (200, 1), (257, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Sq,Sk", LENGTHS, ids=str)
def test_lengths(hip, Sq, Sk, bf16):
    run(hip, 1, Sq, Sk, 2, 2, 64, bf16=bf16, seed=10 * Sq + Sk)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 70), (40, 40), (64, 64), (130, 130), (200, 90), (90, 200), (300, 300)], ids=str)
def test_causal(hip, Sq, Sk):
    """Sq > Sk leaves the first rows without a key."""
    run(hip, 2, Sq, Sk, 2, 1, 64, bf16=Sq % 4 == 0, causal=True, seed=Sq + Sk)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 120, 128])
def test_head_dimensions(hip, D, bf16):
    run(hip, 2, 70, 150, 2, 2, D, bf16=bf16, causal=D % 16 == 0, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (6, 1), (9, 3), (16, 8)], ids=str)
def test_shared_heads_packed_and_padded_rows(hip, H, Hkv):
    run(hip, 3, 77, 77, H, Hkv, 40, packed=True, pad=16, causal=True, seed=H)
    run(hip, 2, 50, 141, H, Hkv, 128, bf16=True, pad=8, seed=H + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk,H,Hkv,D", [(1, 4000, 2, 1, 64), (5, 1500, 4, 4, 128), (1500, 5, 3, 1, 64), (700, 700, 4, 1, 96),
                                           (300, 1030, 2, 2, 40)], ids=str)
def test_walks_shared_by_workgroups(hip, Sq, Sk, H, Hkv, D, causal):
    """Few blocks and long walks: parts of a walk without a visible key, and images of other lengths, among them."""
    run(hip, 3, Sq, Sk, H, Hkv, D, bf16=D > 64, causal=causal, klens=[Sk, 0, Sk // 3], qlens=[Sq, Sq, (Sq + 1) // 2],
        seed=Sq + D)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_lengths_per_image(hip, causal, bf16):
    """Images without queries or keys, with one, with all, and lengths outside their range."""
    run(hip, 7, 150, 150, 2, 1, 64, bf16=bf16, causal=causal, qlens=[0, 1, 150, 64, 33, -5, 400],
        klens=[150, 1, 0, 65, 150, 20, 400], packed=True, seed=3)


@pytest.mark.gpu
def test_what_lies_past_a_length_is_not_read(hip):
    for bf16 in (False, True):
        c = Case(hip, 2, 100, 140, 2, 2, 64, bf16=bf16, qlens=[37, 100], klens=[70, 129], seed=5)
        nan = 0x7fff
        for i, lens in ((0, c.qlens), (1, c.klens), (2, c.klens)):
            t = bits(c.store[i], bf16)
            for b in range(2):
                t[b, lens[b]:] = nan
            c.dev[i].upload(t)
        g = bits(c.grad, bf16)
        g[0, 37:] = nan
        c.dgrad.upload(g)
        c.forward()
        c.backward()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(hip, scale):
    """Negative, zero and large: scores to several hundred, rows that one key takes."""
    run(hip, 1, 70, 200, 2, 2, 64, scale=scale, seed=9)
    run(hip, 1, 70, 200, 2, 2, 64, scale=scale, bf16=True, seed=9)


@pytest.mark.gpu
def test_maxima_that_grow_and_fall(hip):
    for order in (1, -1):
        c = Case(hip, 1, 64, 640, 1, 1, 32, seed=4, scale=1.0)
        ramp = np.linspace(0.05, 3.0, 640)[::order]
        c.store[1] = value(bits((c.store[1] * ramp[None, :, None]).astype(np.float32), False), False)
        c.dev[1].upload(bits(c.store[1], False))
        c.forward()
        c.backward()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [1e-6, 3e-4, 300.0])
def test_small_and_large_gradients(hip, grad):
    """binary16: gradients whose dS lies below 2^-14 or, with V of several hundred, above 65504."""
    c = Case(hip, 1, 90, 2000, 1, 1, 64, seed=8, grad=grad)
    if grad > 1:
        c.store[2] = value(bits(c.store[2] * 200, False), False)
        c.dev[2].upload(bits(c.store[2], False))
        c.store[1] = value(bits(c.store[1] * 1e-3, False), False)   # even probabilities, small enough a dQ
        c.dev[1].upload(bits(c.store[1], False))
        c.store[0] = value(bits(c.store[0] * 1e-2, False), False)
        c.dev[0].upload(bits(c.store[0], False))
    c.forward()
    c.backward()
    c.check()


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the float64 loss sum(out * grad) along random directions of Q, K and V. On top of the
    gradient's own bound, delta takes the rounded out: sum_d |dO| uh |O| times P."""
    for bf16 in (False, True):
        c, (got, bound) = run(hip, 1, 40, 60, 4, 2, 32, bf16=bf16, causal=True, klens=[55], seed=21)
        B, Sq, Sk, H, Hkv, D = c.dims
        uh = 2.0 ** -8 if bf16 else 2.0 ** -11

        def loss(parts):
            total = 0.0
            for h in range(H):
                q, k, v = parts[0][0, :, h], parts[1][0, :, h * Hkv // H], parts[2][0, :, h * Hkv // H]
                see = c.seen(0)
                S = np.where(see, c.scale * q @ k.T, -np.inf)
                P = np.exp(S - S.max(1, keepdims=True))
                total += ((P / P.sum(1, keepdims=True)) @ v * c.grad[0, :, h]).sum()
            return total

        at = [c.part(c.store, i).astype(np.float64) for i in range(3)]
        more = 0.0   # |dS| that the rounding of out may add, summed with the largest factors
        for h in range(H):
            out = value(c.dout.numpy(), bf16)[0, :, h]
            more += (uh * np.abs(c.grad[0, :, h] * out).sum(1)).sum()
        for i in range(3):
            d = O.randn(at[i].shape, 50 + i, 1.0).astype(np.float64)
            eps = 1e-4
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + eps * d, at[i] - eps * d
            slope = (loss(up) - loss(down)) / (2 * eps)
            lim = (bound[i] * 1.01 + uh * np.abs(got[i]) * 1.02 + 2.0 ** -25) * np.abs(d)
            factor = abs(c.scale) * max(np.abs(at[0]).max(), np.abs(at[1]).max()) * np.abs(d).max() * D if i < 2 else 0.0
            # the difference itself: eps^2 / 6 of a third derivative below 1e3 here, and 1e-16 / eps of rounding
            assert abs((got[i] * d).sum() - slope) <= lim.sum() + more * factor + 1e-5


@pytest.mark.gpu
def test_one_row_past_32_bits_of_offset(hip):
    """An image stride of 2^31 + 64 elements: the second image lies past 32 bits of element and byte offset."""
    far, D, S = 2 ** 31 + 64, 64, 40
    c = Case(hip, 2, S, S, 1, 1, D, bf16=True, seed=6)
    big = empty_dev(hip, (far + S * D,), np.uint16)
    grads = empty_dev(hip, (far + S * D,), np.uint16)
    for b in range(2):
        hip.call("omHipCopyD2D", big.ptr + 2 * b * far, c.dev[0].ptr + 2 * b * S * D, 2 * S * D)
    plain = Case(hip, 2, S, S, 1, 1, D, bf16=True, seed=6)
    plain.forward()
    plain.backward()
    args = [big.ptr, plain.dev[1].ptr, plain.dev[2].ptr, D, far, D, S * D, None, None, False]
    hip.HIPBackend.attentionTrainForwardHalf(*args, c.dout, c.dlse, *c.dims, c.scale, bf16=True)
    hip.HIPBackend.attentionBackwardHalf(*args, c.dout, c.dlse, c.dgrad, grads.ptr, *c.ptrs(c.dgrads)[1:], *c.dims, c.scale,
                                         bf16=True)
    assert np.array_equal(c.dout.numpy(), plain.dout.numpy())
    for b in range(2):
        part = empty_dev(hip, (S * D,), np.uint16)
        hip.call("omHipCopyD2D", part.ptr, grads.ptr + 2 * b * far, 2 * S * D)
        assert np.array_equal(part.numpy(), plain.dgrads[0].numpy()[b].reshape(-1))


@pytest.mark.gpu
def test_repeats_agree_and_graphs_replay(hip, streams):
    """Calls agree bit for bit; two graphs captured on two streams replay beside eager work of the same operators."""
    cases = [Case(hip, 2, 150, 150, 4, 2, 64, causal=True, seed=2), Case(hip, 1, 300, 200, 2, 2, 128, bf16=True, seed=3)]
    want = []
    for c in cases:
        c.forward()
        c.backward()
        want.append(c.results())
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
    other = Case(hip, 1, 100, 100, 2, 1, 64, seed=13)
    try:
        for _ in range(3):
            for c in cases:
                for g in c.dgrads:
                    g.upload(np.full(g.shape, 0x1234, np.uint16))
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
    """No keys: zeros and -inf. No queries: zero dK, dV. No images: nothing."""
    H = hip.HIPBackend
    q, out, lse, dq = (empty_dev(hip, (2 * 5 * 64,), t) for t in (np.uint16, np.uint16, np.float32, np.uint16))
    for b, fill in ((q, 0x3c00), (out, 0x1234), (dq, 0x1234)):
        b.upload(np.full(640, fill, np.uint16))
    H.attentionTrainForwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, out, lse, 2, 5, 0, 1, 1, 64, 1.0)
    assert np.all(out.numpy() == 0) and np.all(np.isneginf(lse.numpy()[:10]))
    H.attentionBackwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, out, lse, q, dq, None, None, 2, 5, 0, 1, 1, 64, 1.0)
    assert np.all(dq.numpy() == 0)
    dk, dv = (to_dev(hip, np.full(640, 0x1234, np.uint16)) for _ in range(2))
    H.attentionTrainForwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, None, None, 2, 0, 5, 1, 1, 64, 1.0)
    H.attentionBackwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, None, None, None, None, dk, dv, 2, 0, 5, 1, 1, 64, 1.0)
    assert np.all(dk.numpy() == 0) and np.all(dv.numpy() == 0)
    H.attentionBackwardHalf(*[None] * 3, 64, 0, 64, 0, None, None, False, *[None] * 6, 0, 5, 5, 1, 1, 64, 1.0)


@pytest.mark.gpu
def test_tokens_of_all_images_in_turn(hip):
    """Rows in the order token, image: the image stride is the heads' width, the row stride all images'."""
    B, S, H, D = 3, 70, 2, 64
    w = H * D
    c = Case(hip, B, S, S, H, H, D, seed=17)
    c.forward()
    c.backward()
    turned = [to_dev(hip, np.ascontiguousarray(bits(t, False).transpose(1, 0, 2))) for t in c.store]
    out, lse = empty_dev(hip, (B, S, H, D), np.uint16), empty_dev(hip, (B, H, S))
    grads = [empty_dev(hip, (S, B, w), np.uint16) for _ in range(3)]
    args = [*[t.ptr for t in turned], B * w, w, B * w, w, None, None, False]
    hip.HIPBackend.attentionTrainForwardHalf(*args, out, lse, *c.dims, c.scale)
    hip.HIPBackend.attentionBackwardHalf(*args, out, lse, c.dgrad, *grads, *c.dims, c.scale)
    want = c.results()
    assert np.array_equal(out.numpy(), want[0]) and np.array_equal(lse.numpy(), want[1])
    for g, x in zip(grads, want[2:]):
        assert np.array_equal(g.numpy().transpose(1, 0, 2), x)


@pytest.mark.gpu
def test_keys_shared_by_images(hip):
    """An image stride of 0: the forward pass reads one set of keys for every image."""
    c = Case(hip, 3, 20, 90, 2, 2, 64, seed=18)
    for i in (1, 2):
        c.store[i][1:] = c.store[i][:1]
        c.dev[i].upload(bits(c.store[i], False))
    c.forward()
    out, lse = empty_dev(hip, (3, 20, 2, 64), np.uint16), empty_dev(hip, (3, 2, 20))
    args = c.args()
    args[6] = 0
    hip.HIPBackend.attentionTrainForwardHalf(*args, out, lse, *c.dims, c.scale)
    assert np.array_equal(out.numpy(), c.dout.numpy()) and np.array_equal(lse.numpy(), c.dlse.numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("Sk", [100, 2000])
def test_nan_reaches_its_rows(hip, Sk):
    """A NaN query makes its own row NaN, context and log-sum-exp, and no other head's; one workgroup a row's keys or
    several."""
    c = Case(hip, 1, 40, Sk, 2, 2, 64, seed=19)
    c.store[0][0, 7, :64] = np.nan
    c.dev[0].upload(bits(c.store[0], False))
    c.forward()
    out, lse = value(c.dout.numpy(), False), c.dlse.numpy()
    assert np.isnan(out[0, 7, 0]).all() and np.isnan(lse[0, 0, 7])
    assert np.isnan(lse).sum() == 1 and np.isnan(out).sum() == 64


# ---------------------------------------------------------------- refusals: checked before anything touches a device
GOOD = dict(dtype=0, ldq=128, sq=1280, ldkv=64, skv=640, batch=1, seq_q=10, seq_k=10, heads=2, kv=1, dim=64, scale=0.125,
            ptr=4096, q=4096)
BAD = [dict(dtype=2), dict(dtype=-1), dict(batch=-1), dict(seq_q=-1), dict(seq_k=-3), dict(heads=0), dict(kv=0), dict(heads=3, kv=2),
       dict(dim=4), dict(dim=12), dict(dim=136), dict(dim=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(ldq=120),
       dict(ldkv=56), dict(ldq=129), dict(sq=1284), dict(ldkv=2 ** 23), dict(sq=-8), dict(skv=-8), dict(q=None), dict(q=4098),
       dict(ptr=None), dict(ptr=4104), dict(seq_q=2 ** 30 + 1), dict(batch=2 ** 20, seq_q=2 ** 20)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **bad}
    p = a["ptr"]
    front = [a["dtype"], a["q"], p, p, a["ldq"], a["sq"], a["ldkv"], a["skv"], None, None, 0]
    back = [a["batch"], a["seq_q"], a["seq_k"], a["heads"], a["kv"], a["dim"], a["scale"]]
    for name, middle in (("omHipAttentionTrainForwardHalf", [p, p]), ("omHipAttentionBackwardHalf", [p] * 6)):
        with pytest.raises(om.OmHipError, match=name):
            om.call(name, *front, *middle, *back)


@pytest.mark.parametrize("sq,skv", [(0, 640), (1280, 0), (1272, 640), (1280, 56)], ids=str)
def test_overlapping_gradients_are_refused(sq, skv):
    """Two images of 10 tokens, 2 heads of 64 on one: rows of 128 and 64 elements."""
    import omnimatchdeeplearningtool_amd as om
    args = [0, 4096, 4096, 4096, 128, sq, 64, skv, None, None, 0, *[4096] * 6, 2, 10, 10, 2, 1, 64, 0.125]
    with pytest.raises(om.OmHipError, match="overlap"):
        om.call("omHipAttentionBackwardHalf", *args)


@pytest.mark.parametrize("place", [8, 9])
def test_misaligned_lengths_are_refused(place):
    import omnimatchdeeplearningtool_amd as om
    args = [0, 4096, 4096, 4096, 128, 1280, 64, 640, None, None, 0]
    args[place] = 4098
    for name, n in (("omHipAttentionTrainForwardHalf", 2), ("omHipAttentionBackwardHalf", 6)):
        with pytest.raises(om.OmHipError, match="aligned"):
            om.call(name, *args, *[4096] * n, 1, 10, 10, 2, 1, 64, 0.125)


# One launch takes 2^32 - 1 threads: 256 for each block of 128 queries of a head, 512 for each block of 128 keys of a key
# head in the backward pass. The query pointer is null, so a size that is let through is refused for that.
def sizes(batch, seq_q, seq_k, heads, kv):
    return dict(batch=batch, seq_q=seq_q, seq_k=seq_k, heads=heads, kv=kv, ldq=64 * heads, ldkv=64 * kv, q=None)


def refuse_both(a, forward, backward):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **a}
    p = a["ptr"]
    front = [a["dtype"], a["q"], p, p, a["ldq"], a["sq"], a["ldkv"], a["skv"], None, None, 0]
    back = [a["batch"], a["seq_q"], a["seq_k"], a["heads"], a["kv"], a["dim"], a["scale"]]
    for name, middle, why in (("omHipAttentionTrainForwardHalf", [p, p], forward), ("omHipAttentionBackwardHalf", [p] * 6, backward)):
        with pytest.raises(om.OmHipError, match=f"{name}.*{why}"):
            om.call(name, *front, *middle, *back)


@pytest.mark.parametrize("a,forward,backward", [
    (sizes(2 ** 20, 128, 100, 16, 1), "too many", "too many"),           # 2^24 blocks of queries
    (sizes(2 ** 19, 129, 100, 16, 1), "too many", "too many"),
    (sizes(2 ** 20 - 1, 128, 100, 16, 1), "null", "null"),
    (sizes(2 ** 19, 50, 50, 16, 16), "null", "too many"),                # 2^23 blocks of keys
    (sizes(2 ** 18, 50, 129, 16, 16), "null", "too many"),
    (sizes(2 ** 19 - 1, 50, 50, 16, 16), "null", "null"),
    (sizes(2 ** 30, 2 ** 30, 8, 2 ** 16, 1), "too many", "too many"),    # 2^70 triples: not a 64-bit number
    (sizes(2 ** 30, 8, 2 ** 30, 2 ** 16, 1), "too many", "too many"),
], ids=str)
def test_more_blocks_than_a_launch_takes(a, forward, backward):
    refuse_both(a, forward, backward)
