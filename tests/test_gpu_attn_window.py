"""Attention in a sliding window with first tokens that stay visible, forward and backward, against the formulas in float64,
element by element (attn_views says how far off a result may be)."""
import numpy as np
import pytest

import oracle as O
from attn_views import Viewed
from conftest import empty_dev, to_dev
from test_gpu_attn_train import Case, bits, value
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)


class Window(Viewed):
    def __init__(self, hip, *dims, window, first=0, **kw):
        print(f"window {window} first {first}", end=" ", flush=True)
        super().__init__(hip, *dims, **kw)
        self.window, self.first_keys = window, first

    def forward(self):
        self.hip.HIPBackend.attentionWindowForwardHalf(*self.args(), self.window, self.first_keys, self.dout, self.dlse,
                                                       *self.dims, self.scale, bf16=self.bf16)

    def backward(self):
        self.hip.HIPBackend.attentionWindowBackwardHalf(*self.args(), self.window, self.first_keys, self.dout, self.dlse,
                                                        self.dgrad, *self.ptrs(self.dgrads), *self.dims, self.scale,
                                                        bf16=self.bf16)

    def seen(self, b):
        see, p, j = self.standing(b)
        return see & ((np.abs(p - j) < self.window) | (j < self.first_keys))


def run(hip, *dims, **kw):
    c = Window(hip, *dims, **kw)
    c.forward()
    c.backward()
    return c, c.check()


# borders of windows and first keys around a wave's 32 rows, a tile's 64 and a block's 128; windows past the sequence
@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 3), (7, 1), (32, 0), (33, 64), (64, 4), (65, 65), (100, 130), (128, 1),
                                          (129, 0), (300, 4), (2 ** 31 - 1, 2 ** 31 - 1)], ids=str)
def test_windows(hip, window, first, causal):
    run(hip, 1, 290, 290, 2, 1, 64, window=window, first=first, causal=causal, bf16=window % 2 == 1, seed=window % 1000 + first)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 64), (1, 300), (2, 65), (31, 33), (64, 64), (65, 129), (129, 65), (200, 1), (300, 90),
                                   (90, 400)], ids=str)
def test_lengths(hip, Sq, Sk, causal):
    """Sq > Sk leaves the first rows before the first key: a causal mask hides all, a window all but its own reach."""
    run(hip, 2, Sq, Sk, 2, 2, 64, window=20, first=2, causal=causal, bf16=Sq % 2 == 0, seed=Sq + Sk)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 64, 72, 96, 104, 128])
def test_head_dimensions(hip, D, bf16):
    run(hip, 2, 170, 150, 2, 2, D, bf16=bf16, window=40, first=5, causal=D % 16 == 0, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(4, 2), (6, 1), (9, 3)], ids=str)
def test_shared_heads_packed_and_padded_rows(hip, H, Hkv):
    run(hip, 3, 177, 177, H, Hkv, 40, packed=True, pad=16, causal=True, window=50, first=3, seed=H)
    run(hip, 2, 150, 241, H, Hkv, 128, bf16=True, pad=8, window=70, first=1, seed=H + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_lengths_per_image(hip, causal, bf16):
    """Each image's last query stands at its last key; images without queries or keys, with one, with all, more queries
    than keys, and lengths outside their range."""
    run(hip, 8, 150, 250, 2, 1, 64, bf16=bf16, causal=causal, window=30, first=2, qlens=[0, 1, 150, 64, 33, -5, 400, 100],
        klens=[150, 1, 0, 165, 250, 20, 400, 20], seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("Sq,Sk,H,Hkv,D,window,first", [(1500, 1500, 2, 1, 64, 500, 4), (1500, 1500, 4, 1, 128, 100, 200),
                                                        (40, 2000, 2, 2, 96, 1500, 1), (1, 4000, 4, 1, 64, 2000, 70),
                                                        (2000, 40, 2, 1, 32, 600, 3)], ids=str)
def test_walks_shared_by_workgroups(hip, Sq, Sk, H, Hkv, D, window, first, causal):
    """Few blocks and long walks, and first keys that every query sees: parts of a walk without a visible key, images of
    other lengths."""
    run(hip, 2, Sq, Sk, H, Hkv, D, bf16=D > 64, causal=causal, window=window, first=first, klens=[Sk, Sk // 3],
        qlens=[Sq, (Sq + 1) // 2], seed=Sq + D)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("first", [1, 32, 33, 129, 256, 257, 300])
def test_first_keys_of_far_queries(hip, first, causal):
    """Queries far past their windows, by workgroups for 32 first keys up to 256 of them and by whole walks beyond; images
    without queries or keys, and with fewer keys than first ones."""
    run(hip, 4, 500, 500, 2, 1, 64, window=10, first=first, causal=causal, qlens=[500, 0, 500, 300], klens=[500, 500, 0, 20],
        bf16=first % 2 == 0, seed=first)


@pytest.mark.gpu
def test_what_lies_past_a_length_is_not_read(hip):
    for bf16 in (False, True):
        c = Window(hip, 2, 100, 140, 2, 2, 64, bf16=bf16, qlens=[37, 100], klens=[70, 129], window=30, first=2, seed=5)
        for i, lens in ((0, c.qlens), (1, c.klens), (2, c.klens)):
            t = bits(c.store[i], bf16)
            for b in range(2):
                t[b, lens[b]:] = 0x7fff
            c.dev[i].upload(t)
        g = bits(c.grad, bf16)
        g[0, 37:] = 0x7fff
        c.dgrad.upload(g)
        c.forward()
        c.backward()
        c.check()


@pytest.mark.gpu
def test_keys_out_of_sight_are_not_read(hip):
    """NaN in tiles of 64 keys that no query sees: between the first keys' tile and the window's."""
    for Sq in (1, 30, 150):
        c = Window(hip, 1, Sq, 1000, 4, 2, 64, window=40, first=3, causal=True, seed=Sq)
        for i in (1, 2):
            t = bits(c.store[i], False)
            t[:, 64:(1000 - Sq - 39) // 64 * 64] = 0x7fff
            c.dev[i].upload(t)
        c.forward()
        assert np.isfinite(value(c.dout.numpy(), False)).all() and np.isfinite(c.dlse.numpy()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(hip, scale):
    run(hip, 1, 170, 200, 2, 2, 64, scale=scale, window=60, first=1, seed=9)
    run(hip, 1, 1, 200, 2, 2, 64, scale=scale, bf16=True, window=60, first=1, seed=9)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
def test_a_window_over_everything_is_plain_attention(hip, causal):
    """Bit for bit where both walk alike (context, log-sum-exp, dQ); dK and dV may be shared by other numbers of workgroups."""
    for dims in ((2, 200, 200, 4, 2, 64), (1, 130, 130, 2, 2, 128)):
        c, p = Window(hip, *dims, window=10 ** 9, causal=causal, seed=4), Case(hip, *dims, causal=causal, seed=4)
        for x in (c, p):
            x.forward()
            x.backward()
        for a, b in zip(c.results()[:3], p.results()[:3]):
            assert np.array_equal(a, b)
        c.check()


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the float64 loss sum(out * grad) along random directions of Q, K and V; bounds as in
    test_gpu_attn_train."""
    for bf16 in (False, True):
        c, (got, bound) = run(hip, 1, 80, 90, 4, 2, 32, bf16=bf16, causal=True, klens=[85], window=20, first=2, seed=21)
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
        more = sum((uh * np.abs(c.grad[0, :, h] * value(c.dout.numpy(), bf16)[0, :, h]).sum(1)).sum() for h in range(H))
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
def test_one_token_past_32_bits_of_offset(hip):
    """A cache whose second image starts 2^31 + 64 elements after the first."""
    far, D, S = 2 ** 31 + 64, 64, 200
    c = Window(hip, 2, 1, S, 2, 1, D, bf16=True, window=50, first=4, causal=True, seed=6)
    c.forward()
    cache = [empty_dev(hip, (far + S * D,), np.uint16) for _ in range(2)]
    for k, big in enumerate(cache):
        for b in range(2):
            hip.call("omHipCopyD2D", big.ptr + 2 * b * far, c.dev[1 + k].ptr + 2 * b * S * D, 2 * S * D)
    out, lse = empty_dev(hip, (2, 1, 2, D), np.uint16), empty_dev(hip, (2, 2, 1))
    hip.HIPBackend.attentionWindowForwardHalf(c.dev[0], cache[0], cache[1], 2 * D, 2 * D, D, far, None, None, True, 50, 4, out, lse,
                                              *c.dims, c.scale, bf16=True)
    assert np.array_equal(out.numpy(), c.dout.numpy()) and np.array_equal(lse.numpy(), c.dlse.numpy())


@pytest.mark.gpu
def test_tokens_one_by_one_follow_the_whole_sequence(hip):
    """A cache that grows: step t's query against keys 0 .. t is row t of the sequence's causal attention, to the bounds of
    both (each within its own of the formula)."""
    S = 150
    whole = Window(hip, 1, S, S, 4, 2, 64, window=40, first=3, causal=True, seed=12)
    whole.forward()
    whole.backward()
    whole.check()
    for t in (0, 1, 39, 40, 41, 63, 64, 100, 149):
        step = Window(hip, 1, 1, S, 4, 2, 64, window=40, first=3, causal=True, klens=[t + 1], seed=12)
        step.store[0] = whole.store[0][:, t:t + 1]
        step.store[1:] = whole.store[1:]
        step.dev = [to_dev(hip, bits(x, False)) for x in step.store]
        step.forward()
        step.backward()
        step.check()


@pytest.mark.gpu
def test_repeats_agree_and_graphs_replay(hip, streams):
    """Calls agree bit for bit; graphs captured on two streams replay beside eager work of the same operators."""
    cases = [Window(hip, 2, 1150, 1150, 4, 2, 64, causal=True, window=100, first=4, seed=2),
             Window(hip, 1, 300, 200, 2, 2, 128, bf16=True, window=30, seed=3),
             Window(hip, 3, 1, 700, 8, 2, 128, bf16=True, causal=True, window=300, first=4, klens=[700, 30, 411], seed=4)]
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
    other = Window(hip, 1, 100, 100, 2, 1, 64, window=9, seed=13)
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
def test_more_first_keys_than_a_launch_takes(hip):
    """2^22 + 1 images of 97 first keys: a workgroup of 256 threads for each 32 of them would be more than 2^32 threads. Scores
    are 0, so every key has 1/97 of dO (1) for dV; dP is what delta is, and dK 0."""
    B, Sk, D = 2 ** 22 + 1, 97, 8
    H = hip.HIPBackend
    kv, dk, dv = (empty_dev(hip, (B * Sk * D // 2,)) for _ in range(3))    # two halves each
    q, out, grad, dq = (empty_dev(hip, (B * D // 2,)) for _ in range(4))
    lse = empty_dev(hip, (B,))
    pair = lambda x: float(np.full(2, x, np.float16).view(np.float32)[0])
    for b, n, x in ((kv, B * Sk * D // 2, pair(0.5)), (dk, B * Sk * D // 2, pair(3.)), (dv, B * Sk * D // 2, pair(3.)),
                    (q, B * D // 2, 0.), (out, B * D // 2, pair(0.5)), (grad, B * D // 2, pair(1.)), (lse, B, float(np.log(97.)))):
        H.fillValue(b, n, x)
    H.attentionWindowBackwardHalf(q, kv, kv, D, D, D, Sk * D, None, None, True, 1, Sk, out, lse, grad, dq, dk, dv, B, 1, Sk, 1, 1, D,
                                  1.0)
    for image in (0, 1, 2 ** 20, 2 ** 21 + 1, B - 1):
        got = np.empty((2, Sk, D), np.float16)
        for g, to in zip((dk, dv), got):
            hip.call("omHipCopyD2H", to.ctypes.data, g.ptr + image * Sk * D * 2, to.nbytes)
        assert np.all(got[0] == 0)
        # P and dV are rounded to halves; P's exponent, between 4 and 16 in fp32, is a few half steps of 2^-21 off
        assert np.all(np.abs(got[1].astype(np.float64) * 97 - 1) <= 2 * 2. ** -11 + 2. ** -19)


@pytest.mark.gpu
def test_empty_sequences(hip):
    """No keys: zeros and -inf. No queries: zero dK, dV. No images: nothing."""
    H = hip.HIPBackend
    q, out, lse, dq = (empty_dev(hip, (2 * 5 * 64,), t) for t in (np.uint16, np.uint16, np.float32, np.uint16))
    for b, fill in ((q, 0x3c00), (out, 0x1234), (dq, 0x1234)):
        b.upload(np.full(640, fill, np.uint16))
    w = (8, 2)
    for n in (5, 1):
        H.attentionWindowForwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, *w, out, lse, 2, n, 0, 1, 1, 64, 1.0)
        assert np.all(out.numpy()[:128 * n] == 0) and np.all(np.isneginf(lse.numpy()[:2 * n]))
    H.attentionWindowForwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, *w, out, lse, 2, 5, 0, 1, 1, 64, 1.0)
    H.attentionWindowBackwardHalf(q, None, None, 64, 320, 64, 0, None, None, False, *w, out, lse, q, dq, None, None, 2, 5, 0, 1, 1, 64,
                                  1.0)
    assert np.all(dq.numpy() == 0)
    dk, dv = (to_dev(hip, np.full(640, 0x1234, np.uint16)) for _ in range(2))
    H.attentionWindowForwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, *w, None, None, 2, 0, 5, 1, 1, 64, 1.0)
    H.attentionWindowBackwardHalf(None, q, q, 64, 0, 64, 320, None, None, False, *w, None, None, None, None, dk, dv, 2, 0, 5, 1, 1, 64,
                                  1.0)
    assert np.all(dk.numpy() == 0) and np.all(dv.numpy() == 0)
    for window, first in ((2, 1), (2, 3), (1, 0), (2, 400)):   # first keys whose queries would be out of their window
        for g in (dk, dv):
            g.upload(np.full(640, 0x1234, np.uint16))
        H.attentionWindowBackwardHalf(None, q, q, 64, 0, 64, 320, None, None, first == 1, window, first, None, None, None, None, dk, dv, 2,
                                      0, 5, 1, 1, 64, 1.0)
        assert np.all(dk.numpy() == 0) and np.all(dv.numpy() == 0)
    H.attentionWindowBackwardHalf(*[None] * 3, 64, 0, 64, 0, None, None, False, *w, *[None] * 6, 0, 5, 5, 1, 1, 64, 1.0)


# ---------------------------------------------------------------- refusals: checked before anything touches a device
GOOD = dict(dtype=0, ldq=128, sq=1280, ldkv=64, skv=640, batch=1, seq_q=10, seq_k=10, heads=2, kv=1, dim=64, scale=0.125,
            ptr=4096, q=4096, lens=None, window=5, first=1)
BAD = [dict(window=0), dict(window=-1), dict(first=-1), dict(dtype=2), dict(batch=-1), dict(seq_q=-1), dict(heads=3, kv=2),
       dict(dim=12), dict(dim=136), dict(scale=float("nan")), dict(ldq=120), dict(ldkv=56), dict(sq=1284), dict(sq=-8),
       dict(q=None), dict(q=4098), dict(ptr=None), dict(ptr=4104), dict(lens=4098), dict(seq_q=2 ** 29 + 1),
       dict(seq_k=2 ** 29 + 1), dict(batch=2 ** 20, seq_q=2 ** 20)]


def front(a):
    p = a["ptr"]
    return [a["dtype"], a["q"], p, p, a["ldq"], a["sq"], a["ldkv"], a["skv"], a["lens"], a["lens"], 0, a["window"], a["first"]]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **bad}
    p = a["ptr"]
    back = [a["batch"], a["seq_q"], a["seq_k"], a["heads"], a["kv"], a["dim"], a["scale"]]
    for name, middle in (("omHipAttentionWindowForwardHalf", [p, p]), ("omHipAttentionWindowBackwardHalf", [p] * 6)):
        with pytest.raises(om.OmHipError, match=name):
            om.call(name, *front(a), *middle, *back)


@pytest.mark.parametrize("sq,skv", [(0, 640), (1280, 0), (1272, 640), (1280, 56)], ids=str)
def test_overlapping_gradients_are_refused(sq, skv):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, "sq": sq, "skv": skv}
    with pytest.raises(om.OmHipError, match="overlap"):
        om.call("omHipAttentionWindowBackwardHalf", *front(a), *[4096] * 6, 2, 10, 10, 2, 1, 64, 0.125)
