"""An attention block that knows where its tokens are, from the library's entries: a training step

    qkv = x Wqkv; q, k = rotate(norm(q), norm(k)); ctx = attention(q, k, v) in a window, or with a relative bias; y = ctx Wout

with the gradients of x, the weights, the norms' weights and the biases, eager and as a replayed graph, against float64; and
its next tokens one by one, whose keys go normed and rotated straight into a cache.

Bound of the step: it rounds 12 tensors to the type on the longest way (qkv, q and k, P, ctx, dctx, P, dS, dq and dk, dqkv, dx
and the two operands of a weight gradient), uh each of its elements, uh half a step. The maps between them are averages
(softmax), rotations, normalisations and products with matrices of norm about 1; on data of this scale each passes a relative
error on with a factor below 1.5 and the score path, whose S sum D products of rounded factors, below 4: 12 * 4 uh of a
result's Frobenius norm bounds the sum of all.
"""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_attn_train import bits, value

B, SIDE, H, D, EPS = 3, 7, 4, 16, 1e-6
S, C, T = SIDE * SIDE, H * D, B * SIDE * SIDE
WIDE = 2 * SIDE - 1
WINDOW, FIRST = 9, 2


class Block:
    def __init__(self, hip, bf16, biased):
        self.hip, self.bf16, self.dt, self.biased = hip, bf16, 1 if bf16 else 0, biased
        rnd = lambda shape, k, s: value(bits(O.randn(shape, k, s), bf16), bf16)  # noqa: E731
        self.x, self.dy = rnd((T, C), 1, 1.0), rnd((T, C), 2, 0.3)
        self.wqkv, self.wout = rnd((C, 3 * C), 3, C ** -0.5), rnd((C, C), 4, C ** -0.5)
        self.wq, self.wk = (O.randn((D,), 5 + i, 0.2) + np.float32(1) for i in range(2))
        angle = np.arange(S)[:, None] * 100.0 ** (-np.arange(D // 2) * 2.0 / D)
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.at = (np.arange(SIDE)[:, None] * WIDE + np.arange(SIDE)).reshape(-1).astype(np.int32)
        self.table = O.randn((WIDE * WIDE, H), 9, 0.5)
        half = lambda t: to_dev(hip, bits(t, bf16))  # noqa: E731
        self.d = {k: half(getattr(self, k)) for k in ("x", "dy", "wqkv", "wout")}
        self.d.update({k: to_dev(hip, getattr(self, k)) for k in ("wq", "wk", "cos", "sin", "at", "table")})
        self.d["buckets"] = to_dev(hip, np.arange(WIDE * WIDE, dtype=np.int32))
        # q and k once normed lie as in the projection, so that keys and values keep one stride; likewise their gradients
        for k, shape in dict(qkv=(T, 3 * C), turned=(T, 3 * C), ctx=(T, C), y=(T, C), gctx=(T, C), gturned=(T, 3 * C), gqkv=(T, 3 * C),
                             gx=(T, C)).items():
            self.d[k] = empty_dev(hip, shape, np.uint16)
        for k, shape in dict(lse=(B, H, S), f32=(T, 3 * C), gwout=(C, C), gwqkv=(C, 3 * C), gwq=(D,), gwk=(D,),
                             gtable=(WIDE * WIDE, H)).items():
            self.d[k] = empty_dev(hip, shape)

    def product(self, ta, tb, M, N, K, A, Bm, out):
        self.hip.HIPBackend.gemmStridedBatchedHalf(self.dt, ta, tb, 1, M, N, K, self.d[A], M if ta else K, 0, self.d[Bm],
                                                   K if tb else N, 0, self.d[out], N, 0)

    def to_half(self, src, dst, n):
        self.hip.call("omHipConvertF32ToBF16" if self.bf16 else "omHipConvertF32ToF16", self.d[src].ptr, self.d[dst].ptr, n)

    def step(self):
        h, d, bf = self.hip.HIPBackend, self.d, self.bf16
        parts = lambda k: [d[k].ptr + 2 * i * C for i in range(3)]  # noqa: E731
        ld = (3 * C, 3 * C * S)
        norm = (d["wq"], d["wk"], d["cos"], d["sin"], None)
        sizes = (B, S, H, H, D, D, S, EPS, False, self.dt)
        attn = (B, S, S, H, H, D, D ** -0.5, bf)
        bias = (d["table"], d["buckets"], d["at"], d["at"], WIDE * WIDE, WIDE * WIDE, (SIDE - 1) * WIDE + SIDE - 1)
        h.linearHalf(d["x"], d["wqkv"], None, d["qkv"], T, C, 3 * C, bf16=bf, outHalf=True)
        q, k, v = parts("qkv")
        tq, tk, _ = parts("turned")
        h.qkNormRotary(q, k, *ld, *ld, *norm, tq, tk, *ld, *ld, *sizes)
        front = (tq, tk, v, *ld, *ld, None, None, False)
        if self.biased:
            h.attentionBiasForwardHalf(*front, *bias, d["ctx"], d["lse"], *attn)
        else:
            h.attentionWindowForwardHalf(*front, WINDOW, FIRST, d["ctx"], d["lse"], *attn)
        h.linearHalf(d["ctx"], d["wout"], None, d["y"], T, C, C, bf16=bf, outHalf=True)
        # backward
        self.product(1, 0, C, C, T, "ctx", "dy", "gwout")
        self.product(0, 1, T, C, C, "dy", "wout", "f32")
        self.to_half("f32", "gctx", T * C)
        gq, gk, gv = parts("gqkv")
        hq, hk, _ = parts("gturned")
        back = (d["ctx"], d["lse"], d["gctx"], hq, hk, gv)
        if self.biased:
            h.attentionBiasBackwardHalf(*front, *bias, *back, d["gtable"], *attn)
        else:
            h.attentionWindowBackwardHalf(*front, WINDOW, FIRST, *back, *attn)
        h.qkNormRotaryBackward(hq, hk, *ld, *ld, q, k, *ld, *ld, *norm, gq, gk, d["gwq"], d["gwk"], *sizes)
        self.product(1, 0, C, 3 * C, T, "x", "gqkv", "gwqkv")
        self.product(0, 1, T, C, 3 * C, "gqkv", "wqkv", "f32")
        self.to_half("f32", "gx", T * C)

    def results(self):
        names = ["gwqkv", "gwout", "gwq", "gwk"] + (["gtable"] if self.biased else [])
        return {**{k: value(self.d[k].numpy(), self.bf16) for k in ("y", "gx")}, **{k: self.d[k].numpy() for k in names}}

    def reference(self):
        x, dy, wqkv, wout = (t.astype(np.float64) for t in (self.x, self.dy, self.wqkv, self.wout))
        heads = lambda t: t.reshape(B, S, H, D).transpose(0, 2, 1, 3)  # noqa: E731
        rows = lambda t: t.transpose(0, 2, 1, 3).reshape(T, C)  # noqa: E731
        turn = np.exp(1j * np.arctan2(self.sin, self.cos).astype(np.float64))

        def rotate(t, by):
            z = (t[..., :D // 2] + 1j * t[..., D // 2:]) * by
            return np.concatenate([z.real, z.imag], -1)
        q0, k0, v = (heads(t) for t in np.split(x @ wqkv, 3, 1))
        inv = [1 / np.sqrt((t * t).mean(-1, keepdims=True) + EPS) for t in (q0, k0)]
        hat = [t * i for t, i in zip((q0, k0), inv)]
        q, k = (rotate(t * w, turn) for t, w in zip(hat, (self.wq, self.wk)))
        i, j = np.arange(S)[:, None], np.arange(S)[None]
        which = self.at[i] - self.at[j] + (SIDE - 1) * WIDE + SIDE - 1
        sc = q @ k.transpose(0, 1, 3, 2) * D ** -0.5
        if self.biased:
            sc = sc + self.table[which].transpose(2, 0, 1)
        else:
            sc = np.where((np.abs(i - j) < WINDOW) | (j < FIRST), sc, -np.inf)
        p = np.exp(sc - sc.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        ctx = rows(p @ v)
        gctx = heads(dy @ wout.T)
        dp = gctx @ v.transpose(0, 1, 3, 2)
        ds = p * (dp - (p * dp).sum(-1, keepdims=True))
        back = [rotate(g * D ** -0.5, turn.conj()) for g in (ds @ k, ds.transpose(0, 1, 3, 2) @ q)]
        gw = [(g * t).sum((0, 1, 2)) for g, t in zip(back, hat)]
        gqk = [i * (g * w - t * (g * w * t).mean(-1, keepdims=True)) for g, t, i, w in zip(back, hat, inv, (self.wq, self.wk))]
        gqkv = np.concatenate([rows(t) for t in (*gqk, p.transpose(0, 1, 3, 2) @ gctx)], 1)
        gtable = np.zeros(self.table.shape)
        for h in range(H):
            np.add.at(gtable[:, h], which, ds[:, h].sum(0))
        found = dict(y=ctx @ wout, gx=gqkv @ wqkv.T, gwqkv=x.T @ gqkv, gwout=ctx.T @ dy, gwq=gw[0], gwk=gw[1])
        return {**found, "gtable": gtable} if self.biased else found


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True], ids=["window", "bias"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_training_step(hip, bf16, biased):
    uh = 2.0 ** -8 if bf16 else 2.0 ** -11
    block = Block(hip, bf16, biased)
    block.step()
    got = block.results()
    for name, want in block.reference().items():
        off = np.linalg.norm(got[name] - want) / np.linalg.norm(want)
        print(f"{name}: {off / uh:.2f} half steps")
        assert off <= 12 * 4 * uh, name


@pytest.mark.gpu
def test_training_steps_as_graphs(hip):
    """Two graphs that share the stream's workspaces replay in turn, with eager work of the same entries between them."""
    blocks, other = [Block(hip, False, b) for b in (False, True)], Block(hip, True, True)
    want = []
    for b in blocks:
        b.step()
        want.append(b.results())
    graphs = [hip.Graph(b.step) for b in blocks]
    try:
        for _ in range(3):
            for b in blocks:
                for k in ("y", "gx", "gqkv", "gturned", "turned"):
                    b.d[k].upload(np.full(b.d[k].shape, 0x1234, np.uint16))
            for g in graphs:
                g.launch()
            other.step()
            for b, w in zip(blocks, want):
                got = b.results()
                assert all(np.array_equal(got[k], w[k]) for k in w)
    finally:
        for g in graphs:
            g.destroy()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_next_tokens_through_a_cache(hip, bf16):
    """Two sequences' tokens one at a time, keys normed and rotated into the cache's row, against one call over the whole
    sequences on the same keys and queries: the same q and k bit for bit, contexts to the rounding of P and of themselves in
    either (2 uh each) and the lengths' sums, of sum_j P |V|, which is at most max |V|."""
    h = hip.HIPBackend
    n, seqs, hq, hkv, d, window, first = 70, 2, 4, 2, 64, 20, 3
    w = (hq + 2 * hkv) * d
    uh = 2.0 ** -8 if bf16 else 2.0 ** -11
    x = bits(O.randn((seqs, n, w), 21, 1.0), bf16)
    angle = np.arange(100)[:, None] * 1000.0 ** (-np.arange(d // 2) * 2.0 / d)
    tables = [None, None, to_dev(hip, np.cos(angle).astype(np.float32)), to_dev(hip, np.sin(angle).astype(np.float32))]
    qkv = to_dev(hip, x)
    dt, kv = 1 if bf16 else 0, hkv * d
    # whole sequences
    q, k = empty_dev(hip, (seqs, n, hq * d), np.uint16), to_dev(hip, np.zeros((seqs, n, kv), np.uint16))
    v = to_dev(hip, np.ascontiguousarray(x[:, :, (hq + hkv) * d:]))
    h.qkNormRotary(qkv.ptr, qkv.ptr + 2 * hq * d, w, w * n, w, w * n, *tables, None, q, k, hq * d, hq * d * n, kv, kv * n, seqs, n, hq, hkv,
                   d, d, 100, EPS, True, dt)
    out, lse = empty_dev(hip, (seqs, n, hq, d), np.uint16), empty_dev(hip, (seqs, hq, n))
    h.attentionWindowForwardHalf(q, k, v, hq * d, hq * d * n, kv, kv * n, None, None, True, window, first, out, lse, seqs, n, n, hq,
                                 hkv, d, d ** -0.5, bf16)
    want = value(out.numpy(), bf16)
    # token by token; the second sequence starts 5 tokens later, so the two are at different positions
    cache = to_dev(hip, np.full((seqs, n, kv), 0x7fff, np.uint16))
    row_q, row, one = empty_dev(hip, (seqs, hq * d), np.uint16), empty_dev(hip, (seqs, kv), np.uint16), empty_dev(hip, (seqs, 1, hq, d), np.uint16)
    token, one_lse = empty_dev(hip, (seqs, w), np.uint16), empty_dev(hip, (seqs, hq, 1))
    most = np.abs(value(v.numpy(), bf16)).max()
    for t in range(n):
        at = [t, t - 5]
        token.upload(np.stack([x[b, max(at[b], 0)] for b in range(seqs)]))
        pos, lens = to_dev(hip, np.array(at, np.int32)), to_dev(hip, np.array([a + 1 for a in at], np.int32))
        h.qkNormRotary(token.ptr, token.ptr + 2 * hq * d, w, w, w, w, *tables, pos, row_q, row, hq * d, hq * d, kv, kv, seqs, 1, hq, hkv, d, d,
                       100, EPS, True, dt)
        for b in range(seqs):
            if at[b] >= 0:
                hip.call("omHipCopyD2D", cache.ptr + 2 * (b * n + at[b]) * kv, row.ptr + 2 * b * kv, 2 * kv)
        h.attentionWindowForwardHalf(row_q, cache, v, hq * d, hq * d, kv, kv * n, None, lens, True, window, first, one, one_lse, seqs, 1, n,
                                     hq, hkv, d, d ** -0.5, bf16)
        got = value(one.numpy(), bf16)
        for b in range(seqs):
            if at[b] >= 0:
                assert np.all(np.abs(got[b, 0] - want[b, at[b]]) <= 1.01 * (4 * uh + 2.0 ** -15) * most), (t, b)
            else:
                assert np.all(got[b] == 0) and np.all(np.isneginf(one_lse.numpy()[b]))
    assert np.array_equal(cache.numpy()[0], k.numpy()[0])
