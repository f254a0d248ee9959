"""A training step of an attention block over image tokens from the library's entries, eager and as a replayed graph:

    n = group_norm(x); qkv = n Wqkv + bqkv; ctx = attention(qkv); y = x + dropout(ctx Wout + bout)

and the gradients of x and every parameter from dy, against float64 with the same dropout mask.

Bound: forward and backward round 14 tensors to the type on the longest way (n, qkv, P, ctx, projection; dropout's
gradient, dctx, P, dS, dqkv, dn, dx and the two operands of a weight gradient), uh each of its elements, uh half a step.
The block's maps between them are averages (softmax), products with matrices of norm about 1 and a normalisation; on
data of this scale each passes a relative error on with a factor below 1.5 and the score path, whose S sum D products
of rounded factors, below 4: 14 * 4 uh of a result's Frobenius norm bounds the sum of all.
"""
import numpy as np
import pytest

import oracle as O
import test_gpu_attn_train as attention
import test_gpu_group_norm as group_norm
from conftest import empty_dev, to_dev
from test_gpu_attn_train import bits, value
from test_gpu_dropout import factor, mask, state

pytestmark = pytest.mark.gpu

B, S, H, D, G = 3, 50, 4, 16, 8
C = H * D
T = B * S
P, SEED, STEP, STREAM, EPS = 0.2, 77, 5, 9, 1e-5


class Block:
    def __init__(self, hip, bf16):
        self.hip, self.bf16, self.dt = hip, bf16, 1 if bf16 else 0
        rnd = lambda shape, k, s: value(bits(O.randn(shape, k, s), bf16), bf16)  # noqa: E731
        self.x, self.dy = rnd((T, C), 1, 1.0), rnd((T, C), 2, 0.3)
        self.wqkv, self.wout = rnd((C, 3 * C), 3, C ** -0.5), rnd((C, C), 4, C ** -0.5)
        self.bqkv, self.bout = O.randn((3 * C,), 5, 0.1), O.randn((C,), 6, 0.1)
        self.gamma, self.beta = O.randn((C,), 7, 0.2) + np.float32(1), O.randn((C,), 8, 0.2)
        half = lambda t: to_dev(hip, bits(t, bf16))  # noqa: E731
        self.d = {k: half(getattr(self, k)) for k in ("x", "dy", "wqkv", "wout")}
        self.d.update({k: to_dev(hip, getattr(self, k)) for k in ("bqkv", "bout", "gamma", "beta")})
        for k, shape in dict(n=(T, C), qkv=(T, 3 * C), ctx=(T, C), proj=(T, C), y=(T, C), gproj=(T, C), gctx=(T, C), gqkv=(T, 3 * C),
                             gn=(T, C), gx=(T, C)).items():
            self.d[k] = empty_dev(hip, shape, np.uint16)
        for k, shape in dict(mean=(B, G), inv=(B, G), lse=(B, H, S), gbout=(C,), f32=(T, 3 * C), gwout=(C, C), gwqkv=(C, 3 * C), gbqkv=(3 * C,),
                             ggamma=(C,), gbeta=(C,)).items():
            self.d[k] = empty_dev(hip, shape)
        self.rng = state(hip, SEED, STEP)

    def product(self, ta, tb, M, N, K, A, Bm, out):
        """out (fp32) = A Bm, ta / tb: stored transposed"""
        self.hip.HIPBackend.gemmStridedBatchedHalf(self.dt, ta, tb, 1, M, N, K, self.d[A], M if ta else K, 0, self.d[Bm],
                                                   K if tb else N, 0, self.d[out], N, 0)

    def to_half(self, src, dst, n):
        self.hip.call("omHipConvertF32ToBF16" if self.bf16 else "omHipConvertF32ToF16", self.d[src].ptr, self.d[dst].ptr, n)

    def step(self):
        h, d, bf = self.hip.HIPBackend, self.d, self.bf16
        h.groupNormNhwc(d["x"], d["gamma"], d["beta"], d["n"], d["mean"], d["inv"], B, S, C, G, EPS, 0, self.dt)
        h.linearHalf(d["n"], d["wqkv"], d["bqkv"], d["qkv"], T, C, 3 * C, bf16=bf, outHalf=True)
        qkv, gqkv = ([d[k].ptr + 2 * i * C for i in range(3)] for k in ("qkv", "gqkv"))
        attn = (3 * C, 3 * C * S, 3 * C, 3 * C * S, None, None, False)
        sizes = (B, S, S, H, H, D, D ** -0.5)
        h.attentionTrainForwardHalf(*qkv, *attn, d["ctx"], d["lse"], *sizes, bf16=bf)
        h.linearHalf(d["ctx"], d["wout"], None, d["proj"], T, C, C, bf16=bf, outHalf=True)
        h.dropout(d["proj"], d["bout"], d["x"], d["y"], T, C, P, self.rng, STREAM, self.dt)
        # backward
        h.dropoutBackward(d["dy"], d["gproj"], d["gbout"], T, C, P, self.rng, STREAM, self.dt)
        self.product(1, 0, C, C, T, "ctx", "gproj", "gwout")
        self.product(0, 1, T, C, C, "gproj", "wout", "f32")
        self.to_half("f32", "gctx", T * C)
        h.attentionBackwardHalf(*qkv, *attn, d["ctx"], d["lse"], d["gctx"], *gqkv, *sizes, bf16=bf)
        self.product(1, 0, C, 3 * C, T, "n", "gqkv", "gwqkv")
        self.hip.call("omHipConvertBF16ToF32" if bf else "omHipConvertF16ToF32", d["gqkv"].ptr, d["f32"].ptr, T * 3 * C)
        h.addBiasBackward(d["f32"], d["gbqkv"], T, 3 * C)
        self.product(0, 1, T, C, 3 * C, "gqkv", "wqkv", "f32")
        self.to_half("f32", "gn", T * C)
        h.groupNormNhwcBackward(d["gn"], d["x"], None, d["mean"], d["inv"], d["gamma"], d["beta"], d["gx"], d["ggamma"],
                                d["gbeta"], B, S, C, G, 0, self.dt)

    def results(self):
        half = {k: value(self.d[k].numpy(), self.bf16) for k in ("y", "gx")}
        return {**half, **{k: self.d[k].numpy() for k in ("gwqkv", "gbqkv", "gwout", "gbout", "ggamma", "gbeta")}}

    def reference(self):
        x, dy, wqkv, wout = (t.astype(np.float64) for t in (self.x, self.dy, self.wqkv, self.wout))
        xg = x.reshape(B, S, G, C // G)
        mu = xg.mean((1, 3), keepdims=True)
        inv = 1 / np.sqrt(xg.var((1, 3), keepdims=True) + EPS)
        xhat = ((xg - mu) * inv).reshape(T, C)
        n = xhat * self.gamma + self.beta
        qkv = n @ wqkv + self.bqkv
        heads = lambda t: t.reshape(B, S, H, D).transpose(0, 2, 1, 3)  # noqa: E731
        rows = lambda t: t.transpose(0, 2, 1, 3).reshape(T, C)  # noqa: E731
        q, k, v = (heads(t) for t in np.split(qkv, 3, 1))
        sc = q @ k.transpose(0, 1, 3, 2) * D ** -0.5
        p = np.exp(sc - sc.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        ctx = rows(p @ v)
        keep = mask(T, C, P, SEED, STEP, STREAM) * factor(P)
        y = x + (ctx @ wout + self.bout) * keep
        g = dy * keep
        gctx = heads(g @ wout.T)
        dp = gctx @ v.transpose(0, 1, 3, 2)
        ds = p * (dp - (p * dp).sum(-1, keepdims=True)) * D ** -0.5
        gqkv = np.concatenate([rows(ds @ k), rows(ds.transpose(0, 1, 3, 2) @ q), rows(p.transpose(0, 1, 3, 2) @ gctx)], 1)
        gn = gqkv @ wqkv.T
        dx = (gn * self.gamma).reshape(B, S, G, C // G)
        xh = xhat.reshape(dx.shape)
        avg = lambda t: t.mean((1, 3), keepdims=True)  # noqa: E731
        gx = (inv * (dx - avg(dx) - xh * avg(dx * xh))).reshape(T, C)
        return dict(y=y, gx=gx, gwqkv=n.T @ gqkv, gbqkv=gqkv.sum(0), gwout=ctx.T @ g, gbout=g.sum(0), ggamma=(gn * xhat).sum(0),
                    gbeta=gn.sum(0))


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_training_step(hip, bf16):
    uh = 2.0 ** -8 if bf16 else 2.0 ** -11
    block = Block(hip, bf16)
    block.step()
    got = block.results()
    for name, want in block.reference().items():
        off = np.linalg.norm(got[name] - want) / np.linalg.norm(want)
        print(f"{name}: {off / uh:.2f} half steps")
        assert off <= 14 * 4 * uh, name


def test_training_step_as_a_graph(hip):
    """Replays with eager work of the same entries between them, then with another step of the generator."""
    block, other = Block(hip, False), Block(hip, True)
    block.step()
    want = block.results()
    g = hip.Graph(block.step)
    try:
        for _ in range(3):
            for k in ("y", "gx", "gqkv"):
                block.d[k].upload(np.full(block.d[k].shape, 0x1234, np.uint16))
            g.launch()
            other.step()
            got = block.results()
            assert all(np.array_equal(got[k], want[k]) for k in want)
        block.rng.upload(np.array([SEED, STEP + 1], np.uint64))
        g.launch()
        again = block.results()["y"]
        block.step()
        assert np.array_equal(again, block.results()["y"]) and not np.array_equal(again, want["y"])
    finally:
        g.destroy()


# ---------------------------------------------------------------- each call from what the step left before it
class Left:
    """A buffer that the step left, in another shape."""

    def __init__(self, buf, shape):
        self.a = buf.numpy().reshape(shape)

    def numpy(self):
        return self.a


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_each_call_of_the_step(hip, bf16):
    """Every call's results from the tensors that the step itself left as its inputs, element by element: only the call's own
    roundings remain. uh half a step of the type, u = 2^-24; a product of k terms in fp32 is off by (k + 3) u of its terms'
    magnitudes, its bias among them, and by uh of itself where it is rounded to the type. Attention and group norm are held
    to the bounds of their own tests."""
    uh, u, tiny = 2.0 ** -8 if bf16 else 2.0 ** -11, 2.0 ** -24, 0.0 if bf16 else 2.0 ** -25
    block = Block(hip, bf16)
    block.step()
    d, dt = block.d, block.dt
    halves = {k: value(d[k].numpy(), bf16).astype(np.float64) for k in ("n", "qkv", "ctx", "proj", "y", "gproj", "gctx", "gqkv", "gn")}
    x, dy, wqkv, wout = (t.astype(np.float64) for t in (block.x, block.dy, block.wqkv, block.wout))

    def close(name, got, want, size, terms, half=True):
        off, lim = np.abs(got - want), 1.01 * ((terms + 3) * u * size + (uh * np.abs(want) if half else 0.0)) + (tiny if half else 0.0)
        assert np.all(off <= lim), (name, float((off / lim).max()))

    def product(name, a, b, bias=0.0, half=True, got=None):
        got = halves[name] if got is None else got
        close(name, got, a @ b + bias, np.abs(a) @ np.abs(b) + np.abs(bias), a.shape[1], half)

    product("qkv", halves["n"], wqkv, block.bqkv)
    product("proj", halves["ctx"], wout)
    product("gctx", halves["gproj"], wout.T)
    product("gn", halves["gqkv"], wqkv.T)
    product("gwout", halves["ctx"].T, halves["gproj"], half=False, got=d["gwout"].numpy())
    product("gwqkv", halves["n"].T, halves["gqkv"], half=False, got=d["gwqkv"].numpy())
    close("gbqkv", d["gbqkv"].numpy(), halves["gqkv"].sum(0), np.abs(halves["gqkv"]).sum(0), T, half=False)
    keep = mask(T, C, P, SEED, STEP, STREAM) * factor(P)
    kept = (halves["proj"] + block.bout) * keep
    close("y", halves["y"], x + kept, np.abs(x) + np.abs(kept) + np.abs(halves["proj"] * keep), 1)
    close("gproj", halves["gproj"], dy * keep, np.abs(dy * keep), 0)
    close("gbout", d["gbout"].numpy(), (dy * keep).sum(0), np.abs(dy * keep).sum(0), T, half=False)

    attn = object.__new__(attention.Case)   # check() takes what the calls were given and left
    attn.bf16, attn.causal, attn.qlens, attn.klens, attn.packed, attn.widths = bf16, False, None, None, True, [3 * C]
    attn.dims, attn.scale, attn.first = (B, S, S, H, H, D), float(np.float32(D ** -0.5)), [0, C, 2 * C]
    attn.store, attn.grad = [value(d["qkv"].numpy(), bf16).reshape(B, S, 3 * C)], value(d["gctx"].numpy(), bf16).reshape(B, S, H, D)
    attn.dout, attn.dlse, attn.dgrads = Left(d["ctx"], (B, S, H, D)), d["lse"], [Left(d["gqkv"], (B, S, 3 * C))]
    attn.check()
    norm = object.__new__(group_norm.Case)
    norm.dt, norm.a, norm.dims, norm.shift = dt, 0, (B, S, C, G), 0
    norm.x, norm.g = bits(block.x, bf16).reshape(B, S, C), d["gn"].numpy().reshape(B, S, C)
    norm.gamma, norm.beta = block.gamma, block.beta
    norm.y, norm.gx, norm.mean, norm.inv = Left(d["n"], -1), Left(d["gx"], -1), d["mean"], d["inv"]
    norm.ggamma, norm.gbeta = d["ggamma"], d["gbeta"]
    norm.check()
