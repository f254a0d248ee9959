"""Attention's gradients for training against differences of the loss sum(softmax(scale Q K^T) V * grad) in float64, which
knows nothing of log-sum-exps, delta or the backward pass's formulas.

The directions are the computed gradient itself (the slope is then its norm) and random ones. A gradient is contracted with
its direction d first, so a tolerance along d is (u = 2^-24, uh half a step of the type; signs of errors unknown):
* dV: P rounds to the type and is off by ep = 2 (D + 3) u max sum |scale q k| + 4 u (|S| + |lse|) + 8 u, its sums by
  (n + 4) u: (uh + ep) sum_ij P_ij |dO_i d_j| + (n + 4) u sum_ij P_ij sum |dO_i| |d_j|;
* dQ: dS is off by e = P (ep (|dP| + |delta|) + (D + 2) u (sum |dO V| + sum |dO O|)) + (uh + 2 u) |dS|, so
  sum_ij e_ij |scale k_j d_i|, and (n + 2) u of the sums' magnitudes. delta takes the context as it was rounded: row i's is off
  by r_i = (2 uh + ep + (n + 4) u) sum_d |dO_id| (P |V|)_id (its weights and its result round), which moves the slope by
  r_i |sum_j P_ij scale k_j d_i|; dK likewise with q_i d_j;
* binary16 weights and dS below 2^-33 of the largest, and the result's own rounding, uh |result| |d| and 2^-25 |d|.
The five-point difference is good to 1e-6 of the slope and of sum |grad| eps here."""
import numpy as np
import pytest

import oracle as O
from test_gpu_attn_train import U, Case, bits, value

CASES = [dict(Sq=40, Sk=60, H=4, Hkv=2, D=32, causal=True, klens=55), dict(Sq=130, Sk=70, H=2, Hkv=1, D=64, causal=True),
         dict(Sq=33, Sk=300, H=3, Hkv=3, D=128), dict(Sq=64, Sk=64, H=6, Hkv=2, D=24, scale=-0.4), dict(Sq=1, Sk=90, H=2, Hkv=2, D=64),
         dict(Sq=20, Sk=1500, H=2, Hkv=2, D=40, qlens=17)]


class Problem:
    """One image in float64: parts (Q [Sq, H, D], K and V [Sk, Hkv, D]), gradient, what a query sees."""

    def __init__(self, parts, grad, scale, causal=False, qlens=None, klens=None):
        self.parts, self.grad, self.scale = [p.astype(np.float64) for p in parts], grad.astype(np.float64), scale
        Sq, Sk = parts[0].shape[0], parts[1].shape[0]
        i, j = np.arange(Sq)[:, None], np.arange(Sk)[None]
        self.see = (i < (Sq if qlens is None else qlens)) & (j < (Sk if klens is None else klens)) & ((j <= i + Sk - Sq) | (not causal))
        self.some = self.see.any(1)
        self.heads, self.group = parts[0].shape[1], parts[0].shape[1] // parts[1].shape[1]

    def head(self, h, parts=None):
        q, k, v = parts or self.parts
        return q[:, h], k[:, h // self.group], v[:, h // self.group]

    def loss(self, parts):
        total = 0.0
        for h in range(self.heads):
            q, k, v = self.head(h, parts)
            S = np.where(self.see, self.scale * q @ k.T, -np.inf)[self.some]
            P = np.exp(S - S.max(1, keepdims=True))
            total += ((P / P.sum(1, keepdims=True)) @ v * self.grad[self.some, h]).sum()
        return total

    def slope(self, i, d, h=1e-3):
        f = lambda t: self.loss([p + t * d if n == i else p for n, p in enumerate(self.parts)])  # noqa: E731
        return (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)

    def weights(self, h, see=None):
        """P, dP, delta, dS of a head."""
        see = self.see if see is None else see
        q, k, v = self.head(h)
        some = see.any(1)[:, None]
        S = np.where(see, self.scale * q @ k.T, -np.inf)
        e = np.exp(S - np.where(some, S.max(1, keepdims=True), 0))
        P = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
        g = np.where(some, self.grad[:, h], 0)
        dP, delta = g @ v.T, (g * (P @ v)).sum(1, keepdims=True)
        return P, dP, delta, P * (dP - delta), g

    def gradients(self, mistake=None):
        """The formulas, with one mistake."""
        out = [np.zeros(p.shape) for p in self.parts]
        Sq, Sk = self.see.shape
        for h in range(self.heads):
            see = self.see
            if mistake == "mask by one":
                see = self.see & (np.arange(Sk)[None] < np.arange(Sq)[:, None] + Sk - Sq)
            P, dP, delta, dS, g = self.weights(h, see)
            if mistake == "no delta":
                dS = P * dP
            if mistake == "half delta":
                dS = P * (dP - delta / 2)
            q, k, _ = self.head(h)
            kv = h // self.group
            add = [self.scale * dS @ k, self.scale * dS.T @ q, P.T @ g]
            if mistake == "no scale":
                add[:2] = [a / self.scale for a in add[:2]]
            if mistake == "twentieth more":
                add = [1.05 * a for a in add]
            out[0][:, h] = add[0]
            for i in (1, 2):
                out[i][:, kv] = add[i] + (0 if mistake == "last head" else out[i][:, kv])
        return [np.zeros(o.shape) for o in out] if mistake == "zeros" else out

    def tolerance(self, i, d, result, bf16):
        uh, tiny, least = (2.0 ** -8, 0.0, 0.0) if bf16 else (2.0 ** -11, 2.0 ** -25, 2.0 ** -33)
        D, (Sq, Sk) = self.parts[0].shape[2], self.see.shape
        n, c, total = (Sk if i == 0 else Sq * self.group), abs(self.scale), 0.0
        for h in range(self.heads):
            q, k, v = self.head(h)
            kv = h // self.group
            P, dP, delta, dS, g = self.weights(h)
            S = self.scale * q @ k.T
            lse = np.log(np.where(self.see, np.exp(S), 0).sum(1)[self.some])
            ep = (2 * (D + 3) * U * c * (np.abs(q) @ np.abs(k).T).max() + 4 * U * (np.abs(S[self.see]).max() + np.abs(lse).max()) + 8 * U)
            dh = d[:, h if i == 0 else kv]
            if i == 2:
                along = np.abs(g @ dh.T)
                total += ((uh + ep) * P * along).sum() + (n + 4) * U * (P * (np.abs(g) @ np.abs(dh).T)).sum() + least * along.sum()
                continue
            along = self.scale * (dh @ k.T if i == 0 else q @ dh.T)   # of each (query, key)
            size = c * (np.abs(dh) @ np.abs(k).T if i == 0 else np.abs(q) @ np.abs(dh).T)
            r = (2 * uh + ep + (Sk + 4) * U) * (np.abs(g) * (P @ np.abs(v))).sum(1)
            sums = np.abs(g) @ np.abs(v).T + (np.abs(g) * np.abs(P @ v)).sum(1, keepdims=True)
            e = P * (ep * (np.abs(dP) + np.abs(delta)) + (D + 2) * U * sums) + (uh + 2 * U) * np.abs(dS)
            e += least * np.abs(dS).max(1 - i, keepdims=True)
            total += (e * np.abs(along)).sum() + (r * np.abs((P * along).sum(1))).sum() + (n + 2) * U * (np.abs(dS) * size).sum()
        return 1.01 * (total + ((uh * np.abs(result) + tiny) * np.abs(d)).sum()) + 1e-6 * abs((result * d).sum()) + 1e-12 * np.abs(self.grad).sum()

    def check(self, got, bf16, most):
        """Whether the gradients agree with the differences; the tolerance is to be below `most` of the gradient's norm."""
        ok = True
        for i, g in enumerate(got):
            norm = np.linalg.norm(g)
            if norm == 0:
                return False
            for seed in (None, 1, 2):
                d = g / norm if seed is None else O.randn(g.shape, 70 + 3 * seed + i, 1.0).astype(np.float64)
                d = d / np.linalg.norm(d)
                lim = self.tolerance(i, d, g, bf16)
                if seed is None:
                    print(f"d{'qkv'[i]}: tolerance {lim / norm:.4f} of the norm")
                    assert lim <= most * norm
                ok &= abs((g * d).sum() - self.slope(i, d)) <= lim
        return ok


def rounded(x, bf16):
    return value(bits(x, bf16), bf16)


MEAN = np.float32(0.5)   # of V: delta is then as large as dP, also where many keys average
MOST = {False: 0.01, True: 0.08}   # of the gradient's norm


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=str)
def test_differences_find_mistakes(c, bf16):
    """The formulas in float64 agree with the differences; with a mistake in them they do not."""
    c = dict(c)
    Sq, Sk, H, Hkv, D = (c.pop(k) for k in ("Sq", "Sk", "H", "Hkv", "D"))
    c.setdefault("scale", D ** -0.5)
    parts = [O.randn((Sq, H, D), 1, 1.0), O.randn((Sk, Hkv, D), 2, 1.0), O.randn((Sk, Hkv, D), 3, 1.0) + MEAN]
    p = Problem([rounded(x, bf16) for x in parts], rounded(O.randn((Sq, H, D), 8, 0.1), bf16), **c)
    assert p.check(p.gradients(), bf16, MOST[bf16])
    for mistake in ["zeros", "no delta", "half delta", "no scale"] + ["last head"] * (H > Hkv) + ["mask by one"] * c.get("causal", False) \
            + ["twentieth more"] * (not bf16):
        assert not p.check(p.gradients(mistake), bf16, 1.0), mistake


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=str)
def test_gradients_against_differences(hip, c, bf16):
    c = dict(c)
    dims = [1] + [c.pop(k) for k in ("Sq", "Sk", "H", "Hkv", "D")]
    lens = {k: [c[k]] for k in ("qlens", "klens") if k in c}
    dev = Case(hip, *dims, bf16=bf16, seed=31, **{**c, **lens})
    dev.store[2] = rounded(dev.store[2] + MEAN, bf16)
    dev.dev[2].upload(bits(dev.store[2], bf16))
    dev.forward()
    dev.backward()
    got, _ = dev.check()
    p = Problem([dev.part(dev.store, i)[0] for i in range(3)], dev.grad[0], **{**c, "scale": dev.scale})
    assert p.check([g[0].astype(np.float64) for g in got], bf16, MOST[bf16])
