"""Attention whose queries see some keys, or see them with a bias, against the formulas in float64, element by element: the
cases of test_gpu_attn_train with what a query sees, and the bias, left to a subclass. Bounds as there (u = 2^-24, uh = 2^-11 /
2^-8), and

* the bias, times log2 e, is off by 2 u of itself and rounded once more as it is added: ep gains 8 u max |bias|;
* a table's gradient sums n unrounded dS, each off by P (ep (|dP| + |delta|) + (D + 2) u (sum |dO V| + sum |dO O|)) + 2 u |dS|,
  in fp32: (n + 4) u sum |dS|;
* what lies below fp32's smallest normal number, f = 2^-126, may become zero: a probability, its rounding, a product or a
  result. A weight is off by 2 f more, dS by 2 f and by f of |dP| + |delta|, a bfloat16 result by f.
"""
import numpy as np

from test_gpu_attn_train import Case, U, value

F = 2.0 ** -126


class Viewed(Case):
    def sizes(self, b):
        """Queries and keys of an image."""
        B, Sq, Sk, *_ = self.dims
        return (Sq if self.qlens is None else int(np.clip(self.qlens[b], 0, Sq)),
                Sk if self.klens is None else int(np.clip(self.klens[b], 0, Sk)))

    def standing(self, b):
        """What an image's queries and keys see without more: [Sq, Sk] truth values, the queries' positions, the keys'."""
        B, Sq, Sk, *_ = self.dims
        nq, nk = self.sizes(b)
        i, j = np.arange(Sq)[:, None], np.arange(Sk)[None]
        p = i + nk - nq
        return (i < nq) & (j < nk) & ((j <= p) if self.causal else True), p, j

    def bias(self, b, h):
        return 0.0

    def table_sums(self, b, h, dS, e, see):
        """Takes a head's dS and their bounds."""

    def check(self):
        B, Sq, Sk, H, Hkv, D = self.dims
        uh, tiny = (2.0 ** -8, F) if self.bf16 else (2.0 ** -11, 2.0 ** -25)
        least = 0.0 if self.bf16 else 2.0 ** -33
        out, lse = value(self.dout.numpy(), self.bf16), self.dlse.numpy()
        raw = [g.numpy() for g in self.dgrads]
        got = [value(np.ascontiguousarray(self.part(raw, i)), self.bf16) for i in range(3)]
        want, bound = [np.zeros(g.shape) for g in got], [np.zeros(g.shape) for g in got]
        c = abs(self.scale)
        for b in range(B):
            for h in range(H):
                q, k, v, see = self.head(b, h)
                bias = np.broadcast_to(self.bias(b, h), see.shape)
                see = see & (bias > -1e30)
                some = see.any(1)
                kv = h * Hkv // H
                S = np.where(see, self.scale * q @ k.T + bias, -np.inf)
                top = np.where(some, S.max(1, initial=-np.inf), 0.0)
                e = np.exp(S - top[:, None])
                L = np.where(some, np.log(np.maximum(e.sum(1), 1e-300)) + top, -np.inf)
                assert np.array_equal(np.isneginf(lse[b, h]), ~some)
                big = c * (np.abs(q) @ np.abs(k).T).max(initial=0.0)
                size = np.abs(S[see]).max(initial=0.0) + np.abs(L[some]).max(initial=0.0)
                ep = 2 * (D + 3) * U * big + 4 * U * size + 8 * U + 8 * U * np.abs(bias[see]).max(initial=0.0)
                assert np.all(np.abs(lse[b, h][some] - L[some]) <= ep + 4 * U * np.abs(L[some]) + (Sk + 4) * U)
                P = np.where(see, np.exp(S - np.where(some, L, 0.0)[:, None]), 0.0)
                ref = P @ v
                lim = (2 * uh + ep + (Sk + 4) * U) * 1.01 * (P @ np.abs(v)) + tiny
                lim += (0 if self.bf16 else 2.0 ** -31 * Sk) * np.abs(v).max(initial=0.0) * P.max(1, initial=0.0)[:, None]
                lim += 2 * F * (see @ np.abs(v))
                off = np.abs(out[b, :, h] - ref)
                assert np.all(off <= lim), (b, h, float((off / lim).max()))
                assert np.all(out[b, ~some, h] == 0)
                g, o = self.grad[b, :, h].astype(np.float64), out[b, :, h].astype(np.float64)
                g = np.where(some[:, None], g, 0.0)
                P = np.where(see, np.exp(S - np.where(some, lse[b, h].astype(np.float64), 0.0)[:, None]), 0.0)
                dP, delta = g @ v.T, (g * o).sum(1, keepdims=True)
                dS = P * (dP - delta)
                e = P * (ep * (np.abs(dP) + np.abs(delta)) + (D + 2) * U * (np.abs(g) @ np.abs(v).T + (np.abs(g) * np.abs(o)).sum(1, keepdims=True)))
                e += 2 * U * np.abs(dS)
                e += np.where(see, F * (2 + np.abs(dP) + np.abs(delta)), 0)
                self.table_sums(b, h, dS, e, see)
                e += uh * np.abs(dS)
                want[0][b, :, h] = self.scale * dS @ k
                eq = e + least * np.abs(dS).max(1, initial=0.0)[:, None]
                bound[0][b, :, h] = c * (eq @ np.abs(k) + (Sk + 2) * U * np.abs(dS) @ np.abs(k))
                want[1][b, :, kv] += self.scale * dS.T @ q
                ek = e + least * np.abs(dS).max(0, initial=0.0)[None]
                bound[1][b, :, kv] += c * (ek.T @ np.abs(q) + (Sq + 2) * (H // Hkv) * U * np.abs(dS).T @ np.abs(q))
                want[2][b, :, kv] += P.T @ g
                bound[2][b, :, kv] += (uh + ep + (Sq + 4) * (H // Hkv) * U) * (P.T @ np.abs(g)) + (least + 2 * F) * np.abs(g).sum(0)
        for name, g, w, lim in zip("qkv", got, want, bound):
            off = np.abs(g - w)
            lim = 1.01 * lim + uh * np.abs(w) * 1.01 + tiny
            assert np.all(off <= lim), ("d" + name, float((off / np.maximum(lim, 1e-300)).max()))
        for i, (t, w) in enumerate(zip(raw, self.widths)):   # nothing outside the heads' columns was touched
            used = sum(self.dims[k] * self.dims[5] for k in ((3, 4, 4) if self.packed else ((3,), (4,), (4,))[i]))
            assert np.all(t[:, :, used:] == 0x1234)
        return got, bound
