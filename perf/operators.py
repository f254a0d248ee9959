"""Operators of an attention block's training step over image tokens, as a program that owns its buffers calls them:
attention with saved statistics and its gradient, dropout whose mask is drawn again in the backward pass, and group
norm with an activation on channels-last data.

Inputs and outputs are device tensors; the outputs' buffers, the generator's state and the lengths are in hand before
a call. Where `own` is false the same results come from elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

MAX_PAIRS = 1.4e8    # (query, key, head) triples of a drawn attention: a quarter of the largest listed one's
MAX_TOKENS = 2.5e7   # values of a drawn dropout or group norm: as many as the second largest listed norm has
EPS = 1e-5
ACTS = {"none": 0, "relu": 1, "silu": 2}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DTYPE = {"fp16": 0, "bf16": 1, "fp32": 2}


def attention(name, op, dtype, batch, seq_q, seq_k, heads, kv_heads, head_dim, causal=False, lengths="none", packed=False):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "seq_q": seq_q, "seq_k": seq_k, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal, "lengths": lengths, "packed": packed}


def dropout(name, op, dtype, rows, cols, p, stream, bias=True, residual=True):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "p": p, "stream": stream, "bias": bias,
            "residual": residual}


def group_norm(name, op, dtype, batch, pixels, channels, groups, act):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "pixels": pixels, "channels": channels,
            "groups": groups, "act": act}


def listed():
    return [
        # ViT-B/16 at batch 64: 196 patches and a class token, the projection's packed rows
        attention("forward_vit_b64", "attention_forward", "fp16", 64, 197, 197, 12, 12, 64, packed=True),
        # long token sequences, causal, four query heads to a key head
        attention("forward_causal_4096", "attention_forward", "bf16", 2, 4096, 4096, 16, 4, 128, causal=True),
        # one small image of 7 x 7 patches and a class token: latency
        attention("backward_50_tokens", "attention_backward", "bf16", 1, 50, 50, 4, 4, 64, packed=True),
        attention("backward_vit_b64", "attention_backward", "fp16", 64, 197, 197, 12, 12, 64, packed=True),
        # cross attention to padded sets of keys, one of them empty; a head dimension between the powers of two
        attention("backward_cross_padded", "attention_backward", "fp16", 6, 333, 1001, 8, 8, 96, lengths="both"),
        attention("backward_causal_4096", "attention_backward", "bf16", 2, 4096, 4096, 16, 4, 128, causal=True),
        # the end of a transformer sub-layer in training: output bias, dropout, residual sum
        dropout("dropout_small_odd", "dropout_forward", "fp32", 50, 203, 0.25, 3),
        dropout("dropout_vit_b64", "dropout_forward", "bf16", 64 * 197, 768, 0.1, 1),
        # its gradient, with the bias gradient, at a long batch
        dropout("dropout_backward_long", "dropout_backward", "fp16", 32768, 1024, 0.1, 2),
        # a 56 x 56 feature map of 256 channels (second stage of ResNet-50), batch 32
        group_norm("norm_silu_56", "group_norm_forward", "bf16", 32, 56 * 56, 256, 32, "silu"),
        group_norm("norm_relu_backward_28", "group_norm_backward", "fp16", 32, 28 * 28, 512, 32, "relu"),
        # one image of 7 x 7 pixels: latency; groups of 15 channels
        group_norm("norm_backward_7", "group_norm_backward", "fp32", 1, 7 * 7, 480, 32, "silu"),
    ]


def spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "dropout", "norm"])
    if kind == "attention":
        dim = rng.choice([8, 16, 24, 32, 40, 56, 64, 64, 72, 80, 96, 104, 112, 128, 128])
        kv = rng.randint(1, 8)
        heads = kv * rng.choice([1, 1, 2, 3, 4])
        sq = spread(rng, 1, 4096)   # a few keys at least: the gradient of a softmax over one key is nothing but rounding
        sk = sq if rng.random() < 0.6 and sq >= 8 else spread(rng, 8, 4096)
        most = int(MAX_PAIRS // (sq * sk * heads))
        while most < 1:
            kv, heads = 1, max(1, heads // 2)
            most = int(MAX_PAIRS // (sq * sk * heads))
        return {k: v for k, v in attention("", rng.choice(["attention_forward", "attention_backward"]),
                                           rng.choice(["fp16", "bf16"]), spread(rng, 1, min(64, most)), sq, sk, heads, kv,
                                           dim, rng.random() < 0.4, rng.choice(["none", "none", "keys", "both"]),
                                           sq == sk and rng.random() < 0.5).items() if k != "name"}
    if kind == "dropout":
        cols = spread(rng, 1, 8192)
        rows = spread(rng, 1, max(1, min(65536, int(MAX_TOKENS // cols))))
        c = dropout("", rng.choice(["dropout_forward", "dropout_backward"]), rng.choice(list(TYPES)), rows, cols,
                    rng.choice([0.0, 0.1, 0.2, 0.5, 0.9]), rng.randint(0, 100), rng.random() < 0.6, rng.random() < 0.6)
        return {k: v for k, v in c.items() if k != "name"}
    groups = rng.choice([1, 2, 4, 8, 16, 32])
    channels = groups * spread(rng, 1, 2048 // groups)
    least = -(-16 * groups // channels)   # 16 values in a group: over two, the gradient is nothing but rounding
    pixels = spread(rng, least, min(16384, int(MAX_TOKENS // channels)))
    batch = spread(rng, 1, max(1, min(64, int(MAX_TOKENS // (channels * pixels)))))
    c = group_norm("", rng.choice(["group_norm_forward", "group_norm_backward"]), rng.choice(list(TYPES)), batch,
                   pixels, channels, groups, rng.choice(list(ACTS)))
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------- inputs
class Source:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def randn(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device="cuda") * std + mean).to(dtype)

    def integers(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device="cuda")


def rows_of(t, batch, seq, heads, dim, first):
    """Heads first .. first + heads of token rows [batch, seq, width] as [batch, seq, heads, dim]."""
    return t[:, :, first * dim:(first + heads) * dim].unflatten(2, (heads, dim))


def split(c, t):
    """Q, K and V of a packed [batch, seq, (heads + 2 kv_heads) dim] tensor, or of three."""
    b, h, kv, d = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    if c["packed"]:
        return [rows_of(t, b, c["seq_q"], n, d, at) for n, at in ((h, 0), (kv, h), (kv, h + kv))]
    return [rows_of(x, b, s, n, d, 0) for x, s, n in zip(t, (c["seq_q"], c["seq_k"], c["seq_k"]), (h, kv, kv))]


def attention_buffers(c, make):
    b, h, kv, d, sq, sk = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["seq_q"], c["seq_k"]
    if c["packed"]:
        return make(b, sq, (h + 2 * kv) * d)
    return [make(b, sq, h * d), make(b, sk, kv * d), make(b, sk, kv * d)]


def prepare(case, seed):
    s, c = Source(seed), case
    t = TYPES[c["dtype"]]
    st = {"case": dict(case)}
    if c["op"].startswith("attention"):
        b, h, d, sq, sk = c["batch"], c["heads"], c["head_dim"], c["seq_q"], c["seq_k"]
        st["qkv"] = attention_buffers(c, lambda *shape: s.randn(*shape, dtype=t))
        st["scale"] = 1.0 / math.sqrt(d)
        st["key_lens"] = st["query_lens"] = None
        if c["lengths"] != "none":
            st["key_lens"] = (s.integers(1001, b) * sk // 1000).clamp_min(min(sk, 8)).to(torch.int32)
            if b > 2:   # an image without keys, and one without padding
                st["key_lens"][0], st["key_lens"][1] = 0, sk
            if c["lengths"] == "both":
                st["query_lens"] = (s.integers(1001, b) * sq // 1000).clamp_min(min(sq, 8)).to(torch.int32)
                if sq == sk:
                    st["query_lens"] = st["key_lens"].clone()
        st["out"] = torch.empty((b, sq, h, d), dtype=t, device="cuda")
        st["lse"] = torch.empty((b, h, sq), dtype=torch.float32, device="cuda")
        if c["op"] == "attention_backward":
            out, lse = attention_forward(st)
            st["out"].copy_(out)
            st["lse"].copy_(lse)
            st["grad"] = s.randn(b, sq, h, d, std=0.1, dtype=t)
            st["grads"] = attention_buffers(c, lambda *shape: torch.empty(shape, dtype=t, device="cuda"))
    elif c["op"].startswith("dropout"):
        shape = (c["rows"], c["cols"])
        st["x"] = s.randn(*shape, dtype=t)
        st["bias"] = s.randn(c["cols"], std=0.1) if c["bias"] else None
        st["residual"] = s.randn(*shape, dtype=t) if c["residual"] else None
        st["rng"] = s.integers(1 << 62, 2)   # the generator's state: seed, step
        st["out"] = torch.empty(shape, dtype=t, device="cuda")
        st["grad_bias"] = torch.empty(c["cols"], device="cuda") if c["bias"] else None
    else:
        n, p, ch, g = c["batch"], c["pixels"], c["channels"], c["groups"]
        st["x"] = s.randn(n, p, ch, std=1.5, mean=0.5, dtype=t)
        st["gamma"], st["beta"] = s.randn(ch, std=0.2, mean=1.0), s.randn(ch, std=0.2)
        st["y"] = torch.empty((n, p, ch), dtype=t, device="cuda")
        st["mean"], st["inv_std"] = torch.empty((n, g), device="cuda"), torch.empty((n, g), device="cuda")
        if c["op"] == "group_norm_backward":
            for k, v in norm_forward(st).items():
                st[k].copy_(v)
            st["grad"] = s.randn(n, p, ch, std=0.1, dtype=t)
            st["grad_x"] = torch.empty((n, p, ch), dtype=t, device="cuda")
            st["grad_gamma"], st["grad_beta"] = torch.empty(ch, device="cuda"), torch.empty(ch, device="cuda")
    return st


# ---------------------------------------------------------------- the framework's calls
def ptr(t):
    return None if t is None else t.data_ptr()


def call_attention(st):
    import omnimatchdeeplearningtool_amd as om
    c = st["case"]
    q, k, v = split(c, st["qkv"])
    sizes = (c["batch"], c["seq_q"], c["seq_k"], c["heads"], c["kv_heads"], c["head_dim"], st["scale"])
    strides = (q.stride(1), q.stride(0), k.stride(1), k.stride(0))
    masks = (ptr(st["query_lens"]), ptr(st["key_lens"]), c["causal"])
    bf16 = c["dtype"] == "bf16"
    if c["op"] == "attention_forward":
        om.HIPBackend.attentionTrainForwardHalf(ptr(q), ptr(k), ptr(v), *strides, *masks, ptr(st["out"]), ptr(st["lse"]),
                                                *sizes, bf16=bf16)
        return {"out": st["out"], "lse": st["lse"]}
    dq, dk, dv = split(c, st["grads"])
    om.HIPBackend.attentionBackwardHalf(ptr(q), ptr(k), ptr(v), *strides, *masks, ptr(st["out"]), ptr(st["lse"]),
                                        ptr(st["grad"]), ptr(dq), ptr(dk), ptr(dv), *sizes, bf16=bf16)
    return {"dq": dq, "dk": dk, "dv": dv}


def call_dropout(st):
    import omnimatchdeeplearningtool_amd as om
    c = st["case"]
    where = (c["rows"], c["cols"], c["p"], ptr(st["rng"]), c["stream"], DTYPE[c["dtype"]])
    if c["op"] == "dropout_forward":
        om.HIPBackend.dropout(ptr(st["x"]), ptr(st["bias"]), ptr(st["residual"]), ptr(st["out"]), *where)
        return {"out": st["out"]}
    om.HIPBackend.dropoutBackward(ptr(st["x"]), ptr(st["out"]), ptr(st["grad_bias"]), *where)
    return {"grad_x": st["out"], "grad_bias": st["grad_bias"]}


def call_norm(st):
    import omnimatchdeeplearningtool_amd as om
    c = st["case"]
    sizes = (c["batch"], c["pixels"], c["channels"], c["groups"])
    if c["op"] == "group_norm_forward":
        om.HIPBackend.groupNormNhwc(ptr(st["x"]), ptr(st["gamma"]), ptr(st["beta"]), ptr(st["y"]), ptr(st["mean"]),
                                    ptr(st["inv_std"]), *sizes, EPS, ACTS[c["act"]], DTYPE[c["dtype"]])
        return {k: st[k] for k in ("y", "mean", "inv_std")}
    om.HIPBackend.groupNormNhwcBackward(ptr(st["grad"]), ptr(st["x"]), ptr(st["y"]), ptr(st["mean"]), ptr(st["inv_std"]),
                                        ptr(st["gamma"]), ptr(st["beta"]), ptr(st["grad_x"]), ptr(st["grad_gamma"]),
                                        ptr(st["grad_beta"]), *sizes, ACTS[c["act"]], DTYPE[c["dtype"]])
    return {k: st[k] for k in ("grad_x", "grad_gamma", "grad_beta")}


# ---------------------------------------------------------------- attention, plain
# S = scale Q K^T over the keys a query sees, lse = log sum exp S, O = exp(S - lse) V. Query i sees key j where
# j < its image's key length and, if causal, j <= i + seq_k - seq_q. A query that sees none, or lies past its image's
# query length, has O = 0 and lse = -inf, and no gradient goes through it.
def visible(st):
    """[batch, 1, seq_q, seq_k] truth values."""
    c = st["case"]
    i = torch.arange(c["seq_q"], device="cuda").view(1, 1, -1, 1)
    j = torch.arange(c["seq_k"], device="cuda").view(1, 1, 1, -1)
    see = torch.ones((c["batch"], 1, c["seq_q"], c["seq_k"]), dtype=torch.bool, device="cuda")
    if st["key_lens"] is not None:
        see &= j < st["key_lens"].view(-1, 1, 1, 1)
    if st["query_lens"] is not None:
        see &= i < st["query_lens"].view(-1, 1, 1, 1)
    if c["causal"]:
        see &= j <= i + (c["seq_k"] - c["seq_q"])
    return see


def heads_first(t, heads):
    """[batch, seq, kv, dim] -> float32 [batch, heads, seq, dim], each kv head repeated for the heads that read it."""
    t = t.float().transpose(1, 2)
    return t.unsqueeze(2).expand(-1, -1, heads // t.shape[1], -1, -1).flatten(1, 2).contiguous()


def scores(st):
    c = st["case"]
    q, k, v = (heads_first(t, c["heads"]) for t in split(c, st["qkv"]))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(st["scale"])
    return q, k, v, s.masked_fill_(~visible(st), -math.inf)


def attention_forward(st):
    c = st["case"]
    _, _, v, s = scores(st)
    top = s.amax(3, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(s - top)
    total = e.sum(3, keepdim=True)
    lse = (total.log() + top).squeeze(3)
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2).to(TYPES[c["dtype"]]), lse


def attention_backward(st):
    c = st["case"]
    t = TYPES[c["dtype"]]
    q, k, v, s = scores(st)
    lse = st["lse"].unsqueeze(3)
    p = torch.where(torch.isinf(s), 0.0, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)))
    g = st["grad"].float().transpose(1, 2).contiguous()
    o = st["out"].float().transpose(1, 2)
    delta = (g * o).sum(3, keepdim=True)
    ds = p * (torch.matmul(g, v.transpose(2, 3).contiguous()) - delta)
    dq = torch.matmul(ds, k) * st["scale"]
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * st["scale"]
    g = torch.where(torch.isinf(lse), 0.0, g)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
    shared = lambda x: x.unflatten(1, (c["kv_heads"], -1)).sum(2)  # noqa: E731
    return {"dq": dq.transpose(1, 2).to(t), "dk": shared(dk).transpose(1, 2).to(t), "dv": shared(dv).transpose(1, 2).to(t)}


# ---------------------------------------------------------------- dropout, plain
# Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC11): counter (group, stream, step's low word, step's high word), key the
# seed's low and high word; a group is 8 columns of a row, and its column j takes 16 bits, the low half of word j / 2
# where j is even. Kept where the bits are at least round(65536 p); kept values are scaled by 65536 / (65536 - that).
def threshold(p):
    return int(math.floor(float(np.float32(p)) * 65536.0 + 0.5))


def kept(st):
    c = st["case"]
    low = 0xFFFFFFFF
    per_row = (c["cols"] + 7) // 8
    w = [torch.arange(c["rows"] * per_row, device="cuda") & low, torch.full((1,), c["stream"], device="cuda"),
         (st["rng"][1:] & low), (st["rng"][1:] >> 32) & low]
    k0, k1 = st["rng"][:1] & low, (st["rng"][:1] >> 32) & low
    for _ in range(10):
        a, b = w[0] * 0xD2511F53, w[2] * 0xCD9E8D57
        w = [((b >> 32) & low) ^ w[1] ^ k0, b & low, ((a >> 32) & low) ^ w[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([x.expand(w[0].shape) for x in w], 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).view(c["rows"], per_row * 8)[:, :c["cols"]]
    return bits >= threshold(c["p"])


def dropout_scale(p):
    left = 65536 - threshold(p)
    return 65536.0 / left if left else 0.0


def dropout_forward(st):
    c = st["case"]
    x = st["x"].float()
    if st["bias"] is not None:
        x = x + st["bias"]
    x = torch.where(kept(st), x * dropout_scale(c["p"]), 0.0)
    if st["residual"] is not None:
        x = x + st["residual"].float()
    return {"out": x.to(TYPES[c["dtype"]])}


def dropout_backward(st):
    c = st["case"]
    g = torch.where(kept(st), st["x"].float() * dropout_scale(c["p"]), 0.0)
    return {"grad_x": g.to(TYPES[c["dtype"]]), "grad_bias": g.sum(0, dtype=torch.float64).float() if c["bias"] else None}


# ---------------------------------------------------------------- group norm, plain
# Over an image's pixels and the channels of a group: z = (x - mean) inv_std gamma + beta, y = act(z). ReLU's gate in
# the backward pass is the saved output, SiLU's slope comes from z.
def groups_of(c, t):
    return t.view(c["batch"], -1, c["groups"], c["channels"] // c["groups"])


def norm_forward(st):
    c = st["case"]
    x = groups_of(c, st["x"].float())
    mean = x.mean((1, 3), keepdim=True)
    inv = 1.0 / torch.sqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
    z = ((x - mean) * inv).flatten(2) * st["gamma"] + st["beta"]
    z = z.clamp_min(0.0) if c["act"] == "relu" else z / (1.0 + torch.exp(-z)) if c["act"] == "silu" else z
    return {"y": z.to(TYPES[c["dtype"]]), "mean": mean.flatten(1), "inv_std": inv.flatten(1)}


def norm_backward(st):
    c = st["case"]
    inv = st["inv_std"].view(c["batch"], 1, -1, 1)
    xhat = (groups_of(c, st["x"].float()) - st["mean"].view(c["batch"], 1, -1, 1)) * inv
    g = st["grad"].float()
    if c["act"] == "relu":
        g = torch.where(st["y"] > 0, g, 0.0)
    if c["act"] == "silu":
        z = xhat.flatten(2) * st["gamma"] + st["beta"]
        gate = 1.0 / (1.0 + torch.exp(-z))
        g = g * gate * (1.0 + z * (1.0 - gate))
    grad_gamma, grad_beta = (g * xhat.flatten(2)).sum((0, 1)), g.sum((0, 1))
    g = groups_of(c, g * st["gamma"])
    gx = inv * (g - g.mean((1, 3), keepdim=True) - xhat * (g * xhat).mean((1, 3), keepdim=True))
    return {"grad_x": gx.flatten(2).to(TYPES[c["dtype"]]), "grad_gamma": grad_gamma, "grad_beta": grad_beta}


def run(state):
    op = state["case"]["op"]
    if own:
        return (call_attention if op.startswith("attention") else call_dropout if op.startswith("dropout") else call_norm)(state)
    if op == "attention_forward":
        out, lse = attention_forward(state)
        return {"out": out, "lse": lse}
    return {"attention_backward": attention_backward, "dropout_forward": dropout_forward, "dropout_backward": dropout_backward,
            "group_norm_forward": norm_forward, "group_norm_backward": norm_backward}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"].startswith("attention"):
        sq, sk, h, d, b = c["seq_q"], c["seq_k"], c["heads"], c["head_dim"], c["batch"]
        pairs = sq * sk
        if c["causal"]:   # query i sees i + sk - sq + 1 keys
            first = max(0, sq - sk)
            n = sq - first
            low = sk - sq + 1 + first
            pairs = n * low + n * (n - 1) // 2
        part = 1.0 if c["lengths"] == "none" else 0.5 if c["lengths"] == "keys" or sq == sk else 0.25
        q, kv = b * sq * h * d * size, 2 * b * sk * c["kv_heads"] * d * size
        if c["op"] == "attention_forward":
            return {"bytes": 2 * q + kv + 4 * b * h * sq, "flops": 4.0 * d * b * h * pairs * part}
        return {"bytes": 4 * q + 2 * kv + 4 * b * h * sq, "flops": 10.0 * d * b * h * pairs * part}
    if c["op"].startswith("dropout"):
        n = c["rows"] * c["cols"]
        tensors = 3 if c["op"] == "dropout_forward" and c["residual"] else 2
        return {"bytes": n * size * tensors + 4 * c["cols"] * c["bias"] + 16, "flops": 30.0 * n}
    n = c["batch"] * c["pixels"] * c["channels"]
    tensors = 2 if c["op"] == "group_norm_forward" else 4 if c["act"] == "relu" else 3
    return {"bytes": n * size * tensors + 16 * c["channels"] + 8 * c["batch"] * c["groups"], "flops": 12.0 * n * (tensors - 1)}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["op"].startswith("attention"):
        return exact_attention(c, st)
    if c["op"].startswith("dropout"):
        return exact_dropout(c, st)
    return exact_norm(c, st)


def exact_attention(c, st):
    """Image by image and head by head, each query's row from its own visible keys."""
    sq, sk, h, kv = c["seq_q"], c["seq_k"], c["heads"], c["kv_heads"]
    q, k, v = split(c, st["qkv"])
    back = c["op"] == "attention_backward"
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((c["batch"], h, sq), -math.inf, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v)]
    for b in range(c["batch"]):
        nq = sq if st["query_lens"] is None else int(st["query_lens"][b])
        nk = sk if st["key_lens"] is None else int(st["key_lens"][b])
        if not nq or not nk:
            continue
        for j in range(h):
            Q, K, V = q[b, :nq, j].double(), k[b, :nk, j * kv // h].double(), v[b, :nk, j * kv // h].double()
            S = (Q @ K.T.contiguous()) * st["scale"]
            if c["causal"]:
                S = S + torch.full((nq, nk), -math.inf, dtype=torch.float64, device="cuda").triu(sk - sq + 1)
            L = torch.logsumexp(S, 1)
            some = ~torch.isinf(L)
            P = torch.zeros_like(S)
            P[some] = torch.exp(S[some] - L[some, None])
            lse[b, j, :nq] = L
            if not back:
                out[b, :nq, j] = P @ V
                continue
            G = st["grad"][b, :nq, j].double()
            dP = G @ V.T.contiguous()
            dS = P * (dP - (P * dP).sum(1, keepdim=True))
            grads[0][b, :nq, j] = dS @ K * st["scale"]
            grads[1][b, :nk, j * kv // h] += dS.T.contiguous() @ Q * st["scale"]
            grads[2][b, :nk, j * kv // h] += P.T.contiguous() @ G
    return dict(zip(("dq", "dk", "dv"), grads)) if back else {"out": out, "lse": lse}


def exact_dropout(c, st):
    """The generator on unsigned 64-bit words of the host."""
    seed, step = (int(v) for v in st["rng"].cpu())
    per_row = -(-c["cols"] // 8)
    n = c["rows"] * per_row
    x = np.empty((4, n), np.uint64)
    for row, value in zip(x, (np.arange(n), c["stream"], step % 2 ** 32, step // 2 ** 32)):
        row[:] = value
    low, shift = np.uint64(2 ** 32 - 1), np.uint64(32)
    for i in range(10):
        key = [np.uint64((seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32), np.uint64((seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32)]
        one, two = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = np.stack([(two >> shift) ^ x[1] ^ key[0], two & low, (one >> shift) ^ x[3] ^ key[1], one & low])
    bits = x.T.astype(np.uint32).copy().view(np.uint16).reshape(c["rows"], per_row * 8)[:, :c["cols"]]
    border = int(float(np.float32(c["p"])) * 65536 + 0.5)
    keep = torch.from_numpy(bits.astype(np.int32) >= border).cuda()
    factor = 65536 / (65536 - border) if border < 65536 else 0.0
    v = st["x"].double()
    if c["op"] == "dropout_backward":
        v = v * factor * keep
        return {"grad_x": v, "grad_bias": v.sum(0) if c["bias"] else None}
    v = (v + (st["bias"].double() if c["bias"] else 0.0)) * factor * keep
    return {"out": v + st["residual"].double() if c["residual"] else v}


def exact_norm(c, st):
    n, p, g, per = c["batch"], c["pixels"], c["groups"], c["channels"] // c["groups"]
    x = st["x"].double().reshape(n, p, g, per).permute(0, 2, 1, 3).reshape(n, g, p * per)   # a row per group
    rows = lambda v: v.double().reshape(g, 1, per).expand(g, p, per).reshape(1, g, p * per)  # noqa: E731
    back = lambda t: t.reshape(n, g, p, per).permute(0, 2, 1, 3).reshape(n, p, g * per)  # noqa: E731
    var, mean = torch.var_mean(x, 2, unbiased=False, keepdim=True)
    inv = (var + EPS) ** -0.5
    xhat = (x - mean) * inv
    gamma, beta = rows(st["gamma"]), rows(st["beta"])
    z = xhat * gamma + beta
    if c["op"] == "group_norm_forward":
        y = {"none": z, "relu": z * (z > 0), "silu": z * torch.sigmoid(z)}[c["act"]]
        return {"y": back(y), "mean": mean.squeeze(2), "inv_std": inv.squeeze(2)}
    split_up = lambda t: t.double().reshape(n, p, g, per).permute(0, 2, 1, 3).reshape(n, g, p * per)  # noqa: E731
    s = torch.sigmoid(z)
    slope = {"none": torch.ones_like(z), "relu": (split_up(st["y"]) > 0).double(), "silu": s + z * s * (1 - s)}[c["act"]]
    dz = split_up(st["grad"]) * slope
    per_channel = lambda t: t.reshape(n, g, p, per).sum((0, 2)).reshape(-1)  # noqa: E731
    dxhat = dz * gamma
    dx = inv * (dxhat - dxhat.mean(2, keepdim=True) - xhat * (dxhat * xhat).mean(2, keepdim=True))
    return {"grad_x": back(dx), "grad_gamma": per_channel(dz * xhat), "grad_beta": per_channel(dz)}
