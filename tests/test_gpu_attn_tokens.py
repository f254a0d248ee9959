"""The window's kernel for few queries (a sequence's next tokens): what test_gpu_attn_window does not reach of it, against the
formulas in float64, element by element (attn_views says how far off a result may be)."""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_attn_train import bits, value
from test_gpu_attn_window import Window, run


@pytest.mark.gpu
@pytest.mark.parametrize("what", [0x7fff, 0x7c00], ids=["nan", "inf"])
@pytest.mark.parametrize("Sk,window", [(40, 30), (3000, 2500)], ids=["one workgroup", "several"])
def test_rows_without_a_key_stay_zero_beside_values_that_are_not_finite(hip, Sk, window, what):
    """Queries past their length, and ones before the first key under a causal mask, share tiles with queries that see a value
    of NaN or infinity: theirs are 0 and -inf all the same."""
    c = Window(hip, 2, 5, Sk, 4, 2, 64, causal=True, window=window, first=2, qlens=[3, 5], klens=[Sk, 3], seed=3)
    t = bits(c.store[2], False)
    t[0, Sk - 4], t[1, 1] = what, what
    c.dev[2].upload(t)
    c.forward()
    out, lse = value(c.dout.numpy(), False), c.dlse.numpy()
    for b, rows in ((0, (3, 4)), (1, (0, 1))):   # image 1: five queries on three keys, the first two before them
        for i in rows:
            assert np.all(out[b, i] == 0) and np.all(np.isneginf(lse[b, :, i])), (b, i)
    assert not np.isfinite(out[0, 2]).any() and not np.isfinite(out[1, 4]).any()


# one workgroup for a key head's keys in sight, and several that the last one to arrive joins
WALKS = [(150, 40), (3000, 2500)]
WALK_NAMES = ["one workgroup", "several"]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Sk,window", WALKS, ids=WALK_NAMES)
@pytest.mark.parametrize("D", [8, 24, 32, 40, 72, 96, 104, 128])
def test_head_dimensions(hip, D, Sk, window, bf16):
    """Tiles of 32, 64 and 128 columns, whole and in part."""
    run(hip, 2, 1, Sk, 4, 2, D, bf16=bf16, causal=True, window=window, first=4, klens=[Sk, Sk // 2], seed=D)
    run(hip, 2, 5, Sk, 2, 1, D, bf16=bf16, window=window, first=33, seed=D + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("Sk,window", WALKS, ids=WALK_NAMES)
@pytest.mark.parametrize("Sq,H,Hkv", [(10, 3, 1), (11, 3, 1), (5, 12, 2), (6, 12, 2), (4, 7, 1), (5, 7, 1), (2, 32, 2), (3, 32, 2), (1, 32, 1),
                                      (1, 33, 1), (32, 2, 2), (33, 2, 2)], ids=str)
def test_columns_of_a_key_head(hip, Sq, H, Hkv, Sk, window):
    """Tokens times query heads of a key head, up to the 32 columns that the kernel takes and one token past them."""
    run(hip, 2, Sq, Sk, H, Hkv, 64, bf16=Sq % 2 == 0, causal=Sq % 3 == 0, window=window, first=3, seed=Sq + H)
    run(hip, 1, Sq, Sk, H, Hkv, 128, bf16=Sq % 2 == 1, causal=True, window=window, first=0, seed=Sq + H + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,S", [(3, 3, 30), (6, 2, 9), (6, 1, 5)], ids=str)
def test_packed_and_padded_rows(hip, H, Hkv, S):
    run(hip, 3, S, S, H, Hkv, 40, packed=True, pad=16, causal=True, window=6, first=1, seed=H)
    run(hip, 3, S, 2200, H, Hkv, 104, bf16=True, pad=8, window=2000, first=5, seed=H + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("D", [24, 64, 128])
@pytest.mark.parametrize("Sk,window", [(250, 30), (2500, 2100)], ids=WALK_NAMES)
def test_lengths_per_image(hip, Sk, window, D, causal):
    """Images without queries or keys, with one, with more queries than keys, and lengths outside their range."""
    run(hip, 8, 8, Sk, 4, 1, D, bf16=D == 128, causal=causal, window=window, first=2, qlens=[0, 1, 8, 8, 3, -5, 400, 5],
        klens=[Sk, 1, 0, 5, Sk, 20, 2 * Sk, 2], seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
@pytest.mark.parametrize("D", [32, 96, 128])
def test_scales(hip, D, scale):
    run(hip, 1, 3, 200, 6, 2, D, scale=scale, bf16=D == 96, window=60, first=1, seed=9)
    run(hip, 1, 1, 2000, 6, 2, D, scale=scale, bf16=D != 96, window=1900, first=1, seed=9)


@pytest.mark.gpu
def test_repeats_agree_and_are_right(hip):
    """Caches of several lengths by several workgroups each, again and again."""
    cases = [Window(hip, 3, 1, 700, 8, 2, 128, bf16=True, causal=True, window=300, first=4, klens=[700, 30, 411], seed=4),
             Window(hip, 16, 1, 2048, 8, 2, 96, causal=True, window=1024, first=4, klens=[128 * i for i in range(1, 17)], seed=5)]
    want = []
    for c in cases:
        c.forward()
        c.backward()
        c.check()
        want.append(c.results()[:2])
    for _ in range(5):
        for c, w in zip(cases, want):
            c.forward()
            assert all(np.array_equal(a, b, equal_nan=a.dtype == np.float32) for a, b in zip(w, c.results()))


@pytest.mark.gpu
@pytest.mark.parametrize("Sk,window", WALKS, ids=WALK_NAMES)
@pytest.mark.parametrize("D", [40, 64, 96])
def test_what_lies_past_a_length_is_not_read(hip, D, Sk, window):
    for bf16 in (False, True):
        c = Window(hip, 2, 6, Sk, 4, 1, D, bf16=bf16, causal=True, window=window, first=2, qlens=[2, 6], klens=[Sk // 2, Sk - 1], seed=5)
        for i, lens in ((0, c.qlens), (1, c.klens), (2, c.klens)):
            t = bits(c.store[i], bf16)
            for b in range(2):
                t[b, lens[b]:] = 0x7fff
            c.dev[i].upload(t)
        g = bits(c.grad, bf16)
        g[0, 2:] = 0x7fff
        c.dgrad.upload(g)
        c.forward()
        c.backward()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_new_keys_straight_into_caches(hip, bf16):
    """Caches of different lengths: a call an image writes its new key's row in place, the same bits as one call into a dense
    buffer; caches of one length: one call for all, at the cache's stride. No other row is touched, and the step's attention
    follows the formulas on the cache as it then is."""
    B, S, H, Hkv, D, dt = 3, 200, 4, 2, 64, 1 if bf16 else 0
    w, kv = (H + 2 * Hkv) * D, Hkv * D
    token = to_dev(hip, bits(O.randn((B, w), 5, 1.0), bf16))
    angle = np.arange(S)[:, None] * 1000.0 ** (-np.arange(D // 2) * 2.0 / D)
    tables = [None, None, to_dev(hip, np.cos(angle).astype(np.float32)), to_dev(hip, np.sin(angle).astype(np.float32))]
    norm = hip.HIPBackend.qkNormRotary
    for lens in ([7, 199, 64], [80, 80, 80]):
        c = Window(hip, B, 1, S, H, Hkv, D, bf16=bf16, causal=True, window=50, first=4, klens=[n + 1 for n in lens], seed=8)
        before = c.dev[1].numpy()
        pos = to_dev(hip, np.array(lens, np.int32))
        q, rows = empty_dev(hip, (B, H * D), np.uint16), empty_dev(hip, (B, kv), np.uint16)
        norm(token.ptr, token.ptr + 2 * H * D, w, w, w, w, *tables, pos, q, rows, H * D, H * D, kv, kv, B, 1, H, Hkv, D, D, S, 1e-6, False, dt)
        mine = c.dev[0]
        if len(set(lens)) == 1:
            norm(token.ptr, token.ptr + 2 * H * D, w, w, w, w, *tables, pos, mine, c.dev[1].ptr + 2 * lens[0] * kv, H * D, H * D, kv, S * kv,
                 B, 1, H, Hkv, D, D, S, 1e-6, False, dt)
        else:
            for b, n in enumerate(lens):
                at = token.ptr + 2 * b * w
                norm(at, at + 2 * H * D, w, w, w, w, *tables, pos.ptr + 4 * b, mine.ptr + 2 * b * H * D, c.dev[1].ptr + 2 * (b * S + n) * kv,
                     H * D, H * D, kv, S * kv, 1, 1, H, Hkv, D, D, S, 1e-6, False, dt)
        after = c.dev[1].numpy()
        for b, n in enumerate(lens):
            assert np.array_equal(after[b, n], rows.numpy()[b])
            after[b, n] = before[b, n]
        assert np.array_equal(after, before) and np.array_equal(mine.numpy().reshape(B, -1), q.numpy())
        c.store[0], c.store[1] = value(mine.numpy(), bf16), value(c.dev[1].numpy(), bf16)
        c.forward()
        c.backward()
        c.check()
