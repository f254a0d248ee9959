"""Dropout against its definition on the host: the same bits (Philox4x32-10, with the published known answers), the
values within what their roundings allow.

Bounds (u = 2^-24, uh half a step of the type): the forward pass adds the bias (u), multiplies by s (rounded to fp32: u)
and adds the residual in one fused step (u), each of its value's size, and rounds to the type (uh). A bias gradient adds
n kept values of one product each: (n + 2) u of their magnitudes' sum.
"""
import numpy as np
import pytest

import oracle as O
from conftest import empty_dev, to_dev
from test_gpu_streams import streams  # noqa: F401  (fixture: caller-owned streams)

U = 2.0 ** -24
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8, 2: 2.0 ** -24}
TINY = {0: 2.0 ** -25, 1: 0.0, 2: 0.0}   # binary16 below 2^-14


def store(x, dt):
    return x.astype(np.float16).view(np.uint16) if dt == 0 else O.bf16_bits(x) if dt == 1 else x.astype(np.float32)


def value(b, dt):
    return b.view(np.float16).astype(np.float32) if dt == 0 else (b.astype(np.uint32) << 16).view(np.float32) if dt == 1 else b


def philox(counter, key):
    """Ten rounds on python integers: counter 4 words, key 2."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_philox_known_answers():
    """The published vectors of the generator (zeros, ones, digits of pi)."""
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def threshold(p):
    return int(np.floor(float(np.float32(p)) * 65536 + 0.5))


def mask(rows, cols, p, seed, step, stream):
    groups = -(-cols // 8)
    keep = np.empty((rows, groups * 8), bool)
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for g in range(rows * groups):
        words = philox([g, stream & 0xFFFFFFFF, step & 0xFFFFFFFF, step >> 32], key)
        r, c = divmod(g, groups)
        for j in range(8):
            keep[r, 8 * c + j] = ((words[j // 2] >> (16 * (j % 2))) & 0xFFFF) >= threshold(p)
    return keep[:, :cols]


def factor(p):
    return 65536 / (65536 - threshold(p)) if threshold(p) < 65536 else 0.0


def state(hip, seed, step):
    return to_dev(hip, np.array([seed, step], np.uint64))


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 9), (33, 16), (7, 203), (300, 24), (64, 520), (17, 1001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", SHAPES, ids=str)
def test_values(hip, rows, cols, dt):
    print(f"case {rows}x{cols} dtype {dt}", flush=True)
    p = (0.1, 0.5, 0.25)[(rows + cols) % 3]
    seed, step, stream = 0x123456789ABCDEF0 + rows, (1 << 40) + cols, rows
    rng = state(hip, seed, step)
    keep = mask(rows, cols, p, seed, step, stream)
    x, res = (store(O.randn((rows, cols), k, 1.0), dt) for k in (rows, cols + 1))
    bias = O.randn((cols,), 3, 0.1)
    dx, dres, dbias = to_dev(hip, x), to_dev(hip, res), to_dev(hip, bias)
    vx, vres = value(x, dt).astype(np.float64), value(res, dt).astype(np.float64)
    for b, r in ((True, True), (False, False), (True, False), (False, True)):
        out = empty_dev(hip, x.shape, x.dtype)
        hip.HIPBackend.dropout(dx, dbias if b else None, dres if r else None, out, rows, cols, p, rng, stream, dt)
        kept = (vx + (bias if b else 0.0)) * factor(p)
        want = np.where(keep, kept, 0.0) + (vres if r else 0.0)
        off = np.abs(value(out.numpy(), dt) - want)
        lim = 1.01 * (3 * U * (np.abs(kept) + np.abs(vres)) + HALF_STEP[dt] * np.abs(want)) + TINY[dt]
        assert np.all(off <= lim), float((off / lim).max())
    # gradient, in place too; the bias gradient from unrounded values
    want = np.where(keep, vx * factor(p), 0.0)
    for with_bias in (True, False):
        gx, gb = empty_dev(hip, x.shape, x.dtype), empty_dev(hip, (cols,))
        hip.HIPBackend.dropoutBackward(dx, gx, gb if with_bias else None, rows, cols, p, rng, stream, dt)
        off = np.abs(value(gx.numpy(), dt) - want)
        assert np.all(off <= 1.01 * (2 * U + HALF_STEP[dt]) * np.abs(want) + TINY[dt])
        if with_bias:
            assert np.all(np.abs(gb.numpy() - want.sum(0)) <= 1.01 * (rows + 2) * U * np.abs(want).sum(0))
            again = empty_dev(hip, (cols,))
            place = to_dev(hip, x)
            hip.HIPBackend.dropoutBackward(place, place, again, rows, cols, p, rng, stream, dt)
            assert np.array_equal(again.numpy(), gb.numpy()) and np.array_equal(place.numpy(), gx.numpy())
    # in place over the input and over the residual
    hip.HIPBackend.dropout(dx, dbias, dres, out, rows, cols, p, rng, stream, dt)
    first = out.numpy()
    hip.HIPBackend.dropout(dx, dbias, dres, dres, rows, cols, p, rng, stream, dt)
    assert np.array_equal(dres.numpy(), first)
    dres.upload(res)
    hip.HIPBackend.dropout(dx, dbias, dres, dx, rows, cols, p, rng, stream, dt)
    assert np.array_equal(dx.numpy(), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp16", "bf16", "fp32"])
def test_addresses_off_the_vector(hip, dt):
    """Rows that start anywhere: one element past an allocation's start, an odd number of columns."""
    rows, cols, p = 9, 77, 0.5
    size = 4 if dt == 2 else 2
    rng = state(hip, 5, 6)
    x = store(O.randn((rows * cols + 1,), 1, 1.0), dt)
    dx, out = to_dev(hip, x), empty_dev(hip, x.shape, x.dtype)
    gb = empty_dev(hip, (cols + 1,))
    hip.HIPBackend.dropout(dx.ptr + size, None, None, out.ptr + size, rows, cols, p, rng, 0, dt)
    want = np.where(mask(rows, cols, p, 5, 6, 0), value(x[1:], dt).reshape(rows, cols) * 2.0, 0.0)
    assert np.array_equal(value(out.numpy()[1:], dt).reshape(rows, cols), want)   # a factor of 2 is exact
    hip.HIPBackend.dropoutBackward(dx.ptr + size, out.ptr + size, gb.ptr + 4, rows, cols, p, rng, 0, dt)
    assert np.array_equal(value(out.numpy()[1:], dt).reshape(rows, cols), want)
    assert np.all(np.abs(gb.numpy()[1:] - want.sum(0, dtype=np.float64)) <= 1.01 * (rows + 2) * U * np.abs(want).sum(0))


@pytest.mark.gpu
def test_ends_of_the_probability(hip):
    """0 keeps everything as it is, 1 drops everything (NaN and infinities too), and 2^-18 is 0."""
    rows, cols = 6, 50
    x = O.randn((rows, cols), 2, 1.0)
    x[0, 0], x[1, 1], x[2, 2] = np.nan, np.inf, -np.inf
    rng, dx, out = state(hip, 1, 2), to_dev(hip, x), empty_dev(hip, x.shape)
    res = O.randn((rows, cols), 3, 1.0)
    for p in (0.0, 2.0 ** -18):
        hip.HIPBackend.dropout(dx, None, None, out, rows, cols, p, rng, 0)
        assert np.array_equal(out.numpy(), x, equal_nan=True)
    hip.HIPBackend.dropout(dx, None, to_dev(hip, res), out, rows, cols, 1.0, rng, 0)
    assert np.array_equal(out.numpy(), res)
    gb = empty_dev(hip, (cols,))
    hip.HIPBackend.dropoutBackward(dx, out, gb, rows, cols, 1.0, rng, 0)
    assert np.all(out.numpy() == 0) and np.all(gb.numpy() == 0)


@pytest.mark.gpu
def test_share_kept_and_independence(hip):
    """2^20 values: the share kept is within 6 standard deviations of its probability; seeds, steps and streams that
    differ in any 32-bit word give masks that agree as often as independent ones do."""
    rows, cols = 1024, 1024
    ones, out = to_dev(hip, np.ones((rows, cols), np.float32)), empty_dev(hip, (rows, cols))
    n = rows * cols
    for p in (0.1, 0.9):
        hip.HIPBackend.dropout(ones, None, None, out, rows, cols, p, state(hip, 7, 9), 1)
        q = 1 - threshold(p) / 65536
        assert abs((out.numpy() != 0).mean() - q) <= 6 * np.sqrt(q * (1 - q) / n)
    masks = []
    for seed, step, stream in ((7, 9, 1), (8, 9, 1), (7 + (1 << 32), 9, 1), (7, 10, 1), (7, 9 + (1 << 32), 1), (7, 9, 2), (7, 9, -1)):
        hip.HIPBackend.dropout(ones, None, None, out, rows, cols, 0.5, state(hip, seed, step), stream)
        masks.append(out.numpy() != 0)
    for i in range(len(masks)):
        for j in range(i):
            assert abs((masks[i] == masks[j]).mean() - 0.5) <= 6 * 0.5 / np.sqrt(n)


@pytest.mark.gpu
def test_long_batch(hip):
    """Many chunks of rows in the bias gradient: against float64 of the device's own kept values (scale 2, exact)."""
    rows, cols = 20011, 264
    x = O.randn((rows, cols), 4, 1.0)
    dx, gx, gb = to_dev(hip, x), empty_dev(hip, x.shape), empty_dev(hip, (cols,))
    rng = state(hip, 3, 4)
    hip.HIPBackend.dropoutBackward(dx, gx, gb, rows, cols, 0.5, rng, 0)
    g = gx.numpy()
    assert np.all((g == 0) | (g == 2 * x))
    assert np.array_equal(g[5000:5003] != 0, mask(5003, cols, 0.5, 3, 4, 0)[5000:])
    assert np.all(np.abs(gb.numpy() - g.sum(0, dtype=np.float64)) <= 1.01 * (rows + 2) * U * np.abs(g).sum(0, dtype=np.float64))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [512, 509], ids=str)
def test_large_output(hip, cols):
    """Over 24 MB (streaming stores): every value is kept and doubled or dropped, the mask as on the host, forward and
    backward."""
    rows = 13001
    x = O.randn((rows, cols), 6, 1.0)
    dx, out, gx, gb = to_dev(hip, x), empty_dev(hip, x.shape), empty_dev(hip, x.shape), empty_dev(hip, (cols,))
    rng = state(hip, 12, 34)
    hip.HIPBackend.dropout(dx, None, None, out, rows, cols, 0.5, rng, 2)
    hip.HIPBackend.dropoutBackward(dx, gx, gb, rows, cols, 0.5, rng, 2)
    y = out.numpy()
    assert np.all((y == 0) | (y == 2 * x)) and np.array_equal(gx.numpy(), y)
    assert np.array_equal(y[:20] != 0, mask(20, cols, 0.5, 12, 34, 2))
    assert np.all(np.abs(gb.numpy() - y.sum(0, dtype=np.float64)) <= 1.01 * (rows + 2) * U * np.abs(y).sum(0, dtype=np.float64))


@pytest.mark.gpu
def test_replayed_graph_draws_from_the_state(hip, streams):
    """A graph of forward and backward replays with the state of the moment: fresh masks after it changes, the same
    before; eager work of another size runs between the replays."""
    rows, cols, p = 40, 96, 0.5
    x = O.randn((rows, cols), 8, 1.0)
    dx, out, gx, gb = to_dev(hip, x), empty_dev(hip, x.shape), empty_dev(hip, x.shape), empty_dev(hip, (cols,))
    rng = state(hip, 11, 0)
    s = streams.create()
    hip.set_stream(s)

    def step():
        hip.HIPBackend.dropout(dx, None, None, out, rows, cols, p, rng, 5)
        hip.HIPBackend.dropoutBackward(out, gx, gb, rows, cols, p, rng, 5)

    step()
    streams.sync(s)
    g = hip.Graph(step)
    big = to_dev(hip, O.randn((3000, 1000), 9, 1.0))
    big_out, big_gb = empty_dev(hip, (3000, 1000)), empty_dev(hip, (1000,))
    try:
        for now in (0, 0, 1, 2):
            rng.upload(np.array([11, now], np.uint64))
            g.launch()
            streams.sync(s)
            keep = mask(rows, cols, p, 11, now, 5)
            assert np.array_equal(out.numpy(), np.where(keep, 2 * x, 0))
            assert np.array_equal(gx.numpy(), np.where(keep, 4 * x, 0))
            want = np.where(keep, 4 * x, 0).astype(np.float64)
            assert np.all(np.abs(gb.numpy() - want.sum(0)) <= 1.01 * (rows + 2) * U * np.abs(want).sum(0))
            hip.HIPBackend.dropoutBackward(big, big_out, big_gb, 3000, 1000, p, rng, 5)   # grows this stream's workspace
    finally:
        g.destroy()


@pytest.mark.gpu
def test_no_rows(hip):
    gb = to_dev(hip, np.ones(10, np.float32))
    rng = state(hip, 0, 0)
    hip.HIPBackend.dropout(None, None, None, None, 0, 10, 0.5, rng, 0)
    hip.HIPBackend.dropout(None, None, None, None, 10, 0, 0.5, rng, 0)
    hip.HIPBackend.dropoutBackward(None, None, gb, 0, 10, 0.5, rng, 0)
    assert np.all(gb.numpy() == 0)


GOOD = dict(dt=2, x=4096, out=4096, rows=4, cols=8, p=0.5, rng=4096)
BAD = [dict(dt=3), dict(dt=-1), dict(x=None), dict(out=None), dict(rng=None), dict(rng=4100), dict(rows=-1), dict(cols=-1),
       dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(x=4098), dict(dt=0, x=4097), dict(rows=2 ** 30, cols=100), dict(rows=2 ** 31 - 1, cols=1)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_refusals(bad):
    import omnimatchdeeplearningtool_amd as om
    a = {**GOOD, **bad}
    for name, args in (("omHipDropout", (a["x"], None, None, a["out"])), ("omHipDropoutBackward", (a["x"], a["out"], None))):
        with pytest.raises(om.OmHipError, match=name):
            om.call(name, a["dt"], *args, a["rows"], a["cols"], a["p"], a["rng"], 0)


@pytest.mark.gpu
def test_more_columns_than_one_dimension_of_a_grid(hip):
    """One row of 2^27 + 72 columns: the bias gradient's sums take 32 columns a workgroup of 1024 threads, 2^32 threads and
    more. Of one row they are the kept values themselves (a factor of 2 is exact)."""
    cols = 2 ** 27 + 72
    print(f"case 1x{cols}", flush=True)
    x = np.resize(O.randn((100003,), 5, 1.0).astype(np.float16), cols)
    dx, gx, gb = to_dev(hip, x.view(np.uint16)), empty_dev(hip, (cols,), np.uint16), empty_dev(hip, (cols,))
    hip.HIPBackend.dropoutBackward(dx, gx, gb, 1, cols, 0.5, state(hip, 21, 4), 6, 0)
    g = gx.numpy().view(np.float16)
    assert np.all((g == 0) | (g == 2 * x))
    assert np.array_equal(gb.numpy(), g.astype(np.float32))
    for first in (0, 2 ** 24, cols // 8 - 9):   # groups of 8 columns
        for group in range(first, first + 9):
            words = philox([group, 6, 4, 0], [21, 0])
            keep = [((words[j // 2] >> (16 * (j % 2))) & 0xFFFF) >= threshold(0.5) for j in range(8)]
            at = slice(8 * group, 8 * group + 8)
            assert np.array_equal(g[at], np.where(keep, 2 * x[at], 0).astype(np.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1], ids=["fp16", "bf16"])
@pytest.mark.parametrize("cols", [1024, 1021], ids=str)
def test_large_output_in_half_precision(hip, cols, dt):
    """Over 24 MB of 16-bit values, which leave with streaming stores: kept and doubled (exact) or dropped, with the host's
    mask at both ends, forward and backward, with and without a bias gradient."""
    rows = 12401
    print(f"case {rows}x{cols} dtype {dt}", flush=True)
    x = store(O.randn((rows, cols), 6, 1.0), dt)
    v = value(x, dt)
    dx, rng = to_dev(hip, x), state(hip, 12, 34)
    out, gx, alone = (empty_dev(hip, x.shape, x.dtype) for _ in range(3))
    gb = empty_dev(hip, (cols,))
    hip.HIPBackend.dropout(dx, None, None, out, rows, cols, 0.5, rng, 2, dt)
    hip.HIPBackend.dropoutBackward(dx, gx, gb, rows, cols, 0.5, rng, 2, dt)
    hip.HIPBackend.dropoutBackward(dx, alone, None, rows, cols, 0.5, rng, 2, dt)
    y = value(out.numpy(), dt)
    assert np.all((y == 0) | (y == 2 * v))
    assert np.array_equal(gx.numpy(), out.numpy()) and np.array_equal(alone.numpy(), out.numpy())
    assert np.array_equal(y[:20] != 0, mask(20, cols, 0.5, 12, 34, 2) & (v[:20] != 0))
    last, per_row = rows - 1, -(-cols // 8)
    for c in range(per_row):
        words = philox([last * per_row + c, 2, 34, 0], [12, 0])
        keep = np.array([((words[j // 2] >> (16 * (j % 2))) & 0xFFFF) >= threshold(0.5) for j in range(8)])[:cols - 8 * c]
        at = slice(8 * c, 8 * c + 8)
        assert np.array_equal(y[last, at] != 0, keep & (v[last, at] != 0))
    assert np.all(np.abs(gb.numpy() - y.sum(0, dtype=np.float64)) <= 1.01 * (rows + 2) * U * np.abs(y).sum(0, dtype=np.float64))
