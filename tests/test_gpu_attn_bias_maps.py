"""Sums of a bias table's gradient: held in doubles wherever they fit a CU's LDS."""
import numpy as np
import pytest

from test_gpu_attn_bias import Bias
from test_gpu_attn_train import U, bits


def whole(hip, S, D, offsets, H=2):
    """All queries in one place, key j at an offset of its own, scores 0 and values +-1 that add up to 0: dS_qj is P (1 / S) times
    +-dO_q, exact but for P, and an offset's sum is over the queries. A wave's are small, 2^30 times as large, small, minus that,
    small: their sum is three small ones."""
    c = Bias(hip, 1, S, S, H, H, D, bf16=True, scale=0.0, table_std=0.0, seed=4, buckets=np.arange(offsets), zero=offsets - 1,
             where=(np.zeros(S), np.arange(S) * (offsets // S)))
    sign = np.where(np.arange(S) % 2 == 0, 1.0, -1.0)
    v = np.zeros_like(c.store[2])
    v.reshape(1, S, H, D)[..., 0] = sign[:, None]
    g = np.zeros_like(c.grad)
    small, large = 2.0 ** -10, 2.0 ** 20
    g[0, :5, :, 0] = np.array([small, large, small, -large, small])[:, None]
    c.dev[2].upload(bits(v, True))
    c.dgrad.upload(bits(g, True))
    c.forward()
    c.backward()
    return c.dgtable.numpy()[offsets - 1 - np.arange(S) * (offsets // S)], 3 * small / S * sign


@pytest.mark.gpu
@pytest.mark.parametrize("S,D,offsets", [(70, 32, 2560), (70, 32, 3697), (70, 64, 2811), (70, 64, 3015), (70, 96, 2560), (70, 128, 2560),
                                         (64, 32, 4096), (64, 64, 4096)], ids=str)
def test_small_sums_beside_large_ones_that_cancel(hip, S, D, offsets):
    """A grid of 27 x 27 patches has 53^2 + 2 = 2811 offsets. P is off by (4 log S + 8) u, and three roundings follow to fp32: of the
    waves' sums, of the workgroups' and of the result."""
    print(f"{S} tokens of {D}, {offsets} offsets", flush=True)
    got, want = whole(hip, S, D, offsets)
    lim = 1.01 * (4 * np.log(S) + 8 + 3) * U * np.abs(want)
    assert np.all(np.abs(got - want[:, None]) <= lim[:, None]), (got[:3], want[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D,offsets", [(32, 3697), (32, 3698), (64, 3015), (64, 3016), (128, 2560), (128, 2561)], ids=str)
def test_maps_around_the_sums_in_doubles_by_head_dimension(hip, D, offsets, bf16):
    """The longest map whose sums are doubles, with four waves, and the next one."""
    at = np.arange(150) * 19
    c = Bias(hip, 2, 150, 150, 2, 1, D, seed=9, bf16=bf16, buckets=np.arange(offsets) // 2, zero=offsets // 2, where=(at, at))
    c.forward()
    c.backward()
    c.check()
