"""The window's kernel for few queries (a sequence's next tokens): what test_gpu_attn_window does not reach of it, against the
formulas in float64, element by element (attn_views says how far off a result may be)."""
import numpy as np
import pytest

from test_gpu_attn_train import bits, value
from test_gpu_attn_window import Window


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
