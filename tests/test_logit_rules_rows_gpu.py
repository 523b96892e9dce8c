"""More rows of logits than half of 2^31: their results lie behind 2^31 floats."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_pick_of_rows_past_32_bits(pkg):
    S, k = (1 << 30) + 5, 8
    ctx = pkg.CudaContext(0)
    x = ctx.alloc(S, 1)  # (what the other rows hold does not matter)
    want = np.linspace(-1, 1, k, dtype=np.float32)
    ctx.copyRows(x, ctx.upload(want, k, 1), 0)
    ctx.copyRows(x, ctx.upload(want, k, 1), S - k)
    y = ctx.pickAdjusted(x)
    for row in (0, S - k):
        got = ctx.download(ctx.sliceRows(y, row, k)).reshape(k, 2)
        assert np.array_equal(got[:, 0], np.zeros(k)) and np.array_equal(got[:, 1], want)
    ctx.destroy()
