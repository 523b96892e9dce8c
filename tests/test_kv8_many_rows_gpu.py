"""Rows so many that one call takes several launches (width 256, whose rows go 8 at a time)."""
import numpy as np
import pytest

from .test_kv8_gpu import all_stored, attention, cache, f32, got, make, put  # noqa: F401  (cache: a fixture)

pytestmark = pytest.mark.gpu


def test_several_launches_of_one_call(ctx, cache):  # noqa: F811
    """1025 groups of 8 rows over 2^19 positions: more than 2^24 blocks in all.  The positions repeat 1024 of them, so that each row's
    result is the one over 1024."""
    HD, period, n, T = 256, 1024, 1 << 19, 8200
    rng = np.random.default_rng(21)
    k, v, q = make(rng, 1, period, HD), make(rng, 1, period, HD), make(rng, 1, T, HD, 1 / 16)
    c, batch = cache(1, n, 1, HD), 32 * period
    tk, tv = (put(ctx, np.tile(x, (batch // period, 1))) for x in (k, v))
    for a in range(0, n, batch):
        ctx.kvWrite8(c, tk, tv, a)
    V = all_stored(v, 1, 1)
    want, bound = attention(q.reshape(1, T, 1, HD), all_stored(k, 1, 1), V, [[period] * T])
    bound += (n - period) / 32 * 2.0 ** -24 * float(np.abs(V).max())  # sums over n positions
    for lens in (None, put(ctx, [[n]])):
        out = got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n, lens=lens))
        assert np.abs(out - want).max() <= bound
