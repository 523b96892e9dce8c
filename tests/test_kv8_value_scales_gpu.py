"""Attention over the 8-bit cache where the values' scales lie far apart, against float64, row by row: a row's error is bounded by
what the row itself adds up, not by the largest value of the cache.

Bound: as in test_kv8_gpu, relative to A = sum_j p_j B_j, where B_j is the largest |v| of position j's block (a weight is off by its
score's error and 2^-20; a code stands for a part of B_j), and what a weight loses as f16 value and residue, which end 2^-31 below
the largest p_j B_j, for each of the positions that the row sees."""
import numpy as np
import pytest

from .test_kv8_gpu import all_stored, cache, f32, got, make, put  # noqa: F401  (cache: a fixture)

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def rows_and_bounds(q, K, V, limit):
    """One stream: q [T, HQ, HD], K, V [H, N, HD] as stored, limit [T] -> result, bound [T, HQ*HD] in f64"""
    T, HQ, HD = q.shape
    G = HQ // K.shape[0]
    out, bound = np.zeros((T, HQ, HD)), np.zeros((T, HQ, HD))
    for h in range(K.shape[0]):
        k, v = K[h].astype(np.float64), V[h].astype(np.float64)
        B = np.concatenate([np.full(len(v[a:a + 32]), np.abs(v[a:a + 32]).max()) for a in range(0, len(v), 32)])
        for j in range(h * G, (h + 1) * G):
            for i in range(T):
                n, x = limit[i], q[i, j].astype(np.float64)
                z = k[:n] @ x
                p = np.exp(z - z.max())
                p /= p.sum()
                ds = 2 * EPS * np.abs(x).max() * np.abs(k[:n]).sum(1).max() + (HD + 4) * EPS * (np.abs(k[:n]) @ np.abs(x)).max()
                out[i, j] = p @ v[:n]
                bound[i, j] = (2 * ds + 2.0 ** -20 + (n / 32 + 64) * EPS) * (p @ B[:n]) + n * 2.0 ** -31 * (p * B[:n]).max()
    return out.reshape(T, -1), bound.reshape(T, -1)


def held(ctx, cache, k, v, H=1):  # noqa: F811
    c = ctx.kvWrite8(cache(1, len(k), H, k.shape[1] // H), put(ctx, k), put(ctx, v))
    return c, all_stored(k, 1, H)[0], all_stored(v, 1, H)[0]


# rows of a key head for each form: up to 4, up to 8, up to 16, several groups of 16, one row tile and two of a prompt
ROWS = [3, 7, 14, 40, 60, 200]


@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("power", [12, 20, 40, 100])
def test_later_tokens_do_not_change_earlier_rows(ctx, cache, T, HD, power):  # noqa: F811
    """Values from the second half's first block on are 2^power times the others: rows in front of it are those of a prompt without."""
    n, H = 70, 1
    rng = np.random.default_rng(T + HD + power)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD)
    qkv = np.concatenate([make(rng, 1, T, HD, 1 / np.sqrt(HD)), make(rng, 1, T, 2 * HD)], 1)
    border = -(-(n + T // 2) // 32) * 32 - n  # the first new row whose block is in the second half
    outs = []
    for f in (1.0, 2.0 ** power):
        x = qkv.copy()
        x[border:, 2 * HD:] *= f32(f)
        c = cache(1, n + T, H, HD)
        ctx.kvWrite8(c, put(ctx, k), put(ctx, v))
        out = got(ctx, ctx.attnAppendKv8(put(ctx, x), c, 1, n))
        K, V = all_stored(np.concatenate([k, x[:, HD:2 * HD]]), 1, H)[0], all_stored(np.concatenate([v, x[:, 2 * HD:]]), 1, H)[0]
        want, bound = rows_and_bounds(x[:, :HD].reshape(T, 1, HD), K, V, [n + i + 1 for i in range(T)])
        assert (np.abs(out - want) <= bound).all()
        outs.append(out[:border])
    assert np.array_equal(*outs)


@pytest.mark.parametrize("HD,G", [(64, 1), (128, 2), (20, 1)])
@pytest.mark.parametrize("T", ROWS)
def test_a_block_without_weight_takes_nothing_from_the_others(ctx, cache, T, HD, G):  # noqa: F811
    """One block's values are 2^60 times the others', its scores 130 below them (weights of 2^-187); and the other way about."""
    n = 300
    rng = np.random.default_rng(T * HD)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD)
    q = make(rng, 1, T, G * HD, 0.1 / np.sqrt(HD))
    k[:, 0], q.reshape(T, G, HD)[:, :, 0] = 0, 8
    k[64:96], k[64:96, 0] = 0, -16.25
    for f in (2.0 ** 60, 2.0 ** -60):
        w = v.copy()
        w[64:96] *= f32(f)
        c, K, V = held(ctx, cache, k, w)
        want, bound = rows_and_bounds(q.reshape(T, G, HD), K, V, [n] * T)
        assert (np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, G, n)) - want) <= bound).all()


@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("step", [-7, 5])
def test_scales_that_fall_or_rise_from_block_to_block(ctx, cache, T, step):  # noqa: F811
    """Scores rise from block to block as well, so that weights and scales go against each other, or together; some blocks are zeros."""
    n, HD = 500, 64
    rng = np.random.default_rng(10 * T + step + 7)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD)
    block = np.arange(n) // 32
    k[:, 0] = block * f32(0.5)
    v *= np.exp2(step * block)[:, None].astype(f32)
    v[(block == 3) | (block == 11)] = 0
    q = make(rng, 1, T, HD, 0.3 / np.sqrt(HD))
    q[:, 0] = np.linspace(-12, 12, T)
    c, K, V = held(ctx, cache, k, v)
    want, bound = rows_and_bounds(q.reshape(T, 1, HD), K, V, [n] * T)
    assert (np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n)) - want) <= bound).all()


@pytest.mark.parametrize("T", [1, 14, 60])
@pytest.mark.parametrize("power", [-90, 90])
def test_values_of_any_size(ctx, cache, T, power):  # noqa: F811
    """All values tiny or huge, over tiles enough to be split among thread blocks (one stream, one head)."""
    n, HD = 2100, 64
    rng = np.random.default_rng(power + 90 + T)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD) * f32(2.0 ** power)
    q = make(rng, 1, T, HD, 1 / 8)
    c, K, V = held(ctx, cache, k, v)
    want, bound = rows_and_bounds(q.reshape(T, 1, HD), K, V, [n] * T)
    assert (np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n)) - want) <= bound).all()
    zero, _, _ = held(ctx, cache, k, np.zeros_like(v))
    assert not got(ctx, ctx.attnKv8(put(ctx, q), zero, 1, n)).any()


@pytest.mark.parametrize("T,size", [(t, x) for t in ROWS for x in (30.0, 1e4, 1e5, 1e7, 3e9, 1e20) if t < 49 or x < 1e6])
def test_scores_of_any_size(ctx, cache, T, size):  # noqa: F811
    """Two positions of a row share the largest score, in blocks whose values lie 2^30 apart, all others are as far below zero.
    Keys are +-1 in the first channel, the only one that queries have, so that equal scores are equal in every form.  From 49 rows on the
    exponent of a weight is the score less a reference plus the logarithm of the block's scale, an f32 of the score's size: half a step
    of it, 2^-24 (score + |log scale| + log 2^6), is what each of the two weights may be off by; |log scale| is below 30 here."""
    n, HD = 420, 64
    rng = np.random.default_rng(T)
    k, v = rng.uniform(-1, 1, (n, HD)).astype(f32), make(rng, 1, n, HD)
    k[:, 0] = -1
    k[[40, 333], 0] = 1
    v[320:352] *= f32(2.0 ** 30)
    q = np.zeros((T, HD), f32)
    q[:, 0] = size * (1 + np.arange(T) / 7)
    c, K, V = held(ctx, cache, k, v)
    for order in (1, -1):  # the small values' block first, and last
        if order < 0:
            k, v = k[::-1].copy(), v[::-1].copy()
            v *= f32(2.0 ** -20)
            c, K, V = held(ctx, cache, k, v)
        a, b = np.flatnonzero(k[:, 0] > 0)
        assert K[0, a, 0] == K[0, b, 0] and (K[0][k[:, 0] < 0, 0] == -K[0, a, 0]).all()
        V64 = V[0].astype(np.float64)
        want = (V64[a] + V64[b]) / 2
        B = [np.abs(V64[i // 32 * 32:i // 32 * 32 + 32]).max() for i in (a, b)]
        rest = n * np.exp(-2 * size) * np.abs(V64).max()
        step = 2 * EPS * (np.abs(q[:, :1]).astype(np.float64) + 35) if T > 48 else 0.0
        out = got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n))
        assert (np.abs(out - want) <= (2.0 ** -20 + (n / 32 + 64) * EPS + step) * (B[0] + B[1]) / 2 + n * 2.0 ** -31 * max(B) + rest).all()
        # b is not seen: the first alone
        out = got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n, lens=put(ctx, [[b]])))
        assert (np.abs(out - V64[a]) <= (2.0 ** -20 + (n / 32 + 64) * EPS + step + n * 2.0 ** -31) * B[0] + rest).all()
