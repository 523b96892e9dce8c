"""Many rows to a key head over the 8-bit cache (prompts, wide groups of query heads), against float64; bounds as for single tokens,
with what the weights lose beside the largest scale of a range's values: 2^-25 of 2^6 for each of N positions."""
import numpy as np
import pytest

from .test_kv8_gpu import all_stored, attention, cache, f32, got, heads, make, put, rows, stored  # noqa: F401  (cache: a fixture)

pytestmark = pytest.mark.gpu


def bound_of(bound, V, n):
    return bound + n * 2.0 ** -31 * float(np.abs(V).max())


# streams, query heads, heads, width, queries, positions: each stored width and widths between, one row tile and several, ragged
# last ones, positions that end in the first block of a tile, tiles enough to be split over thread blocks
SHAPES = [(1, 1, 1, 64, 49, 1), (1, 1, 1, 64, 128, 128), (2, 3, 3, 32, 129, 129), (1, 14, 2, 64, 9, 300), (2, 2, 2, 96, 200, 97), (1, 5, 5, 80, 64, 260),
          (1, 4, 1, 128, 33, 140), (3, 1, 1, 13, 60, 61), (1, 2, 1, 64, 40, 4100), (1, 8, 1, 128, 20, 3000), (1, 64, 1, 64, 1, 700), (2, 1, 1, 1, 50, 40),
          (2, 2, 2, 33, 55, 1030), (1, 3, 3, 256, 70, 100)]


@pytest.mark.parametrize("S,HQ,H,HD,T,n", SHAPES)
def test_complete_cache(ctx, cache, S, HQ, H, HD, T, n):  # noqa: F811
    rng = np.random.default_rng(HD * 7 + n)
    k, v = make(rng, S, n, H * HD), make(rng, S, n, H * HD)
    q = make(rng, S, T, HQ * HD, 1 / np.sqrt(HD))
    c = ctx.kvWrite8(cache(S, n + 5, H, HD), put(ctx, k), put(ctx, v))
    K, V = all_stored(k, S, H), all_stored(v, S, H)
    for lens in (None, rng.integers(0, n + 1, S)):
        if lens is not None:
            lens[S - 1] = 0
        want, bound = attention(q.reshape(S, T, HQ, HD), K, V, [[n if lens is None else int(lens[s])] * T for s in range(S)])
        out = got(ctx, ctx.attnKv8(put(ctx, q), c, HQ, n, lens=None if lens is None else put(ctx, [lens])))
        assert np.abs(out - want).max() <= bound_of(bound, V, n)
        if lens is not None:
            assert not out[(S - 1) * T:].any()


@pytest.mark.parametrize("S,HQ,H,HD,T,n", [(2, 2, 2, 64, 100, 0), (1, 6, 2, 64, 50, 37), (1, 2, 2, 128, 150, 640), (2, 1, 1, 32, 300, 5), (1, 1, 1, 96, 65, 2500)])
def test_append(ctx, cache, S, HQ, H, HD, T, n):  # noqa: F811
    rng = np.random.default_rng(HD + T + n)
    D, E = HQ * HD, H * HD
    k, v = make(rng, S, n, E), make(rng, S, n, E)
    qkv = np.concatenate([make(rng, S, T, D, 1 / np.sqrt(HD)), make(rng, S, T, 2 * E)], 1)
    c = cache(S, n + T, H, HD)
    if n:
        ctx.kvWrite8(c, put(ctx, k), put(ctx, v))
    K, V = (all_stored(rows(np.concatenate([heads(a, S, H) if n else np.zeros((S, H, 0, HD), f32), heads(b, S, H)], 2)), S, H)
            for a, b in ((k, qkv[:, D:D + E]), (v, qkv[:, D + E:])))
    want, bound = attention(qkv[:, :D].reshape(S, T, HQ, HD), K, V, [[n + i + 1 for i in range(T)]] * S)
    assert np.abs(got(ctx, ctx.attnAppendKv8(put(ctx, qkv), c, HQ, n)) - want).max() <= bound_of(bound, V, n + T)
    rk, rv = ctx.kvRead8(c, 0, n + T)
    assert np.array_equal(got(ctx, rk), rows(K)) and np.array_equal(got(ctx, rv), rows(V))


def test_append_of_prompts_of_different_lengths(ctx, cache):  # noqa: F811
    S, HQ, H, HD, T = 4, 2, 2, 64, 60
    rng = np.random.default_rng(8)
    D, E, pos, counts = HQ * HD, H * HD, [0, 30, 130, 61], [60, 55, 0, 1]
    k, v = make(rng, S, 140, E), make(rng, S, 140, E)
    qkv = np.concatenate([make(rng, S, T, D, 1 / 8), make(rng, S, T, 2 * E)], 1)
    c = cache(S, 200, H, HD)
    ctx.kvWrite8(c, put(ctx, k), put(ctx, v), counts=put(ctx, [pos]))
    out = got(ctx, ctx.attnAppendKv8(put(ctx, qkv), c, HQ, pos=put(ctx, [pos]), counts=put(ctx, [counts])))
    new, old = [heads(qkv[:, a:a + E], S, H) for a in (D, D + E)], [heads(x, S, H) for x in (k, v)]
    for s in range(S):
        K, V = (np.stack([stored(np.concatenate([o[s, h, :pos[s]], w[s, h, :counts[s]]])) for h in range(H)])[None] for o, w in zip(old, new))
        want, bound = attention(qkv[s * T:(s + 1) * T, :D].reshape(1, T, HQ, HD), K, V, [[pos[s] + i + 1 if i < counts[s] else 0 for i in range(T)]])
        assert np.abs(out[s * T:(s + 1) * T] - want).max() <= bound_of(bound, V, 200)
        assert not out[s * T + counts[s]:(s + 1) * T].any()


@pytest.mark.parametrize("HD", [64, 128])
def test_maxima_that_move_far_and_scales_far_apart(ctx, cache, HD):  # noqa: F811
    """Scores that rise by hundreds from tile to tile (the running result is rescaled each time), blocks of zeros, of keys and of
    values 2^20 below the others."""
    n, T = 700, 64
    rng = np.random.default_rng(6)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD)
    k *= (np.arange(n)[:, None] / 100).astype(f32)
    k[96:128], v[160:192] = 0, 0
    v[256:288] *= f32(2.0 ** -20)
    k[320:352] *= f32(2.0 ** -20)
    q = make(rng, 1, T, HD, 1.0)
    q[5] = 0
    c = ctx.kvWrite8(cache(1, n, 1, HD), put(ctx, k), put(ctx, v))
    K, V = all_stored(k, 1, 1), all_stored(v, 1, 1)
    want, bound = attention(q.reshape(1, T, 1, HD), K, V, [[n] * T])
    assert np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n)) - want).max() <= bound_of(bound, V, n)


def test_what_is_not_finite_stays_where_it_is_seen(ctx, cache):  # noqa: F811
    """A NaN block makes NaN of the rows that see it and of no other; a query row that is not finite is its own alone."""
    H, HD, T = 1, 64, 100
    rng = np.random.default_rng(5)
    qkv = np.concatenate([make(rng, 1, T, HD, 1 / 8), make(rng, 1, T, 2 * HD)], 1)
    qkv[70, HD + 3], qkv[90, 2 * HD + 1] = np.nan, np.inf  # keys of block 2, values of block 2
    qkv[10, 5] = np.inf
    out = got(ctx, ctx.attnAppendKv8(put(ctx, qkv), cache(1, T, H, HD), 1, 0))
    assert np.isnan(out[64:]).all() and np.isnan(out[10]).all()
    assert np.isfinite(np.delete(out[:64], 10, 0)).all()
    clean = np.nan_to_num(qkv, posinf=0.0)
    want, bound = attention(clean[:, :HD].reshape(1, T, 1, HD), all_stored(clean[:, HD:2 * HD], 1, 1), all_stored(clean[:, 2 * HD:], 1, 1),
                            [[i + 1 for i in range(T)]])
    assert np.abs(np.delete(out[:64] - want[:64], 10, 0)).max() <= bound


def test_long_sums_of_one_sign(ctx, cache):  # noqa: F811
    """8000 positions of positive values under equal weights: a sum that loses a little at every step would show."""
    S, n, T, HD = 40, 8000, 50, 64  # thread blocks enough that positions are not split
    rng = np.random.default_rng(4)
    v = (1 + rng.random((n, HD))).astype(f32)
    c = cache(S, n, 2, HD)
    t = put(ctx, np.tile(np.concatenate([v, v], 1), (S, 1)))
    ctx.kvWrite8(c, t, t)
    out = got(ctx, ctx.attnKv8(ctx.upload(np.zeros((S * T, 2 * HD), f32), S * T, 2 * HD), c, 2, n))
    want = stored(v).astype(np.float64).mean(0)
    assert np.abs(out - np.tile(want, 2)).max() < 4e-6 * want.max()  # (63 tiles x 2^-24 x half, the products' own 8 steps)


def test_recorded_prompt_and_product(ctx, cache):  # noqa: F811
    S, H, HD, T = 2, 4, 64, 60
    rng = np.random.default_rng(9)
    D = H * HD
    x = put(ctx, np.concatenate([make(rng, S, T, D, 1 / 8), make(rng, S, T, 2 * D)], 1))
    w = put(ctx, make(rng, 1, D, 256, 1 / 16), True)
    c = cache(S, 200, H, HD)
    run = lambda: ctx.matmul(ctx.attnAppendKv8(x, c, H, 64), w)  # noqa: E731
    first = got(ctx, run())
    batch, y = ctx.recordBatch(run)
    for _ in range(3):
        batch.launch()
        assert np.array_equal(got(ctx, y), first)
    batch.free()
    out = ctx.attnAppendKv8(x, c, H, 64)
    assert np.array_equal(got(ctx, ctx.matmul(put(ctx, got(ctx, out)), w)), first)
