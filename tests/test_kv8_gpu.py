"""The 8-bit key and value cache and the attention over it, against the definition in float64.

What is stored is compared exactly: scale = f32(max|x| / 127), code = round-half-even(x / scale), value = f32(code * scale).

Bound of an attention output: a query is split into f16 value and residue, off by at most 2^-23 of its row's largest element
(half a step of the residue: 2^-11 * 2^-11 / 2); products are exact, a score is a sum of HD of them in f32 (HD half steps of
sum|q k|) and two more roundings; a weight is off by twice the largest score error (its own and the maximum's) and a few
steps of exp, the weight's split and the rescaling (2^-20 together); sums over N positions run 32 to a chain and over the
chains' results: (N / 32 + 64) half steps.  All of it relative to the largest |v|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32


def stored(x):
    """[T, HD] rows of one head -> the values that the cache holds."""
    out = np.zeros(x.shape, f32)
    for a in range(0, x.shape[0], 32):
        b = x[a:a + 32].astype(np.float64)
        scale = f32(np.abs(b).max() / 127)
        if not np.isfinite(scale):
            out[a:a + 32] = np.nan
        elif scale > 0:
            out[a:a + 32] = np.clip(np.rint(b / np.float64(scale)), -127, 127).astype(f32) * scale
    return out


def heads(x, S, H):
    """[S*T, H*HD] -> [S, H, T, HD]"""
    return x.reshape(S, x.shape[0] // S, H, -1).transpose(0, 2, 1, 3)


def rows(x):
    S, H, T, HD = x.shape
    return x.transpose(0, 2, 1, 3).reshape(S * T, H * HD)


def all_stored(x, S, H, counts=None):
    x = heads(x, S, H)
    out = np.zeros_like(x)
    for s in range(S):
        n = x.shape[2] if counts is None else counts[s]
        for h in range(H):
            out[s, h, :n] = stored(x[s, h, :n])
    return out


def attention(q, K, V, limit):
    """q [S, T, HQ, HD], K, V [S, H, N, HD], limit [S][T] -> (result [S*T, HQ*HD] f64, bound)"""
    S, T, HQ, HD = q.shape
    G, N = HQ // K.shape[1], K.shape[2]
    out, worst = np.zeros((S, T, HQ, HD)), 0.0
    eps = 2.0 ** -24
    for s in range(S):
        for j in range(HQ):
            k, v = K[s, j // G].astype(np.float64), V[s, j // G].astype(np.float64)
            for i in range(T):
                n = limit[s][i]
                if n <= 0:
                    continue
                x = q[s, i, j].astype(np.float64)
                z = k[:n] @ x
                p = np.exp(z - z.max())
                out[s, i, j] = (p @ v[:n]) / p.sum()
                ds = 2 * eps * np.abs(x).max() * np.abs(k[:n]).sum(1).max() + (HD + 4) * eps * (np.abs(k[:n]) @ np.abs(x)).max()
                worst = max(worst, 2 * ds + 2.0 ** -20 + (N / 32 + 64) * eps)
    return out.reshape(S * T, HQ * HD), worst * max(1e-30, float(np.abs(V).max()) if V.size else 0.0)


def make(rng, S, T, cols, scale=1.0):
    x = rng.standard_normal((S * T, cols)) * np.exp(0.7 * rng.standard_normal((1, cols))) * scale
    return x.astype(f32)


def put(ctx, x, f16=False):
    x = np.ascontiguousarray(x, dtype=f32)
    return (ctx.uploadF16 if f16 else ctx.upload)(x, *x.shape)


def got(ctx, t):
    return ctx.download(t).reshape(t.rows, t.cols)


@pytest.fixture
def cache(ctx):
    made = []

    def make_cache(*a):
        made.append(ctx.kvCache8(*a))
        return made[-1]

    yield make_cache
    for c in made:
        ctx.freeKvCache8(c)


# streams, rows, heads, width: single rows, edges of a block, widths that no kernel is built for, one and many heads
WRITES = [(1, 1, 1, 1), (2, 31, 3, 13), (1, 32, 2, 64), (3, 33, 2, 64), (2, 100, 5, 32), (1, 129, 1, 80), (2, 70, 2, 128), (2, 65, 1, 256), (1, 40, 2, 200)]


@pytest.mark.parametrize("S,T,H,HD", WRITES)
@pytest.mark.parametrize("f16", [False, True])
def test_write_stores_the_definition(ctx, cache, S, T, H, HD, f16):
    rng = np.random.default_rng(T * HD)
    k, v = make(rng, S, T, H * HD), make(rng, S, T, H * HD, 40.0)
    if f16:
        k, v = k.astype(np.float16).astype(f32), v.astype(np.float16).astype(f32)
    c = ctx.kvWrite8(cache(S, T + 3, H, HD), put(ctx, k, f16), put(ctx, v, f16))
    rk, rv = ctx.kvRead8(c, 0, T)
    assert np.array_equal(got(ctx, rk), rows(all_stored(k, S, H)))
    assert np.array_equal(got(ctx, rv), rows(all_stored(v, S, H)))
    a, n = T // 3, T - T // 3 + 2  # a range that begins inside a block and runs past what was written
    rk, _ = ctx.kvRead8(c, a, n)
    want = np.concatenate([all_stored(k, S, H), np.zeros((S, H, 3, HD), f32)], 2)[:, :, a:a + n]
    assert np.array_equal(got(ctx, rk), rows(want))


def test_codes_at_ties_and_of_small_and_large_values(ctx, cache):
    """Half steps go to the even code; zeros, subnormal and huge blocks; a block with an infinity or a NaN reads as NaN."""
    T, H, HD = 32, 7, 64
    rng = np.random.default_rng(1)
    x = np.zeros((1, H, T, HD), f32)
    x[0, 0] = rng.integers(-254, 255, (T, HD)) * f32(0.5)  # scale 1: every other value is a tie
    x[0, 0, 0, 0] = 127
    x[0, 1] = x[0, 0] * f32(2.0 ** -20)
    x[0, 2] = rng.standard_normal((T, HD)).astype(f32) * f32(1e-42)  # subnormal, as the scale is
    x[0, 3] = rng.standard_normal((T, HD)).astype(f32) * f32(5e37)
    x[0, 4] = rng.standard_normal((T, HD))
    x[0, 4, 5, 6] = np.inf
    x[0, 5] = rng.standard_normal((T, HD))
    x[0, 5, 31, 63] = np.nan
    c = cache(1, T, H, HD)
    ctx.kvWrite8(c, put(ctx, rows(x)), put(ctx, rows(x[:, ::-1])))
    rk, rv = ctx.kvRead8(c, 0, T)
    with np.errstate(invalid="ignore"):
        want = np.stack([stored(x[0, h]) for h in range(H)])[None]
    assert np.array_equal(got(ctx, rk), rows(want), equal_nan=True)
    assert np.array_equal(got(ctx, rv), rows(want[:, ::-1]), equal_nan=True)
    # a query over the blocks: NaN where the head's block is NaN, finite elsewhere
    out = got(ctx, ctx.attnKv8(put(ctx, np.ones((1, 2 * HD)) * 0.01), cache_of(ctx, c, x[:, 4:6], cache), 2, T))
    assert np.isnan(out).all()


def cache_of(ctx, like, x, cache):
    c = cache(x.shape[0], x.shape[2], x.shape[1], x.shape[3])
    t = put(ctx, rows(x))
    return ctx.kvWrite8(c, t, t)


@pytest.mark.parametrize("steps", [[1] * 70, [5, 1, 26, 32, 1, 64, 3], [33, 31, 40], [100, 1, 1]])
@pytest.mark.parametrize("H,HD", [(3, 64), (1, 20)])
def test_rows_that_join_a_block_code_it_anew(ctx, cache, steps, H, HD):
    S, total = 2, sum(steps)
    rng = np.random.default_rng(total)
    k, v = (heads(make(rng, S, total, H * HD), S, H) for _ in range(2))
    c, n = cache(S, total, H, HD), 0
    for T in steps:
        ctx.kvWrite8(c, put(ctx, rows(k[:, :, n:n + T])), put(ctx, rows(v[:, :, n:n + T])), n)
        n += T
        if T == 1 and n % 7 and n != total:
            continue
        rk, rv = ctx.kvRead8(c, 0, n)
        assert np.array_equal(got(ctx, rk), rows(all_stored(rows(k[:, :, :n]), S, H)))
        assert np.array_equal(got(ctx, rv), rows(all_stored(rows(v[:, :, :n]), S, H)))


def test_going_back_to_an_earlier_block(ctx, cache):
    """Rows in front of the new one in a block that is not the last written one are taken at their stored values."""
    rng = np.random.default_rng(3)
    x, y = make(rng, 1, 80, 64), make(rng, 1, 1, 64, 9.0)
    c = cache(1, 96, 1, 64)
    ctx.kvWrite8(c, put(ctx, x), put(ctx, x))
    ctx.kvWrite8(c, put(ctx, y), put(ctx, y), 70)  # inside the last block: from the f32 rows
    want = np.concatenate([x[:70], y])
    assert np.array_equal(got(ctx, ctx.kvRead8(c, 64, 7)[0]), stored(want[64:]))
    ctx.kvWrite8(c, put(ctx, y), put(ctx, y), 10)
    want = stored(np.concatenate([stored(x[:32])[:10], y]))
    assert np.array_equal(got(ctx, ctx.kvRead8(c, 0, 11)[0]), want)
    assert np.array_equal(got(ctx, ctx.kvRead8(c, 32, 32)[1]), stored(x[32:64]))  # other blocks stay
    ctx.kvWrite8(c, put(ctx, x[:5]), put(ctx, x[:5]), 0)  # from the start again
    assert np.array_equal(got(ctx, ctx.kvRead8(c, 0, 5)[0]), stored(x[:5]))


@pytest.mark.parametrize("HD", [64, 30])
def test_places_that_nothing_wrote_are_zeros(ctx, cache, HD):
    """Rows behind a gap, in a new block, in a block of which the f32 rows are held, and behind a shorter rewrite."""
    rng = np.random.default_rng(8)
    x, z = make(rng, 1, 80, HD), np.zeros((6, HD), f32)
    c = cache(1, 128, 1, HD)
    write = lambda a, b: ctx.kvWrite8(c, put(ctx, x[a:b]), put(ctx, x[a:b]), a)  # noqa: E731
    write(0, 32)  # the f32 rows of a full block are held
    write(32, 34)
    write(40, 41)  # 34..39 are nobody's, and not rows 2..7 of the block before
    for t in ctx.kvRead8(c, 32, 9):
        assert np.array_equal(got(ctx, t), stored(np.concatenate([x[32:34], z, x[40:41]])))
    write(34, 35)  # ends the block behind it
    write(36, 37)
    for t in ctx.kvRead8(c, 32, 9):
        assert np.array_equal(got(ctx, t), stored(np.concatenate([x[32:35], z[:1], x[36:37], z[:4]])))
    write(69, 72)  # a block without its first rows
    for t in ctx.kvRead8(c, 64, 8):
        assert np.array_equal(got(ctx, t), stored(np.concatenate([z[:5], x[69:72]])))
    assert np.array_equal(got(ctx, ctx.kvRead8(c, 0, 32)[0]), stored(x[:32]))


def test_streams_at_positions_of_their_own(ctx, cache):
    S, H, HD, T = 5, 2, 64, 40
    rng = np.random.default_rng(4)
    first = [0, 1, 31, 32, 50]
    k, v, k2, v2 = (make(rng, S, n, H * HD) for n in (64, 64, T, T))
    c = cache(S, 128, H, HD)
    ctx.kvWrite8(c, put(ctx, k), put(ctx, v), counts=put(ctx, [first]))
    counts = [T, 3, 33, 0, 1]
    ctx.kvWrite8(c, put(ctx, k2), put(ctx, v2), pos=put(ctx, [first]), counts=put(ctx, [counts]))
    rk, rv = (heads(got(ctx, t), S, H) for t in ctx.kvRead8(c, 0, 128))
    for r, a, b in ((rk, k, k2), (rv, v, v2)):
        a, b = heads(a, S, H), heads(b, S, H)
        for s in range(S):
            x = np.concatenate([a[s, :, :first[s]], b[s, :, :counts[s]]], 1)
            for h in range(H):
                assert np.array_equal(r[s, h, :x.shape[1]], stored(x[h]))
                behind = -(-x.shape[1] // 32) * 32  # rows behind the last block are left as they were
                assert not r[s, h, behind:].any()


# streams, query heads, heads, width, queries, positions in use
ATTEND = [(1, 1, 1, 64, 1, 1), (1, 20, 20, 64, 1, 1500), (3, 5, 5, 32, 1, 33), (2, 8, 1, 64, 1, 31), (2, 6, 2, 80, 3, 77), (1, 9, 1, 128, 1, 257),
          (2, 4, 4, 96, 9, 64), (1, 28, 4, 128, 5, 300), (2, 3, 3, 13, 17, 50), (1, 16, 2, 256, 2, 129), (70, 2, 2, 64, 1, 96), (2, 2, 2, 64, 130, 200),
          (1, 4, 2, 64, 1, 5000), (1, 1, 1, 1, 1, 3), (1, 33, 1, 33, 1, 65)]


@pytest.mark.parametrize("S,HQ,H,HD,T,n", ATTEND)
def test_attention_over_a_complete_cache(ctx, cache, S, HQ, H, HD, T, n):
    rng = np.random.default_rng(HD * 100 + n)
    k, v = make(rng, S, n, H * HD), make(rng, S, n, H * HD)
    q = make(rng, S, T, HQ * HD, 1 / np.sqrt(HD))
    c = ctx.kvWrite8(cache(S, n + 40, H, HD), put(ctx, k), put(ctx, v))
    want, bound = attention(q.reshape(S, T, HQ, HD), all_stored(k, S, H), all_stored(v, S, H), [[n] * T] * S)
    for _ in range(2):  # the second launch finds the tickets as the first left them
        out = ctx.attnKv8(put(ctx, q), c, HQ, n)
        assert np.abs(got(ctx, out) - want).max() <= bound
    lens = rng.integers(0, n + 1, S)
    lens[-1] = 0
    want, bound = attention(q.reshape(S, T, HQ, HD), all_stored(k, S, H), all_stored(v, S, H), [[int(m)] * T for m in lens])
    out = got(ctx, ctx.attnKv8(put(ctx, q), c, HQ, n, lens=put(ctx, [lens])))
    assert np.abs(out - want).max() <= bound
    assert not out[(S - 1) * T:].any()  # a stream of length 0 gives zeros


@pytest.mark.parametrize("S,HQ,H,HD,T,n", [(1, 20, 20, 64, 1, 0), (3, 20, 20, 64, 1, 31), (2, 4, 2, 64, 1, 32), (2, 6, 2, 32, 5, 30), (1, 7, 1, 128, 70, 0),
                                           (2, 2, 2, 64, 224, 0), (2, 3, 3, 40, 33, 64), (1, 8, 4, 256, 3, 95), (64, 20, 20, 64, 1, 15)])
def test_append_and_causal_attention(ctx, cache, S, HQ, H, HD, T, n):
    rng = np.random.default_rng(HD + T + n)
    D, E = HQ * HD, H * HD
    k, v = make(rng, S, n, E), make(rng, S, n, E)
    qkv = np.concatenate([make(rng, S, T, D, 1 / np.sqrt(HD)), make(rng, S, T, 2 * E)], 1)
    c = cache(S, n + T, H, HD)
    if n:
        ctx.kvWrite8(c, put(ctx, k), put(ctx, v))
    K, V = (rows(np.concatenate([heads(a, S, H) if n else np.zeros((S, H, 0, HD), f32), heads(b, S, H)], 2))
            for a, b in ((k, qkv[:, D:D + E]), (v, qkv[:, D + E:])))
    K, V = all_stored(K, S, H), all_stored(V, S, H)
    want, bound = attention(qkv[:, :D].reshape(S, T, HQ, HD), K, V, [[n + i + 1 for i in range(T)]] * S)
    out = ctx.attnAppendKv8(put(ctx, qkv), c, HQ, n)
    assert np.abs(got(ctx, out) - want).max() <= bound
    rk, rv = ctx.kvRead8(c, 0, n + T)
    assert np.array_equal(got(ctx, rk), rows(K)) and np.array_equal(got(ctx, rv), rows(V))


def test_append_at_positions_of_their_own(ctx, cache):
    S, HQ, H, HD, T = 4, 4, 2, 64, 6
    rng = np.random.default_rng(8)
    D, E, pos, counts = HQ * HD, H * HD, [0, 30, 32, 61], [6, 5, 0, 1]
    k, v = make(rng, S, 64, E), make(rng, S, 64, E)
    qkv = np.concatenate([make(rng, S, T, D, 1 / 8), make(rng, S, T, 2 * E)], 1)
    c = cache(S, 70, H, HD)
    ctx.kvWrite8(c, put(ctx, k), put(ctx, v), counts=put(ctx, [pos]))
    out = got(ctx, ctx.attnAppendKv8(put(ctx, qkv), c, HQ, pos=put(ctx, [pos]), counts=put(ctx, [counts])))
    new = [heads(qkv[:, a:a + E], S, H) for a in (D, D + E)]
    old = [heads(x, S, H) for x in (k, v)]
    for s in range(S):
        K, V = (np.stack([stored(np.concatenate([o[s, h, :pos[s]], w[s, h, :counts[s]]])) for h in range(H)])[None] for o, w in zip(old, new))
        limit = [[pos[s] + i + 1 if i < counts[s] else 0 for i in range(T)]]
        want, bound = attention(qkv[s * T:(s + 1) * T, :D].reshape(1, T, HQ, HD), K, V, limit)
        assert np.abs(out[s * T:(s + 1) * T] - want).max() <= bound
        assert not out[s * T + counts[s]:(s + 1) * T].any()


def test_a_large_value_in_a_masked_place_does_not_show(ctx, cache):
    """Infinities and NaN behind a stream's length, in later blocks and in rows that do not count."""
    S, H, HD, n = 2, 1, 64, 100
    rng = np.random.default_rng(5)
    k, v = make(rng, S, n, HD), make(rng, S, n, HD)
    k[64:100], v[164:] = np.nan, np.inf  # stream 0 from position 64 on, stream 1 from position 64 on
    q = make(rng, S, 1, HD, 1 / 8)
    c = ctx.kvWrite8(cache(S, n, H, HD), put(ctx, k), put(ctx, v))
    out = got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n, lens=put(ctx, [[64, 64]])))
    want, bound = attention(q.reshape(S, 1, 1, HD), all_stored(np.nan_to_num(k, posinf=0), S, H)[:, :, :64], all_stored(np.nan_to_num(v, posinf=0), S, H)[:, :, :64], [[64]] * S)
    assert np.abs(out - want).max() <= bound
    c2 = ctx.kvWrite8(cache(S, n, H, HD), put(ctx, k), put(ctx, v), counts=put(ctx, [[50, 64]]))
    out = got(ctx, ctx.attnKv8(put(ctx, q), c2, 1, n, lens=put(ctx, [[50, 64]])))
    assert np.isfinite(out).all()


@pytest.mark.parametrize("T", [1, 12])
def test_scores_far_apart(ctx, cache, T):
    """Scores of +-80 and blocks whose values differ by 2^40: the largest weight of a block is 1 whatever the others hold."""
    n, HD = 160, 64
    rng = np.random.default_rng(6)
    k, v = make(rng, 1, n, HD), make(rng, 1, n, HD)
    v[32:64] *= f32(2.0 ** -40)
    k[96:128] *= f32(2.0 ** -30)
    q = make(rng, 1, T, HD, 1.5)
    c = ctx.kvWrite8(cache(1, n, 1, HD), put(ctx, k), put(ctx, v))
    want, bound = attention(q.reshape(1, T, 1, HD), all_stored(k, 1, 1), all_stored(v, 1, 1), [[n] * T])
    assert np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n)) - want).max() <= bound


def test_a_query_that_is_not_finite(ctx, cache):
    n, HD = 40, 64
    rng = np.random.default_rng(7)
    c = ctx.kvWrite8(cache(1, n, 1, HD), put(ctx, make(rng, 1, n, HD)), put(ctx, make(rng, 1, n, HD)))
    q = make(rng, 1, 4, HD, 1 / 8)
    q[0, 3], q[1, 60], q[2] = np.nan, -np.inf, 0
    out = got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n))
    assert np.isnan(out[:2]).all() and np.isfinite(out[2:]).all()


def test_offsets_past_32_bits(ctx, cache):
    """A cache of 5.2 GB: the last stream's codes lie behind 2^32 bytes."""
    S, P, H, HD, n = 5, 1 << 21, 1, 256, 70
    c = cache(S, P, H, HD)
    rng = np.random.default_rng(9)
    k, v, q = make(rng, S, n, HD), make(rng, S, n, HD), make(rng, S, 1, HD, 1 / 16)
    ctx.kvWrite8(c, put(ctx, k), put(ctx, v))
    want, bound = attention(q.reshape(S, 1, 1, HD), all_stored(k, S, H), all_stored(v, S, H), [[n]] * S)
    assert np.abs(got(ctx, ctx.attnKv8(put(ctx, q), c, 1, n)) - want).max() <= bound
    ctx.kvWrite8(c, put(ctx, k), put(ctx, v), P - n)  # at the end of each stream
    assert np.array_equal(got(ctx, ctx.kvRead8(c, P - n, n)[1])[-n + 6:], all_stored(np.concatenate([np.zeros((26, HD), f32), v[-n:]]), 1, 1)[0, 0, 32:])


def test_the_product_that_follows_reads_the_same_values(ctx, cache):
    for S, n in ((3, 50), (100, 40)):
        H, HD = 4, 64
        rng = np.random.default_rng(S)
        c = ctx.kvWrite8(cache(S, n, H, HD), put(ctx, make(rng, S, n, H * HD)), put(ctx, make(rng, S, n, H * HD)))
        out = ctx.attnKv8(put(ctx, make(rng, S, 1, H * HD, 1 / 8)), c, H, n)
        w = put(ctx, make(rng, 1, H * HD, 512, 1 / 16), True)
        a = got(ctx, ctx.matmul(out, w))
        assert np.array_equal(a, got(ctx, ctx.matmul(put(ctx, got(ctx, out)), w)))


def test_recorded_and_replayed(ctx, cache):
    """A recording of a step at positions that the device holds: replays see the positions of their time."""
    S, H, HD, P = 3, 2, 64, 80
    rng = np.random.default_rng(10)
    D = H * HD
    qkv = np.concatenate([make(rng, S, P, D, 1 / 8), make(rng, S, P, 2 * D)], 1).reshape(S, P, 3 * D)
    eager, played = cache(S, P, H, HD), cache(S, P, H, HD)
    x, pos = ctx.alloc(S, 3 * D), ctx.alloc(1, S)

    def at(i):
        ctx.copyRows(x, put(ctx, qkv[:, i]), 0)
        ctx.copyRows(pos, put(ctx, [[i] * S]), 0)

    at(0)
    ctx.freeTensor(ctx.attnAppendKv8(x, played, H, pos=pos))
    batch, y = ctx.recordBatch(lambda: ctx.attnAppendKv8(x, played, H, pos=pos))
    for i in range(P):
        at(i)
        batch.launch()
        want = ctx.attnAppendKv8(x, eager, H, i)
        a, b = got(ctx, y), got(ctx, want)
        # the recorded launch is sized for the whole cache: the same sums, joined in other groups
        assert np.abs(a - b).max() <= 2.0 ** -20 * np.abs(qkv).max()
    assert all(np.array_equal(got(ctx, a), got(ctx, b)) for a, b in zip(ctx.kvRead8(eager, 0, P), ctx.kvRead8(played, 0, P)))
    batch.free()


@pytest.mark.parametrize("S,H,n", [(1, 20, 447), (48, 12, 200), (3, 4, 31)])
def test_tokens_in_a_row_without_a_pause(ctx, cache, S, H, n):
    """Each token reads what the call before it wrote: one recording against calls that wait for one another."""
    rng = np.random.default_rng(23)
    steps, w = 6, H * 64
    k, v = make(rng, S, n, w), make(rng, S, n, w)
    xs = [put(ctx, make(rng, S, 1, 3 * w, 0.3)) for _ in range(steps)]
    tk, tv = put(ctx, k), put(ctx, v)

    def run(c, pause):
        ctx.kvWrite8(c, tk, tv)
        out = []
        for i in range(steps):
            out.append(ctx.attnAppendKv8(xs[i], c, H, n + i))
            if pause:
                ctx.sync()
        return out

    c = cache(S, n + steps, H, 64)
    want = [got(ctx, t) for t in run(c, True)]
    graph, outs = ctx.recordBatch(lambda: run(c, False))
    for _ in range(3):
        graph.launch()
        for t, y in zip(outs, want):
            assert np.array_equal(got(ctx, t), y)
    graph.free()


def test_lengths_outside_are_reported(ctx, cache, pkg):
    S, H, HD, n = 2, 1, 64, 40
    rng = np.random.default_rng(11)
    c = cache(S, n, H, HD)
    t = put(ctx, make(rng, S, n, HD))
    q, qkv = put(ctx, make(rng, S, 1, HD)), put(ctx, make(rng, S, 1, 3 * HD))
    calls = [lambda bad: ctx.kvWrite8(c, t, t, counts=bad(n + 1)), lambda bad: ctx.kvWrite8(c, q, q, pos=bad(n)),
             lambda bad: ctx.attnKv8(q, c, 1, n, lens=bad(n + 1)), lambda bad: ctx.attnAppendKv8(qkv, c, 1, pos=bad(n))]
    for call in calls:
        for over in (True, False, float("nan")):
            bad = lambda top: put(ctx, [[0, top if over is True else -1 if over is False else over]])  # noqa: E731
            ctx.sync()
            call(bad)
            with pytest.raises(pkg.CudaError, match="8-bit cache"):
                ctx.sync()
            ctx.sync()


def test_refusals(ctx, cache, pkg):
    c = cache(2, 64, 2, 32)
    t, q = ctx.alloc(20, 64), ctx.alloc(2, 128)
    f16 = ctx.allocF16(20, 64)
    qkv, two = ctx.alloc(2, 256), ctx.alloc(1, 2)
    other = pkg.CudaContext(0)
    foreign = other.kvCache8(2, 64, 2, 32)
    gone = ctx.kvCache8(1, 1, 1, 1)
    stale = pkg.KvCache8(gone.h, 1, 1, 1, 1)
    ctx.freeKvCache8(gone)
    bad = [lambda: ctx.kvCache8(0, 1, 1, 1), lambda: ctx.kvCache8(1, 0, 1, 1), lambda: ctx.kvCache8(1, 1, 0, 1), lambda: ctx.kvCache8(1, 1, 1, 257),
           lambda: ctx.kvCache8(1, (1 << 24) + 1, 1, 1), lambda: ctx.kvCache8(65536, 1, 1, 1), lambda: ctx.kvCache8(1, 1, 1, 0),
           lambda: ctx.freeKvCache8(stale), lambda: ctx.kvRead8(stale, 0, 1), lambda: ctx.kvWrite8(foreign, t, t),
           lambda: ctx.kvWrite8(c, t, f16), lambda: ctx.kvWrite8(c, q, q), lambda: ctx.kvWrite8(c, t, t, 55), lambda: ctx.kvWrite8(c, t, t, -1),
           lambda: ctx.kvWrite8(c, t, ctx.alloc(18, 64)), lambda: ctx.kvWrite8(c, ctx.alloc(3, 64), ctx.alloc(3, 64)),
           lambda: ctx.kvWrite8(c, t, t, counts=ctx.alloc(1, 3)), lambda: ctx.kvWrite8(c, t, t, pos=ctx.allocF16(1, 2)),
           lambda: ctx.kvRead8(c, 0, 65), lambda: ctx.kvRead8(c, -1, 1), lambda: ctx.kvRead8(c, 64, 1), lambda: ctx.kvRead8(c, 0, -1),
           lambda: ctx.attnKv8(q, c, 4, 65), lambda: ctx.attnKv8(q, c, 4, -1), lambda: ctx.attnKv8(q, c, 3, 5), lambda: ctx.attnKv8(q, c, 2, 5),
           lambda: ctx.attnKv8(q, c, 0, 5), lambda: ctx.attnKv8(ctx.allocF16(2, 128), c, 4, 5), lambda: ctx.attnKv8(ctx.alloc(3, 128), c, 4, 5),
           lambda: ctx.attnKv8(q, c, 4, 5, lens=ctx.alloc(2, 2)), lambda: ctx.attnAppendKv8(qkv, c, 4, 64), lambda: ctx.attnAppendKv8(q, c, 4, 0),
           lambda: ctx.attnAppendKv8(ctx.alloc(130, 256), c, 4, pos=two)]
    for i, call in enumerate(bad):
        with pytest.raises(pkg.CudaError) as e:
            call()
        assert e.value.code == 1, i
    with pytest.raises(pkg.CudaError, match="recorded"):
        ctx.recordBatch(lambda: ctx.kvCache8(1, 1, 1, 1))
    ctx.sync()
    # nothing to do is no error
    ctx.kvWrite8(c, ctx.alloc(0, 64), ctx.alloc(0, 64), 64)
    assert ctx.attnKv8(ctx.alloc(0, 128), c, 4, 0).rows == 0
    assert ctx.kvRead8(c, 64, 0)[0].rows == 0
    assert not got(ctx, ctx.attnKv8(put(ctx, np.ones((2, 128))), c, 4, 0)).any()
    other.destroy()


def test_two_contexts_at_once(ctx, cache, pkg):
    """Two streams of the GPU through caches of their own, neither waiting for the other."""
    S, H, HD, n = 2, 4, 64, 700
    rng = np.random.default_rng(12)
    other = pkg.CudaContext(0)
    k, v, q = make(rng, S, n, H * HD), make(rng, S, n, H * HD), make(rng, S, 1, H * HD, 1 / 8)
    both = [(x, x.kvWrite8(x.kvCache8(S, n, H, HD), put(x, k), put(x, v)), put(x, q)) for x in (ctx, other)]
    outs = [[], []]
    for _ in range(50):
        for i, (x, c, t) in enumerate(both):
            outs[i].append(x.attnKv8(t, c, H, n))
    first = got(ctx, outs[0][0])
    for i, (x, c, t) in enumerate(both):
        assert all(np.array_equal(got(x, o), first) for o in outs[i])
    ctx.freeKvCache8(both[0][1])
    other.destroy()
