"""Penalties, biases and masks on logits against the formulas.

Every step of the rules is rounded to f32 by itself, so numpy's f32 arithmetic in the same order gives the same bits; that
order is compared with float64 within its five half steps."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32


def rules(x, V, hist=None, n=0, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None, t=f32):
    x = x[:, :V].astype(t)
    S = x.shape[0]
    if hist is not None and n:
        c = np.zeros((S, V), t)
        for s in range(S):
            ids = hist[:n, s]
            ids = ids[(ids >= 0) & (ids < V)].astype(np.int64)
            np.add.at(c[s], ids, t(1))
        r, p, f = (t(f32(a)) for a in (repetition, presence, frequency))
        with np.errstate(all="ignore"):
            x = np.where(c > 0, (np.where(x > 0, x / r, x * r) - c * f) - p, x)
    if bias is not None:
        x = x + bias[:, :V].astype(t)
    return x if allowed is None else np.where(allowed, x, t(-np.inf))


def pick(y, allowed):
    """first largest allowed value, NaN never"""
    out = np.zeros((y.shape[0], 2), f32)
    for s in range(y.shape[0]):
        could = ~np.isnan(y[s]) & (True if allowed is None else allowed[s])
        at = np.nonzero(could)[0]
        if at.size:
            j = at[np.argmax(y[s, at])]
            out[s] = j, y[s, j]
        else:
            out[s] = -1, -np.inf
    return out


def bits(allowed):
    """[rows, V] truth values -> rows of little-endian 32-bit words"""
    pad = -allowed.shape[1] % 32
    return np.packbits(np.pad(allowed, ((0, 0), (0, pad))), axis=1, bitorder="little")


def put(ctx, x):
    x = np.ascontiguousarray(x, dtype=f32)
    return ctx.upload(x, *x.shape)


def got(ctx, t):
    return ctx.download(t).reshape(t.rows, t.cols)


# rows, columns, columns in use, history rows in use, biases, mask rows (-1: a table with an index)
CASES = [(1, 1, 1, 1, 0, 0), (1, 33, 32, 5, 1, 1), (3, 31, 31, 0, 3, 3), (5, 257, 250, 40, 0, -1), (1, 51866, 51866, 224, 1, 1), (64, 5187, 5187, 448, 0, -1),
         (2, 51868, 51866, 3000, 2, 2), (300, 1000, 999, 17, 1, 0), (2, 300001, 300001, 64, 0, 1), (700, 40, 40, 100, 700, 700)]


@pytest.mark.parametrize("S,C,V,n,nbias,nmask", CASES)
def test_rules_and_pick(ctx, S, C, V, n, nbias, nmask):
    rng = np.random.default_rng(C + S)
    x = (3 * rng.standard_normal((S, C))).astype(f32)
    x[:, V:] = 100  # columns behind the ones asked for
    hist = np.floor(V * rng.random((n + 3, S)) ** 4)
    hist[rng.random(hist.shape) < 0.1] = -1
    hist[rng.random(hist.shape) < 0.05] = V  # outside the columns: no token
    bias = (rng.standard_normal((nbias, C)) * (rng.random((nbias, C)) < 0.1)).astype(f32) if nbias else None
    kw, allowed, opts = {}, None, dict(n=n, repetition=1.3, presence=0.7, frequency=0.11)
    if nmask:
        table = rng.random((4 if nmask < 0 else nmask, V)) < 0.6
        kw["mask"] = ctx.uploadBytes(bits(table))
        index = rng.integers(0, 4, S) if nmask < 0 else np.arange(S) if nmask > 1 else np.zeros(S, int)
        if nmask < 0:
            kw["maskRows"] = put(ctx, index[:, None])
        allowed = table[index]
        allowed[S // 2] = allowed[S // 2] if nmask < 0 or nmask == 1 else False
        if nmask > 1:
            kw["mask"] = ctx.uploadBytes(bits(allowed))
    if nbias:
        kw["bias"] = put(ctx, bias)
    want = rules(x, V, hist, bias=bias, allowed=allowed, **opts)
    tx, th = put(ctx, x), put(ctx, hist)
    y = got(ctx, ctx.adjustLogits(tx, V, history=th, **opts, **kw))
    assert np.array_equal(y, want)
    assert np.array_equal(got(ctx, ctx.pickAdjusted(tx, V, history=th, **opts, **kw)), pick(want, allowed))
    exact = rules(x, V, hist, bias=bias, allowed=allowed, t=np.float64, **opts)
    fin = np.isfinite(exact)
    size = 1.3 * np.abs(x).max() + 0.11 * n + 0.7 + (np.abs(bias).max() if nbias else 0)  # no intermediate is larger
    assert np.abs(y[fin] - exact[fin]).max(initial=0) <= 5 * 2.0 ** -24 * size


def test_no_rules_is_the_row_argmax(ctx):
    rng = np.random.default_rng(1)
    x = rng.integers(-20, 20, (9, 4099)).astype(f32)  # many ties
    t = put(ctx, x)
    assert np.array_equal(got(ctx, ctx.pickAdjusted(t)), got(ctx, ctx.argmaxRowsIndex(t)))
    assert np.array_equal(got(ctx, ctx.adjustLogits(t)), x)
    assert np.array_equal(got(ctx, ctx.adjustLogits(t, 77, history=put(ctx, np.zeros((4, 9))), n=4)), x[:, :77])


def test_infinities_nans_and_empty_rows(ctx):
    V = 100
    x = np.zeros((7, V), f32)
    x[0] = np.nan                      # nothing to pick
    x[1] = -np.inf                     # the first token, at -inf
    x[2, 50] = np.nan                  # a NaN never wins
    x[3, 10], x[3, 11] = np.inf, 3     # the mask takes the infinity away
    x[4, 20] = np.float32(-3.4e38)     # the lowest value under the penalty overflows to -inf
    x[5] = np.nan                      # masked to one finite token
    x[5, 99] = -7
    allowed = np.ones((7, V), bool)
    allowed[3, 10] = False
    allowed[5, :99] = False
    allowed[6] = False                 # a grammar that allows nothing
    hist = np.tile(np.array([[20.0]], f32), (3, 7))
    kw = dict(n=3, repetition=2.0, presence=0.5, frequency=0.25)
    with np.errstate(all="ignore"):
        want = rules(x, V, hist, allowed=allowed, **kw)
    t, m, h = put(ctx, x), ctx.uploadBytes(bits(allowed)), put(ctx, hist)
    assert np.array_equal(got(ctx, ctx.adjustLogits(t, mask=m, history=h, **kw)), want, equal_nan=True)
    best = got(ctx, ctx.pickAdjusted(t, mask=m, history=h, **kw))
    assert np.array_equal(best, pick(want, allowed))
    assert best[0].tolist() == [-1, -np.inf] and best[1].tolist() == [0, -np.inf] and best[3].tolist() == [11, 3]
    assert best[5].tolist() == [99, -7] and best[6].tolist() == [-1, -np.inf]


def test_history_values_that_are_no_tokens(ctx):
    x = np.ones((1, 64), f32)
    for bad in (np.nan, np.inf, -np.inf, -1, 64, 1e30, -0.5):
        y = got(ctx, ctx.adjustLogits(put(ctx, x), history=put(ctx, [[bad]]), n=1, presence=1.0))
        assert np.array_equal(y, x), bad


def test_one_token_many_times(ctx):
    n = 70000  # more than 16 bits count
    x = np.ones((1, 50), f32)
    y = got(ctx, ctx.adjustLogits(put(ctx, x), history=put(ctx, np.full((n, 1), 7)), n=n, frequency=1.0))
    assert y[0, 7] == 1 - n and np.array_equal(np.delete(y, 7), np.ones(49, f32))


@pytest.mark.parametrize("S", [1, 400])
@pytest.mark.parametrize("n", [65535, 65536])
def test_counts_at_the_end_of_16_bits(ctx, S, n):
    x = np.ones((S, 50), f32)
    hist = np.full((n, 1), 6) + np.arange(S) % 2  # the even one of a pair, or the odd one
    y = got(ctx, ctx.adjustLogits(put(ctx, x), history=put(ctx, hist), n=n, frequency=1.0))
    want = x.copy()
    want[np.arange(S), 6 + np.arange(S) % 2] = 1 - n
    assert np.array_equal(y, want)


def test_recorded_with_a_growing_history(ctx):
    """A decode of a few tokens, picks written into the history on the device, recorded once and replayed."""
    S, V, n = 3, 501, 6
    rng = np.random.default_rng(2)
    x = put(ctx, rng.standard_normal((S, V)))
    hist = ctx.alloc(n, S)

    def body():
        for i in range(n):
            t = ctx.pickAdjusted(x, history=hist, n=i, presence=50.0)
            ctx.copyRows(hist, ctx.reshapeView(ctx.sliceCols(t, 0, 1), 1, S), i)

    body()
    order = np.argsort(-got(ctx, x), axis=1, kind="stable")[:, :n].T
    assert np.array_equal(got(ctx, hist), order)  # each token once, best first
    batch, _ = ctx.recordBatch(body)
    for _ in range(2):
        ctx.copyRows(hist, put(ctx, np.zeros((n, S))), 0)
        batch.launch()
        assert np.array_equal(got(ctx, hist), order)
    batch.free()


def test_mask_rows_outside_the_table_are_reported(ctx, pkg):
    x, m = put(ctx, np.zeros((2, 40))), ctx.uploadBytes(np.full(3 * 8, 255, np.uint8))
    for bad in (3, -1, np.nan):
        ctx.sync()
        ctx.pickAdjusted(x, mask=m, maskRows=put(ctx, [[0, bad]]))
        with pytest.raises(pkg.CudaError, match="mask row"):
            ctx.sync()
        ctx.sync()


def test_refusals(ctx, pkg):
    x, h = ctx.alloc(2, 64), ctx.alloc(5, 2)
    m = ctx.uploadBytes(np.zeros(3 * 8, np.uint8))
    bad = [dict(ncols=65), dict(history=ctx.alloc(5, 3)), dict(history=h, n=6), dict(history=h, n=-1), dict(history=h, n=1, repetition=0.0),
           dict(history=h, n=1, repetition=-1.0), dict(history=h, n=1, repetition=float("inf")), dict(history=h, n=1, repetition=float("nan")),
           dict(history=ctx.allocF16(5, 2)), dict(bias=ctx.alloc(1, 63)), dict(bias=ctx.alloc(3, 64)), dict(mask=m),
           dict(mask=ctx.uploadBytes(np.zeros(7, np.uint8))), dict(mask=m, maskRows=ctx.alloc(1, 3)), dict(maskRows=ctx.alloc(1, 2)),
           dict(mask=ctx.uploadBytes(np.zeros(0, np.uint8)))]
    for i, kw in enumerate(bad):
        for call in (ctx.adjustLogits, ctx.pickAdjusted):
            with pytest.raises(pkg.CudaError) as e:
                call(x, **kw)
            assert e.value.code == 1, i
    with pytest.raises(pkg.CudaError):
        ctx.pickAdjusted(ctx.allocF16(2, 64))
    assert ctx.pickAdjusted(ctx.alloc(0, 64)).rows == 0
