"""The decoder over 8-bit caches with rules for the pick: against the same engine whose attention runs in float64 on what the caches hold.

Bound: the two differ in the attention's f32-grade sums alone (2^-20 of the largest value and what the scores' roundings add,
under 1e-5 here); two layers of O(1) weights and the vocabulary product carry that to logits of O(1) within 1e-4.  A code that
falls to the other side of a tie for it moves one value by a step s, 1/127 of its block's largest, 0.03 here; the position's
weight is 0.1 at most (38 positions and more, scores of O(1)) and the output and vocabulary matrices pass on less than a third,
so every stored value that differs by a step (they are counted) adds 1e-3 to the bound.  int8 products take three digits, and
products their rows as value and residue throughout (f16_hilo_rows): a row rounded to f16 alone would move by 2^-11."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32


class OnStoredValues:
    """The context, with the two attention members computed on the host from kvRead8."""

    def __init__(self, ctx):
        self.ctx = ctx

    def __getattr__(self, name):
        if name == "decoderStepKv8":
            raise AttributeError(name)
        return getattr(self.ctx, name)

    def _attend(self, q, cache, HQ, limit):
        c, S, T = self.ctx, cache.S, q.shape[0] // cache.S
        n = int(max(max(r) for r in limit))
        if n == 0:
            return c.upload(np.zeros(q.shape, f32), *q.shape)
        K, V = (c.download(t).astype(np.float64).reshape(S, n, cache.H, cache.HD) for t in c.kvRead8(cache, 0, n))
        q, out = q.reshape(S, T, HQ, cache.HD).astype(np.float64), np.zeros((S, T, HQ, cache.HD))
        for s in range(S):
            for i in range(T):
                m = int(limit[s][i])
                if m:
                    z = np.einsum("hd,jhd->hj", q[s, i], K[s, :m])
                    p = np.exp(z - z.max(1, keepdims=True))
                    out[s, i] = np.einsum("hj,jhd->hd", p / p.sum(1, keepdims=True), V[s, :m])
        return c.upload(out.reshape(S * T, -1).astype(f32), S * T, HQ * cache.HD)

    def attnKv8(self, q, cache, HQ, n, *, lens=None):
        lens = self.ctx.download(lens) if lens is not None else np.full(cache.S, n)
        return self._attend(self.ctx.download(q).reshape(q.rows, q.cols), cache, HQ, [[m] * (q.rows // cache.S) for m in lens])

    def attnAppendKv8(self, qkv, cache, HQ, n=0):
        c, D, E, T = self.ctx, HQ * cache.HD, cache.H * cache.HD, qkv.rows // cache.S
        c.kvWrite8(cache, c.sliceCols(qkv, D, E), c.sliceCols(qkv, D + E, E), n)
        q = c.download(c.sliceCols(qkv, 0, D)).reshape(qkv.rows, D)
        return self._attend(q, cache, HQ, [[n + i + 1 for i in range(T)]] * cache.S)


@pytest.fixture(autouse=True)
def f32_grade_products(ctx):
    ctx.setOption("f16_hilo_rows", 1 << 30)
    ctx.setOption("int8_limbs", 3)
    yield
    ctx.setOption("f16_hilo_rows", 64)
    ctx.setOption("int8_limbs", 2)


def stored(ctx, caches, s=None, rows=None):
    """What caches hold, of stream s alone if one is given."""
    got = []
    for c in caches:
        for t in ctx.kvRead8(c, 0, rows or c.positions):
            x = ctx.download(t).reshape(c.S, -1)
            got.append(x if s is None else x[s])
    return got


def steps_apart(a, b):
    """How many stored values differ by a step (1e-3 is far below one, far above rounding)."""
    return sum(int((np.abs(x - y) > 1e-3).sum()) for x, y in zip(a, b))


CFG = dict(D=256, NH=4, FFN=1024, layers=2, VOCAB=2003, maxPos=80, Tenc=96)


def _setup(ctx, S, quant=None, **kw):
    from fluidaudio_web_b200.engines import synth, whisper_decoder as wd

    cfg = dict(CFG, **kw)
    dec = wd.load_decoder(ctx, synth.decoder_weights(cfg, seed=11), cfg["NH"], quant=quant)
    states = np.concatenate(synth.encoder_states(cfg, S, seed=13))
    return wd, cfg, dec, ctx.upload(states, S * cfg["Tenc"], cfg["D"])


@pytest.mark.parametrize("S,NH,quant,lens", [(1, 4, None, None), (3, 4, None, [96, 50, 0]), (5, 16, None, None), (3, 4, "int8", [1, 96, 33]), (1, 5, None, None)])
def test_steps_and_prompts(ctx, S, NH, quant, lens):
    wd, cfg, dec, states = _setup(ctx, S, quant, NH=NH, D=240 if NH == 5 else 256)
    tl = None if lens is None else ctx.upload(np.asarray(lens, f32), 1, S)
    prompts = np.arange(S * 37).reshape(S, 37) % 1000 + 1
    runs, held = [], []
    for c in (ctx, OnStoredValues(ctx)):
        kv = wd.cross_kv_streams(c, dec, states, "int8", S=S, lens=tl)
        st = wd.decode_init_streams(c, dec, S, 60, "int8")
        got = [wd.prefill_streams(c, dec, kv, st, prompts, want_logits=True)[1]]
        got += [wd.decode_next_streams(c, dec, kv, st, [t] * S, want_logits=True)[1] for t in (1, 7, 3)]
        got.append(wd.prefill_streams(c, dec, kv, st, prompts[:, :5], want_logits=True)[1])
        assert st["n"] == 45
        held.append(stored(ctx, st["self8"]))
        wd.free_caches(c, kv, st)
        runs.append(got)
    for a, b in zip(*runs):
        assert np.abs(a - b).max() < 1e-4 + 1e-3 * steps_apart(*held)
    assert steps_apart(*held) < 20
    assert np.abs(runs[0][0] - runs[0][1]).max() > 1e-2


@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("quant", [None, "int8"])
def test_native_loop_gives_the_host_loops_bits(ctx, S, quant):
    wd, cfg, dec, states = _setup(ctx, S, quant)
    layers, runs, held = dec["layers"], [], []
    fused = [{k: v for k, v in w.items() if k != "native"} for w in layers]
    parts = [{k: v for k, v in w.items() if not k.startswith("sqkv") and k != "native"} for w in layers]
    for use in (layers, fused, parts):
        dec["layers"] = use
        kv, st = wd.cross_kv_streams(ctx, dec, states, "int8", S=S), wd.decode_init_streams(ctx, dec, S, 20, "int8")
        before = ctx.handleCount()
        held.append(st["self8"])
        runs.append([wd.prefill_streams(ctx, dec, kv, st, np.tile([3, 1, 4], (S, 1)), want_logits=True)[1]]
                    + [wd.decode_next_streams(ctx, dec, kv, st, [t] * S, want_logits=True)[1] for t in (1, 5)])
        assert use is not layers or ctx.handleCount() == before
        held[-1] = stored(ctx, st["self8"])
        wd.free_caches(ctx, kv, st)
    for a, b, c in zip(*runs):
        assert np.array_equal(a, b)
        assert np.abs(a - c).max() < 1e-4 + 1e-3 * steps_apart(held[0], held[2])


def test_a_short_clip_among_long_ones_decodes_as_on_its_own(ctx):
    S, short = 4, 41
    wd, cfg, dec, states = _setup(ctx, S)
    lens = ctx.upload(np.array([96, short, 96, 70], f32), 1, S)
    kv, st = wd.cross_kv_streams(ctx, dec, states, "int8", S=S, lens=lens), wd.decode_init_streams(ctx, dec, S, 10, "int8")
    alone = ctx.sliceRows(states, 96, short)
    kv1, st1 = wd.cross_kv_streams(ctx, dec, [alone], "int8"), wd.decode_init_streams(ctx, dec, 1, 10, "int8")
    for t in (1, 9, 4):
        many = wd.decode_next_streams(ctx, dec, kv, st, [t] * S, want_logits=True)[1]
        one = wd.decode_next_streams(ctx, dec, kv1, st1, [t], want_logits=True)[1]
        apart = steps_apart(stored(ctx, [c["cache"] for c in kv], 1, short), stored(ctx, [c["cache"] for c in kv1], 0))
        apart += steps_apart(stored(ctx, st["self8"], 1), stored(ctx, st1["self8"], 0))
        assert apart < 20 and np.abs(many[1] - one[0]).max() < 1e-4 + 1e-3 * apart
    wd.free_caches(ctx, kv, st)
    wd.free_caches(ctx, kv1, st1)


def test_greedy_decoding_with_caches_lengths_and_rules(ctx):
    """All of it together, as a transcription runs it: ragged clips, a prompt, penalties, a mask; against the host's picks."""
    S, n, prefix = 3, 12, [2, 3, 5, 7]
    wd, cfg, dec, states = _setup(ctx, S)
    V = cfg["VOCAB"]
    encs = [ctx.sliceRows(states, s * 96, 96) for s in range(S)]
    lens = ctx.upload(np.array([96, 20, 77], f32), 1, S)
    allowed = np.random.default_rng(3).random((2, V)) < 0.5
    rows = [1, 0, 1]
    rules = dict(repetition=1.5, presence=0.25, frequency=0.5, mask=ctx.uploadBytes(np.packbits(np.pad(allowed, ((0, 0), (0, -V % 32))), axis=1, bitorder="little")),
                 maskRows=ctx.upload(np.array(rows, f32), S, 1), bias=ctx.upload(np.linspace(0, 0.1, V, dtype=f32), 1, V))
    got = wd.greedy_decode_streams(ctx, dec, encs, prefix, n, cache="int8", lens=lens, rules=rules)
    kv, st = wd.cross_kv_streams(ctx, dec, encs, "int8", lens=lens), wd.decode_init_streams(ctx, dec, S, 20, "int8")
    lg = wd.prefill_streams(ctx, dec, kv, st, np.tile(prefix, (S, 1)), want_logits=True)[1]
    seen = np.zeros((S, V))
    for i in range(n):
        y = lg.astype(np.float64)
        y = np.where(seen > 0, np.where(y > 0, y / 1.5, y * 1.5) - 0.5 * seen - 0.25, y) + np.linspace(0, 0.1, V)
        y[~allowed[rows]] = -np.inf
        pick = y.argmax(1)
        top = np.sort(y, 1)[:, -2:]
        assert np.all((pick == got[:, i]) | (top[:, 1] - top[:, 0] < 1e-5))
        assert all(allowed[r][t] for r, t in zip(rows, got[:, i]))
        seen[np.arange(S), got[:, i]] += 1
        lg = wd.decode_next_streams(ctx, dec, kv, st, got[:, i], want_logits=True)[1]
    wd.free_caches(ctx, kv, st)


def test_a_penalty_keeps_tokens_from_coming_twice(ctx):
    S, n = 2, 15
    wd, cfg, dec, states = _setup(ctx, S)
    encs = [ctx.sliceRows(states, s * 96, 96) for s in range(S)]
    for kw in (dict(), dict(cache="int8")):  # the rules do not need the 8-bit caches
        got = wd.greedy_decode_streams(ctx, dec, encs, [1, 2], n, rules=dict(presence=1e6), **kw)
        assert all(len(set(r)) == n for r in got.tolist())
    pidx = [ctx.upload(np.full(S, t, f32), S, 1) for t in (1, 2)]
    resident = ctx.download(wd.greedy_decode_streams_resident(ctx, dec, states, S, pidx, n, rules=dict(presence=1e6))).reshape(n, S).T
    assert np.array_equal(resident, wd.greedy_decode_streams(ctx, dec, encs, [1, 2], n, rules=dict(presence=1e6)))


def test_what_the_engine_refuses(ctx, pkg):
    S = 2
    wd, cfg, dec, states = _setup(ctx, S)
    kv8, st8 = wd.cross_kv_streams(ctx, dec, states, "int8", S=S), wd.decode_init_streams(ctx, dec, S, 10, "int8")
    kv, st = wd.cross_kv_streams(ctx, dec, states), wd.decode_init_streams(ctx, dec, S, 10)
    lens = ctx.upload(np.ones(S, f32), 1, S)
    for bad in (lambda: wd.cross_kv_streams(ctx, dec, states, "fp4", S=S), lambda: wd.cross_kv_streams(ctx, dec, states, "int8", S=5),
                lambda: wd.cross_kv_streams(ctx, dec, states, lens=lens), lambda: wd.decode_init_streams(ctx, dec, S, 10, "fp4"),
                lambda: wd.decode_next_streams(ctx, dec, kv, st8, [1, 2]), lambda: wd.decode_next_streams(ctx, dec, kv8, st, [1, 2]),
                lambda: wd.prefill_streams(ctx, dec, kv, st, np.ones((S, 3))), lambda: wd.prefill_streams(ctx, dec, kv8, st8, np.ones((S + 1, 3))),
                lambda: wd.prefill_streams(ctx, dec, kv8, st8, np.ones((S, 0))), lambda: wd.decode_next_streams(ctx, dec, kv8, st8, [1, -1]),
                lambda: wd.decode_next_streams(ctx, dec, kv8, st8, [1, 1], want_logits=True, rules={})):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg.CudaError, match="rows"):  # a prompt that does not fit the cache
        wd.prefill_streams(ctx, dec, kv8, st8, np.ones((S, 11)))
    none = ctx.uploadBytes(np.zeros(((cfg["VOCAB"] + 31) // 32) * 4, np.uint8))
    st8["n"] = 0
    assert wd.decode_next_streams(ctx, dec, kv8, st8, [1, 2], rules=dict(mask=none))[0].tolist() == [-1, -1]
    wd.free_caches(ctx, kv8, st8)
    wd.free_caches(ctx, kv8, st8)  # twice is no error: the handles are gone


def test_caches_go_back_when_one_cannot_be_made(ctx, pkg, monkeypatch):
    wd, cfg, dec, states = _setup(ctx, 2)
    live, make, free = set(), ctx.kvCache8, ctx.freeKvCache8

    def limited(*a):
        if len(live) == limit:
            raise pkg.CudaError(-2, "out of memory")
        c = make(*a)
        live.add(id(c))
        return c

    def back(c):
        live.discard(id(c))
        free(c)

    monkeypatch.setattr(ctx, "kvCache8", limited)
    monkeypatch.setattr(ctx, "freeKvCache8", back)
    layers = len(dec["layers"])
    for limit, call in ((1, lambda: wd.cross_kv_streams(ctx, dec, states, "int8", S=2)), (1, lambda: wd.decode_init_streams(ctx, dec, 2, 10, "int8")),
                        (layers + 1, lambda: wd.greedy_decode_streams(ctx, dec, list(two), [1, 2], 3, cache="int8"))):
        two = [ctx.upload(np.ones((cfg["Tenc"], cfg["D"]), f32), cfg["Tenc"], cfg["D"]) for _ in range(2)]
        with pytest.raises(pkg.CudaError, match="out of memory"):
            call()
        assert not live
