"""What the lock-step decoder refuses before anything is computed, on the CPU oracle."""
import numpy as np
import pytest

from oracle.wasm_oracle import WasmOracle


class WithRules(WasmOracle):
    """The oracle with the members of the pick on the device, on the host: a presence penalty, a mask [VOCAB] or [S, VOCAB] of truth values."""

    def argmaxRowsIndex(self, x, ncols=0):
        return WithRules.pickAdjusted(self, x, ncols)

    def pickAdjusted(self, x, ncols=0, *, history=None, n=0, presence=0.0, mask=None):
        y = x.array()[:, :ncols].copy()
        assert history is None or n <= history.rows
        for row in history.array()[:n] if n else ():
            for s, t in enumerate(row):
                if t >= 0:
                    y[s, int(t)] -= presence
        if mask is not None:
            y = np.where(mask, y, -np.inf)
        best = y.argmax(1)
        value = y.max(1)
        return self.upload(np.stack([np.where(value > -np.inf, best, -1), value], 1).astype(np.float32), x.rows, 2)


@pytest.fixture
def setup(pkg):
    from fluidaudio_web_b200.engines import synth, whisper_decoder as wd

    cfg, ctx, S = synth.TINY_DEC, WasmOracle(), 2
    dec = wd.load_decoder(ctx, synth.decoder_weights(cfg), cfg["NH"])
    encs = [ctx.upload(e, cfg["Tenc"], cfg["D"]) for e in synth.encoder_states(cfg, S)]
    return wd, ctx, dec, encs, S


def test_tokens_behind_the_position_table(setup):
    """A cache may be longer than the table: the last place of the table works, one behind it is refused and nothing moves."""
    wd, ctx, dec, encs, S = setup
    table = dec["pos"].shape[0]
    kv, st = wd.cross_kv_streams(ctx, dec, encs), wd.decode_init_streams(ctx, dec, S, table + 8)
    st["n"] = table - 1
    wd.decode_next_streams(ctx, dec, kv, st, [1] * S)
    assert st["n"] == table
    with pytest.raises(IndexError):
        wd.decode_next_streams(ctx, dec, kv, st, [1] * S)
    assert st["n"] == table
    # prompts: with one row of the table left it would stand for all tokens
    for n, T in ((table - 1, 2), (table - 1, 5), (table, 2), (0, table + 1)):
        with pytest.raises(IndexError):
            wd.prefill_streams(ctx, dec, kv, dict(n=n, S=S, self8=[]), np.ones((S, T)))


def test_rules_are_refused_where_nobody_follows_them(setup):
    """The oracle has no pickAdjusted: its pick on the host would be the plain one."""
    wd, ctx, dec, encs, S = setup
    assert not hasattr(ctx, "pickAdjusted")
    kv, st = wd.cross_kv_streams(ctx, dec, encs), wd.decode_init_streams(ctx, dec, S, 8)
    for rules in (dict(presence=1e6), dict()):
        for call in (lambda: wd.decode_next_streams(ctx, dec, kv, st, [1] * S, rules=rules), lambda: wd.prefill_streams(ctx, dec, kv, st, np.ones((S, 1)), rules=rules),
                     lambda: wd.greedy_decode_streams(ctx, dec, encs, [1, 2], 3, rules=rules)):
            with pytest.raises(ValueError, match="pickAdjusted"):
                call()
    assert st["n"] == 0
    wd.greedy_decode_streams(ctx, dec, encs, [1, 2], 3)


def test_history_of_a_state_that_is_set_back(setup):
    """Picks behind the position that a state is set back to are of another run; those in front of it stay."""
    wd, _, dec, encs, S = setup
    ctx = WithRules()
    kv, st = wd.cross_kv_streams(ctx, dec, encs), wd.decode_init_streams(ctx, dec, S, 6)
    rules = dict(presence=1e6)

    def run(state, first, count):
        out, t = [], first
        for _ in range(count):
            t = wd.decode_next_streams(ctx, dec, kv, state, t, rules=rules)[0]
            out.append(t.tolist())
        return out

    want = run(wd.decode_init_streams(ctx, dec, S, 6), [1] * S, 6)
    assert all(len({r[s] for r in want}) == 6 for s in range(S))
    for _ in range(3):
        st["n"] = 0
        assert run(st, [1] * S, 6) == want
    st["n"] = 2  # the two tokens before it count, the four behind it do not
    assert run(st, want[1], 4) == want[2:]


@pytest.mark.parametrize("n", [1, 7])
def test_a_stream_that_may_pick_nothing_ends_alone(setup, n):
    """A few tokens are allowed for stream 0, each once: it ends behind the last of them.  The other stream decodes as it does without it."""
    wd, _, dec, encs, S = setup
    ctx = WithRules()
    V = dec["cfg"]["VOCAB"]

    class Taking(WithRules):
        def __init__(self, only):
            super().__init__()
            self.left = np.ones((S, V), bool)
            self.left[0] = np.isin(np.arange(V), only)

        def pickAdjusted(self, x, ncols=0, **kw):
            pick = super().pickAdjusted(x, ncols, mask=self.left, **kw)
            t = int(pick.array()[0, 0])
            if t >= 0:
                self.left[0, t] = False
            return pick

    got = {}
    for only in ([3, 50, 7, 120, 9], [3], []):
        out = wd.greedy_decode_streams(Taking(only), dec, encs, [1, 2], n, rules=dict(presence=1e6))
        have = min(n, len(only))
        assert set(out[0, :have]) <= set(only) and len(set(out[0, :have])) == have and (out[0, have:] == -1).all()
        got[len(only)] = out[1].tolist()
    want = wd.greedy_decode_streams(ctx, dec, encs, [1, 2], n, rules=dict(presence=1e6))[1].tolist()
    assert all(r == want for r in got.values()) and min(want) >= 0
    none = dict(mask=np.zeros(V, bool))
    assert (wd.greedy_decode_streams(ctx, dec, encs, [1, 2], n, rules=none) == -1).all()


class Counting(WithRules):
    """Which tensors are pinned and not given back; 8-bit caches that hold nothing; the `fail`-th product fails."""

    def __init__(self, fail=0):
        super().__init__()
        self.live, self.products, self.fail = {}, 0, fail

    def matmul(self, *a, **kw):
        self.products += 1
        if self.products == self.fail:
            raise MemoryError("no room")
        return super().matmul(*a, **kw)

    def pin(self, t, toParent=False):
        self.live[id(t)] = t
        return t

    def freeTensor(self, t):
        self.live.pop(id(t), None)

    def kvCache8(self, *shape):
        return self.pin(object())

    def kvWrite8(self, cache, *a, **kw):
        pass

    def freeKvCache8(self, cache):
        self.freeTensor(cache)


@pytest.mark.parametrize("cache", [None, "int8"])
def test_what_was_made_goes_back_when_a_product_fails(setup, cache):
    wd, _, dec, encs, S = setup
    products = 2 * len(dec["layers"])
    for fail in range(1, products + 1):
        ctx = Counting(fail)
        with pytest.raises(MemoryError):
            wd.cross_kv_streams(ctx, dec, encs, cache)
        assert ctx.products == fail and not ctx.live
    ctx = Counting()
    kv = wd.cross_kv_streams(ctx, dec, encs, cache)
    assert len(ctx.live) == (len(dec["layers"]) if cache else products)
    wd.free_caches(ctx, kv)
    assert len(ctx.live) == (0 if cache else products)


def test_a_states_history_goes_back(setup):
    wd, _, dec, encs, S = setup
    ctx = Counting()
    kv, st = wd.cross_kv_streams(ctx, dec, encs), wd.decode_init_streams(ctx, dec, S, 6)
    before = set(ctx.live)
    first = wd.decode_next_streams(ctx, dec, kv, st, [1] * S, rules=dict(presence=1e6))[0].tolist()
    assert len(ctx.live) == len(before) + 1
    wd.free_caches(ctx, kv, st)
    assert set(ctx.live) == before
    wd.free_caches(ctx, kv, st)  # twice is no error
    st["n"] = 0
    assert wd.decode_next_streams(ctx, dec, kv, st, [1] * S, rules=dict(presence=1e6))[0].tolist() == first
    # a history that the loop made for a state of its own, and one that stays with the caller's
    held = len(ctx.live)
    wd.greedy_decode_streams(ctx, dec, encs, [1, 2], 3, kv=kv, st=st, rules=dict(presence=1e6))
    assert len(ctx.live) == held
