"""8-bit caches of another number of streams than the call's: rows that happen to fit would meet other streams' keys."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32


def make(ctx, layers):
    from fluidaudio_web_b200.engines import synth, whisper_decoder as wd

    cfg = dict(D=64, NH=4, FFN=128, layers=layers, VOCAB=203, maxPos=32, Tenc=24)
    dec = wd.load_decoder(ctx, synth.decoder_weights(cfg, seed=3), cfg["NH"])
    states = np.concatenate(synth.encoder_states(cfg, 4, seed=5))
    return wd, cfg, dec, ctx.upload(states, 4 * cfg["Tenc"], cfg["D"])


def test_step_over_caches_of_different_stream_counts(ctx, pkg):
    wd, cfg, dec, states = make(ctx, 2)
    layers = dec["layers"]
    made = {S: (wd.cross_kv_streams(ctx, dec, states, "int8", S=S), wd.decode_init_streams(ctx, dec, S, 8, "int8")) for S in (1, 2, 4)}
    made[8] = (wd.cross_kv_streams(ctx, dec, states, "int8", S=8), None)
    # the host's loop and the native one
    for use in ([{k: v for k, v in w.items() if k != "native"} for w in layers], layers):
        dec["layers"] = use
        for a, b in ((4, 2), (4, 1), (2, 1)):
            with pytest.raises(ValueError, match="streams"):
                wd.decode_next_streams(ctx, dec, made[a][0], made[b][1], [1] * b)
            made[b][1]["n"] = 0
        for a, b in ((2, 4), (1, 4), (4, 4)):  # streams that share a clip
            wd.decode_next_streams(ctx, dec, made[a][0], made[b][1], [1] * b)
            made[b][1]["n"] = 0
    # the member itself, a single layer's cache being another's
    native = [wd.native_struct(w, wd.NATIVE_KEYS, wd._native_of(ctx)) for w in layers]
    x = ctx.upload(np.ones((4, cfg["D"]), f32), 4, cfg["D"])
    pick = lambda m, which: [e["cache"] for e in m[0]] if which == 0 else list(m[1]["self8"])  # noqa: E731
    for side in (0, 1):
        for layer in (0, 1):
            for S in (1, 2) if side else (8,):
                caches = [pick(made[4], 0), pick(made[4], 1)]
                caches[side][layer] = pick(made[S], side)[layer]
                with pytest.raises(pkg.CudaError) as e:
                    ctx.decoderStepKv8(native, x, caches[0], cfg["Tenc"], caches[1], 0, cfg["NH"], dec["lnf"], dec["embedT"].native())
                assert e.value.code == 1 and "streams" in str(e.value)
    gone = ctx.kvCache8(4, 8, cfg["NH"], 16)
    stale = pkg.KvCache8(gone.h, 4, 8, cfg["NH"], 16)
    ctx.freeKvCache8(gone)
    with pytest.raises(pkg.CudaError, match="layer 1"):
        ctx.decoderStepKv8(native, x, pick(made[4], 0), cfg["Tenc"], [made[4][1]["self8"][0], stale], 0, cfg["NH"], dec["lnf"], dec["embedT"].native())
    for m in made.values():
        wd.free_caches(ctx, *m)
    ctx.sync()


def test_streams_that_share_a_clip(ctx):
    """Two streams to a clip: the same logits as with the clip's keys and values there twice.  One layer: what its own cache holds
    comes before the attention over the clips, so the two hold the same codes and differ in the f32-grade sums of one attention
    alone, 1e-5 of values of O(1) (two queries a pass, four), which O(1) weights carry to logits of O(1) within 1e-4."""
    wd, cfg, dec, states = make(ctx, 1)
    w = cfg["Tenc"]
    twice = ctx.concatRows([ctx.sliceRows(states, s // 2 * w, w) for s in range(4)])
    st, other = wd.decode_init_streams(ctx, dec, 4, 8, "int8"), wd.decode_init_streams(ctx, dec, 4, 8, "int8")
    kv2, kv4 = wd.cross_kv_streams(ctx, dec, ctx.sliceRows(states, 0, 2 * w), "int8", S=2), wd.cross_kv_streams(ctx, dec, twice, "int8", S=4)
    for tokens in ([[1, 2, 3], [4, 5, 6], [7, 8, 9], [1, 1, 1]], [[5], [6], [7], [8]]):
        a, b = (wd.prefill_streams(ctx, dec, kv, s, np.array(tokens), want_logits=True)[1] for kv, s in ((kv2, st), (kv4, other)))
        assert np.abs(a - b).max() < 1e-4 and np.abs(a[0] - a[2]).max() > 1e-2
    wd.free_caches(ctx, kv2, st)
    wd.free_caches(ctx, kv4, other)
