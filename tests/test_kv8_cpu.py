"""The 8-bit cache and the logit rules at the boundary, without a GPU: calls without a context are refused with a message, and the
structs are laid out as the header says."""
import ctypes as C


def test_calls_without_a_context_are_refused(pkg):
    lib = pkg.load_library()
    out, out2 = C.c_void_p(), C.c_void_p()
    calls = [("kvCache8", lambda: lib.fa_kv8_create(None, 1, 1, 1, 1, C.byref(out))), ("freeKvCache8", lambda: lib.fa_kv8_free(None, None)),
             ("kvWrite8", lambda: lib.fa_kv8_write(None, None, None, None, 0, None, None)),
             ("kvRead8", lambda: lib.fa_kv8_read(None, None, 0, 1, C.byref(out), C.byref(out2))),
             ("attnKv8", lambda: lib.fa_attn_kv8(None, None, None, 1, 1, None, C.byref(out))),
             ("attnAppendKv8", lambda: lib.fa_attn_append_kv8(None, None, None, 1, 1, None, None, C.byref(out))),
             ("adjustLogits", lambda: lib.fa_adjust_logits(None, None, 0, None, C.byref(out))),
             ("pickAdjusted", lambda: lib.fa_pick_adjusted(None, None, 0, None, C.byref(out)))]
    for name, call in calls:
        assert call() == 1
        assert name.encode() in lib.fa_last_error(None)


def test_rules_struct(pkg):
    from fluidaudio_web_b200 import _lib

    r = _lib.LogitRules
    assert [getattr(r, n).offset for n, _ in r._fields_] == [0, 8, 12, 16, 20, 24, 32, 40] and C.sizeof(r) == 48
