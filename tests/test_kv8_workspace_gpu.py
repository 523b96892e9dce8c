"""Memory that the attention over the 8-bit cache works in: decoding on takes no more of it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,HQ,H,HD,T", [(1, 20, 20, 64, 1), (1, 8, 2, 128, 3), (3, 2, 2, 64, 1), (1, 2, 1, 256, 6)])
def test_a_growing_cache_allocates_nothing(pkg, S, HQ, H, HD, T):
    """From the first token on, an appended token and a query over all that is there find their memory in the pool."""
    ctx = pkg.CudaContext(0)
    c = ctx.kvCache8(S, 1200, H, HD)
    qkv = ctx.upload(np.ones((S * T, (HQ + 2 * H) * HD), np.float32), S * T, (HQ + 2 * H) * HD)
    q = ctx.upload(np.ones((S * T, HQ * HD), np.float32), S * T, HQ * HD)

    def token(n):
        for t in (ctx.attnAppendKv8(qkv, c, HQ, n), ctx.attnKv8(q, c, HQ, n + T)):
            ctx.freeTensor(t)

    token(0)
    before = ctx.memStats()
    for n in range(T, 1200 - T, 31):
        token(n)
    ctx.sync()
    after = ctx.memStats()
    assert (after["created"], after["poolBytes"]) == (before["created"], before["poolBytes"])
    ctx.destroy()
