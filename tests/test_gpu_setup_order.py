"""GPU: what a constructor clears or uploads is there before the first launch on a stream that does not wait for the
legacy stream, however busy that one is."""
import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import _lib as L

pytestmark = pytest.mark.gpu
LEGACY = 1                     # cudaStreamLegacy, the legacy default stream's own handle


@pytest.fixture
def busy(ctx):
    """Call it to queue some ten milliseconds of copies on the legacy stream."""
    n = 512 << 20
    a, b = anc.DBuf.zeros((n,), np.uint8, ctx), anc.DBuf.zeros((n,), np.uint8, ctx)

    def queue():
        for _ in range(60):
            L.check(L.lib().anc_d2d(ctx.handle, b.ptr, a.ptr, n, LEGACY))
    yield queue
    L.check(L.lib().anc_ctx_sync(ctx.handle, LEGACY))
    a.free()
    b.free()


@pytest.mark.parametrize("n", [0, 1, 5000, 3_000_000])
def test_clip_plan_is_ready_when_it_is_returned(ctx, busy, n):
    host = np.random.default_rng(n).standard_normal(n).astype(np.float32)
    d = anc.DBuf(host, ctx)
    junk = [anc.DBuf(np.full(k, 0xFF, np.uint8), ctx) for k in (512, 1024, 4096)]      # what the allocator may hand out
    for j in junk:
        j.free()
    busy()
    clip = anc.GradClip([dict(g=d, numel=n)], grad_dtype="f32", ctx=ctx)
    clip.norm(1.0)                                                 # on the context's stream
    norm, factor = clip.read()
    want = float(np.sqrt(np.sum(host.astype(np.float64) ** 2)))
    assert abs(norm - want) <= 6 * 2.0 ** -24 * want
    assert abs(factor - min(1.0, 1.0 / (want + 1e-6))) <= 6 * 2.0 ** -24
    clip.free()
    d.free()
    assert ctx.status() == 0


def test_a_new_context_does_not_clear_the_first_launchs_status(ctx, busy):
    table, ids = anc.DBuf.zeros((4, 8), np.uint16, ctx), anc.DBuf(np.array([9, 1], np.int64), ctx)
    out = anc.DBuf.zeros((2, 8), np.uint16, ctx)
    busy()
    other = anc.Context(ctx.device)
    anc.kernels.embedding_lookup(table, ids, out, 2, 4, 8, ctx=other)                  # id 9 of a table of 4 rows
    L.check(L.lib().anc_ctx_sync(ctx.handle, LEGACY))
    assert other.status() == 0x8
    assert other.status() == 0
    for x in (table, ids, out):
        x.free()
    other.destroy()
