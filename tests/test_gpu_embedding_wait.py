"""GPU: the wait of the blocks that finish a row of the embedding's gradient, made to run out: the rows whose tokens lie
in one block's piece are added, the others are as they were, status bit 0x10 is set, and the next call is right."""
import ctypes as C

import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import _lib as L
from ancora_cutile_b200.kernels import embedding_grad, embedding_grad_workspace
from oracle import embed_ref

pytestmark = pytest.mark.gpu


def _run_out(ctx, dy, ids, dw, T, V, D, work, nbytes=None, polls=200):
    return L.lib().anc_embedding_wait_selftest(ctx.handle, dy.ptr, ids.ptr, dw.ptr, T, V, D, work.ptr,
                                               work.nbytes if nbytes is None else nbytes, polls, None)


@pytest.mark.parametrize("T", [3000, 9000])                        # the counted list and the sorted one
@pytest.mark.parametrize("D", [8, 77, 1024, 1304])
def test_the_wait_runs_out(ctx, D, T):
    """The list runs from the last row of the table down: row 9 with five tokens lies in the first piece, row 5 with all
    others but the padding spans pieces of any length used.  Small whole numbers: float32 sums are exact."""
    V, rng = 10, np.random.default_rng(D + T)
    ids = np.full(T, 5, np.int64)
    ids[rng.permutation(T)[:5]] = 9
    ids[ids == 5] = np.where(rng.random((ids == 5).sum()) < 0.05, -1, 5)
    dy = rng.integers(-8, 9, (T, D)).astype(np.float32)
    base = rng.integers(-8, 9, (V, D)).astype(np.float32)
    d_dy, d_ids, d_dw = anc.DBuf(dy, ctx), anc.DBuf(ids, ctx), anc.DBuf(base, ctx)
    work = anc.DBuf.empty((embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    want = embed_ref.grad(dy, ids, V, 1.0, base)[0].astype(np.float32)
    ctx.sync()
    assert ctx.status() == 0
    for _ in range(2):
        d_dw.upload(base)
        L.check(_run_out(ctx, d_dy, d_ids, d_dw, T, V, D, work))
        ctx.sync()
        assert ctx.status() == 0x10
        got = d_dw.to_numpy()
        assert np.array_equal(got[9], want[9])
        assert np.array_equal(got[:9], base[:9])
    assert ctx.status() == 0
    d_dw.upload(base)
    embedding_grad(d_dy, d_ids, d_dw, T, V, D, work, dy_dtype="f32", dw_dtype="f32", mode="add", ctx=ctx)
    ctx.sync()
    assert np.array_equal(d_dw.to_numpy(), want)
    assert ctx.status() == 0
    for b in (d_dy, d_ids, d_dw, work):
        b.free()


def test_refusals(ctx):
    T, V, D = 200, 10, 8
    d_dy, d_ids = anc.DBuf.zeros((T, D), np.float32, ctx), anc.DBuf.zeros((T,), np.int64, ctx)
    d_dw = anc.DBuf.zeros((V, D), np.float32, ctx)
    work = anc.DBuf.empty((embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    for kw in (dict(polls=0), dict(polls=(1 << 14) + 1), dict(nbytes=16), dict(V=0)):
        kw = dict(dict(T=T, V=V, D=D), **kw)
        assert _run_out(ctx, d_dy, d_ids, d_dw, kw.pop("T"), kw.pop("V"), kw.pop("D"), work, **kw) == L.E_INVALID
    assert L.lib().anc_embedding_wait_selftest(None, None, None, None, 1, 1, 8, None, C.c_uint64(0), C.c_uint32(5),
                                               None) == L.E_INVALID
    for b in (d_dy, d_ids, d_dw, work):
        b.free()
