"""GPU: rows without a token.  The lookup's rows of padding are zero whatever the sign of the scale, and ids that
count as padding leave no gradient on any of the ways the list of tokens is made."""
import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200.kernels import embedding_grad, embedding_grad_workspace, embedding_lookup
from oracle import bf16 as obf, embed_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("w_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [8, 77, 1024, 1303])
@pytest.mark.parametrize("scale", [-1.5, -0.0])
def test_lookup_with_a_negative_scale(ctx, scale, D, w_dtype, out_dtype):
    """Bit for bit, signs of zeros included."""
    rng = np.random.default_rng(D)
    T, V = 45, 30
    table = rng.standard_normal((V, D)).astype(np.float32)
    table[3] = 0.0
    table[4] = -0.0
    ids = rng.integers(-1, V + 1, T)
    ids[:4] = (-1, V, 3, 4)
    bits = obf.rne_bits(table)
    d_w = anc.DBuf(bits if w_dtype == "bf16" else table, ctx)
    d_i = anc.DBuf(ids, ctx)
    d_o = anc.DBuf(np.full((T, D), 0x7ABC, np.uint16) if out_dtype == "bf16" else np.full((T, D), 7.5, np.float32), ctx)
    embedding_lookup(d_w, d_i, d_o, T, V, D, scale=scale, table_dtype=w_dtype, out_dtype=out_dtype, ctx=ctx)
    ctx.sync()
    want = embed_ref.lookup(obf.bits_f32(bits) if w_dtype == "bf16" else table, ids, scale, out_dtype)
    got = d_o.to_numpy()
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    assert ctx.status() == 0x8                                     # the ids at V
    for b in (d_w, d_i, d_o):
        b.free()


@pytest.mark.parametrize("padding_idx", [0, 17, 39])
@pytest.mark.parametrize("mode", ["write", "add"])
@pytest.mark.parametrize("T", [100, 600, 9000])
def test_padding_idx_on_every_way_the_list_is_made(ctx, T, mode, padding_idx):
    """Up to 128 tokens, up to 4096, and above; the row of padding_idx gets nothing, also with NaN in its tokens'
    gradients.  Whole multiples of 2^-7 below 2^16 in sum: every float32 sum is exact."""
    V, D = 40, 24
    rng = np.random.default_rng(T + padding_idx)
    ids = rng.integers(-1, V + 1, T)
    ids[:6] = (padding_idx, -1, V, padding_idx, 39, 0)
    dy = (rng.integers(-8, 9, (T, D)) * 2.0 ** -7).astype(np.float32)
    base = (rng.integers(-8, 9, (V, D)) * 2.0 ** -7).astype(np.float32)
    want = embed_ref.grad(dy, ids, V, -0.5, base if mode == "add" else None, padding_idx)[0].astype(np.float32)
    dy[(ids < 0) | (ids >= V) | (ids == padding_idx)] = np.nan
    d_dy, d_i, d_dw = anc.DBuf(dy, ctx), anc.DBuf(ids, ctx), anc.DBuf(base, ctx)
    work = anc.DBuf.empty((embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    embedding_grad(d_dy, d_i, d_dw, T, V, D, work, scale=-0.5, dy_dtype="f32", dw_dtype="f32", mode=mode,
                   padding_idx=padding_idx, ctx=ctx)
    ctx.sync()
    assert np.array_equal(d_dw.to_numpy(), want)
    assert ctx.status() == 0x8
    for b in (d_dy, d_i, d_dw, work):
        b.free()
