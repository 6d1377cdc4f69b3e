"""GPU: embedding lookup and its gradient by sorted tokens.

Lookup: one float32 product and one rounding per element, so it equals numpy bit for bit.

Gradient: with u = 2^-24, a float32 sum of n terms in any order is off by at most (n - 1) u / (1 - n u) times the
sum of the absolute values M (n u < 0.02 here, so 1.02 n u M covers it); the product by the scale adds u |S|,
the sum with the old value u |result|, and the rounding to the output type half a step, e = 2^-8 (bf16) or u
relative plus half the smallest denormal.  Where all values are small integers every sum is exact and float32 results
must be equal."""
import ctypes as C

import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import _lib as L, kernels
from oracle import bf16 as obf, embed_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _dev(ctx, x, dtype):
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        b = obf.rne_bits(x)
        return anc.DBuf(b, ctx), obf.bits_f32(b)
    return anc.DBuf(x, ctx), x


def _values(buf, dtype):
    x = buf.to_numpy()
    return obf.bits_f32(x) if dtype == "bf16" else x


def _ids(rng, T, V, kind):
    if kind == "one row":
        return np.full(T, V // 2, np.int64)
    if kind == "distinct":
        return rng.permutation(max(T, V))[:T].astype(np.int64) % V
    ids = (np.exp(rng.random(T) * np.log(V + 1)).astype(np.int64) - 1).clip(0, V - 1)
    ids = ids * 7 % V
    if kind == "padded" and T:
        ids[rng.random(T) < 0.3] = -1
        ids[T - T // 5:] = -100
    if kind == "all padding":
        ids[:] = -1
    return ids


LOOKUPS = [(1, 1, 1), (1, 5, 8), (3, 100, 7), (5, 100, 24), (17, 300, 256), (9, 50, 257), (300, 1000, 264),
           (1000, 2000, 1024), (33, 64, 1500), (2, 9, 5000)]


@pytest.mark.parametrize("shape", LOOKUPS)
@pytest.mark.parametrize("table_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
def test_lookup_bit_exact(ctx, shape, table_dtype, out_dtype):
    T, V, D = shape
    rng = np.random.default_rng(T * 31 + D)
    w = rng.standard_normal((V, D)).astype(np.float32)
    w[0, 0] = np.inf
    w[-1, -1] = 1e-40
    table, vals = _dev(ctx, w, table_dtype)
    for ids_dtype, scale in (("i64", 1.0), ("i32", np.float32(np.sqrt(D)))):
        ids = _ids(rng, T, V, "padded" if T > 1 else "distinct")
        di = anc.DBuf(ids.astype(np.int64 if ids_dtype == "i64" else np.int32), ctx)
        out = anc.DBuf(np.full((T + 1, D), 0x1234 if out_dtype == "bf16" else 9,
                               np.uint16 if out_dtype == "bf16" else np.float32), ctx)
        kernels.embedding_lookup(table, di, out, T, V, D, scale=float(scale), table_dtype=table_dtype,
                                 out_dtype=out_dtype, ids_dtype=ids_dtype, ctx=ctx)
        ctx.sync()
        got = out.to_numpy()
        want = embed_ref.lookup(vals, ids, scale, out_dtype)
        assert np.array_equal(got[:T].view(np.uint16), want.view(np.uint16))
        assert (got[T] == (0x1234 if out_dtype == "bf16" else 9)).all()        # the row behind is left alone
        di.free()
        out.free()
    assert ctx.status() == 0
    table.free()


@pytest.mark.parametrize("offset,table_ld,out_ld", [(0, 40, 48), (1, 33, 41), (8, 64, 32), (3, 32, 40)])
def test_lookup_strides_and_unaligned_starts(ctx, offset, table_ld, out_ld):
    T, V, D = 70, 20, 32
    rng = np.random.default_rng(offset)
    w = obf.rne_bits(rng.standard_normal(V * table_ld + 16))
    table, ids = anc.DBuf(w, ctx), rng.integers(0, V, T)
    di = anc.DBuf(ids, ctx)
    out = anc.DBuf(np.full(T * out_ld + 16, 7, np.uint16), ctx)
    kernels.embedding_lookup(table.ptr + 2 * offset, di, out.ptr + 2 * offset, T, V, D, table_ld=table_ld, out_ld=out_ld,
                             ctx=ctx)
    ctx.sync()
    want = np.full(T * out_ld + 16, 7, np.uint16)
    for t in range(T):
        src = offset + ids[t] * table_ld
        want[offset + t * out_ld:offset + t * out_ld + D] = w[src:src + D]
    assert np.array_equal(out.to_numpy(), want)
    for b in (table, di, out):
        b.free()


def test_ids_outside_the_table_are_reported_and_touch_nothing(ctx):
    V, D = 50, 16
    rng = np.random.default_rng(0)
    w, vals = _dev(ctx, rng.standard_normal((V, D)), "f32")
    for ids in ([3, V, 4], [2 ** 31, 0, 1], [-1, -2 ** 40, 2 ** 62]):
        ids = np.array(ids, np.int64)
        di, out = anc.DBuf(ids, ctx), anc.DBuf(np.full((3, D), 5, np.float32), ctx)
        kernels.embedding_lookup(w, di, out, 3, V, D, table_dtype="f32", out_dtype="f32", ctx=ctx)
        ctx.sync()
        assert np.array_equal(out.to_numpy(), embed_ref.lookup(vals, ids, 1.0, "f32"))
        expect = 0x8 if (ids >= V).any() else 0
        assert ctx.status() == expect
        work = anc.DBuf.empty((kernels.embedding_grad_workspace(3, V, D),), np.uint8, ctx)
        dw = anc.DBuf(np.full((V, D), 2, np.float32), ctx)
        kernels.embedding_grad(out, di, dw, 3, V, D, work, dy_dtype="f32", dw_dtype="f32", mode="add", ctx=ctx)
        ctx.sync()
        # one token per row at most: a single float32 sum, the rounded float64 one
        want = embed_ref.grad(out.to_numpy(), ids, V, 1.0, np.full((V, D), 2.0))[0].astype(np.float32)
        assert np.array_equal(dw.to_numpy(), want)
        assert ctx.status() == expect
        for b in (di, out, work, dw):
            b.free()
    w.free()


@pytest.mark.parametrize("T", [500, 5000])
@pytest.mark.parametrize("mode", ["write", "add"])
def test_long_lists_with_ids_outside_the_table(ctx, T, mode):
    V, D = 70, 24
    rng = np.random.default_rng(T)
    ids = rng.integers(-3, V, T)
    ids[[0, 77, T - 1]] = V, 2 ** 40, V + 1
    dy = rng.integers(-8, 9, (T, D)).astype(np.float32)
    dy[(ids < 0) | (ids >= V)] = np.nan                    # rows of no id are not read
    old = rng.integers(-8, 9, (V, D)).astype(np.float32)
    got, _, _, _ = _run_grad(ctx, dy, ids, V, 1.0, "f32", "f32", mode, old)
    assert np.array_equal(got, embed_ref.grad(dy, ids, V, 1.0, old if mode == "add" else None)[0].astype(np.float32))
    assert ctx.status() == 0x8


def _run_grad(ctx, dy, ids, V, scale, dy_dtype, dw_dtype, mode, old, padding_idx=None, ids_dtype="i64"):
    T, D = dy.shape
    d_dy, dyv = _dev(ctx, dy, dy_dtype)
    d_ids = anc.DBuf(ids.astype(np.int64 if ids_dtype == "i64" else np.int32), ctx)
    d_dw, oldv = _dev(ctx, old, dw_dtype)
    work = anc.DBuf.empty((kernels.embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    kernels.embedding_grad(d_dy, d_ids, d_dw, T, V, D, work, scale=scale, dy_dtype=dy_dtype, dw_dtype=dw_dtype,
                           mode=mode, padding_idx=padding_idx, ids_dtype=ids_dtype, ctx=ctx)
    ctx.sync()
    bits = d_dw.to_numpy()
    got = _values(d_dw, dw_dtype)
    for b in (d_dy, d_ids, d_dw, work):
        b.free()
    return got, bits, dyv, oldv


def _check_grad(got, dyv, oldv, ids, V, scale, dw_dtype, mode, padding_idx=None):
    want, count, mag = embed_ref.grad(dyv, ids, V, scale, oldv if mode == "add" else None, padding_idx)
    half = 2.0 ** -8 if dw_dtype == "bf16" else U
    tiny = 2.0 ** -134 if dw_dtype == "bf16" else 2.0 ** -150
    assert count.max(initial=0) * U < 0.02
    err = 1.02 * count[:, None] * U * mag + 2 * U * (np.abs(want) + mag)
    tol = err + half * (np.abs(want) + err) + tiny
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= tol).all(), (off.max(), np.unravel_index((off - tol).argmax(), off.shape))
    untouched = count == 0
    if mode == "add":
        assert np.array_equal(got[untouched], oldv[untouched])
    else:
        assert not got[untouched].any()


# token counts around a warp's part, a piece, and the sort's cluster sizes; row lengths around the slice and vectors
GRADS = [(0, 10, 8, "zipf"), (1, 1, 1, "zipf"), (1, 7, 8, "zipf"), (2, 5, 3, "one row"), (31, 40, 17, "zipf"),
         (32, 40, 16, "one row"), (33, 4, 256, "zipf"), (255, 100, 257, "padded"), (256, 300, 264, "one row"),
         (257, 64, 1000, "zipf"), (300, 1000, 1024, "distinct"), (513, 2, 72, "zipf"), (1000, 511, 24, "zipf"),
         (1025, 512, 24, "zipf"), (4096, 513, 8, "zipf"), (4097, 5000, 40, "one row"), (8193, 2000, 33, "padded"),
         (20000, 151936, 16, "zipf"), (20000, 262143, 8, "distinct"), (3000, 262144, 8, "zipf"),
         (3000, 300000, 8, "distinct"), (777, 90, 48, "all padding"), (70001, 300, 9, "zipf")]


@pytest.mark.parametrize("case", GRADS, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("dy_dtype,dw_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("mode", ["write", "add"])
def test_gradient(ctx, case, dy_dtype, dw_dtype, mode):
    T, V, D, kind = case
    rng = np.random.default_rng(T + V + D)
    ids = _ids(rng, T, V, kind)
    dy = rng.standard_normal((T, D)).astype(np.float32)
    dy[ids < 0] = np.nan                                   # padded rows are not read
    old = rng.standard_normal((V, D)).astype(np.float32)
    scale = 0.75
    got, _, dyv, oldv = _run_grad(ctx, dy, ids, V, scale, dy_dtype, dw_dtype, mode, old,
                                  ids_dtype="i32" if T % 2 else "i64")
    _check_grad(got, dyv, oldv, ids, V, scale, dw_dtype, mode)
    assert ctx.status() == 0


@pytest.mark.parametrize("T,V,D,kind", [(5000, 37, 130, "zipf"), (40000, 3, 264, "zipf"), (66000, 70000, 24, "padded"),
                                        (300, 20, 2048, "zipf"), (30000, 5, 1024, "zipf"), (9000, 2000, 512, "padded"),
                                        (20000, 9, 1536, "one row"), (200000, 100, 8, "zipf"), (129, 3, 512, "one row")])
def test_integer_gradients_are_exact(ctx, T, V, D, kind):
    rng = np.random.default_rng(T)
    ids = _ids(rng, T, V, kind)
    dy = rng.integers(-8, 9, (T, D)).astype(np.float32)
    old = rng.integers(-100, 101, (V, D)).astype(np.float32)
    for mode in ("write", "add"):
        got, _, _, _ = _run_grad(ctx, dy, ids, V, 2.0, "bf16", "f32", mode, old)
        want, _, _ = embed_ref.grad(dy, ids, V, 2.0, old if mode == "add" else None)
        assert np.array_equal(got, want.astype(np.float32)), mode


def test_the_same_bits_every_time(ctx):
    rng = np.random.default_rng(1)
    T, V, D = 30000, 500, 72
    ids = _ids(rng, T, V, "zipf")
    dy, old = rng.standard_normal((T, D)), rng.standard_normal((V, D))
    runs = [_run_grad(ctx, dy, ids, V, 1.0, "f32", "f32", "add", old)[1] for _ in range(3)]
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


def test_padding_idx_and_special_values(ctx):
    rng = np.random.default_rng(3)
    T, V, D = 600, 30, 40
    ids = _ids(rng, T, V, "zipf")
    dy = rng.standard_normal((T, D)).astype(np.float32)
    old = rng.standard_normal((V, D)).astype(np.float32)
    dy[ids == 0] = np.inf                                  # the padding row's gradients do not reach the table
    got, _, dyv, oldv = _run_grad(ctx, dy, ids, V, 1.0, "f32", "f32", "add", old, padding_idx=0)
    _check_grad(got, np.where((ids == 0)[:, None], 0, dyv), oldv, ids, V, 1.0, "f32", "add", padding_idx=0)
    dy[:] = 1.0
    row = int(ids[5])
    dy[5, 3], dy[5, 4] = np.nan, -np.inf                   # a NaN or infinity stays in its own row and column
    got, _, _, _ = _run_grad(ctx, dy, ids, V, 1.0, "f32", "f32", "write", old)
    assert np.isnan(got[row, 3]) and got[row, 4] == -np.inf
    got[row, 3:5] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("T", [129, 255, 4095, 4096, 4097, 8193])
@pytest.mark.parametrize("V,D", [(260, 40), (32768, 256), (32769, 256), (300000, 128)])
def test_list_by_counting_and_by_sorting(ctx, T, V, D):
    """Sizes on either side of where the list is counted instead of sorted (tokens, and zeros to write): integer
    sums are exact, every row of a written table is defined,."""
    rng = np.random.default_rng(T + V)
    ids = _ids(rng, T, V, "zipf")
    ids[::7] = V - 1 - ids[::7]
    ids[5::11] = -1
    dy = rng.integers(-8, 9, (T, D)).astype(np.float32)
    old = rng.integers(-100, 101, (V, D)).astype(np.float32)
    for mode in ("write", "add"):
        want, _, _ = embed_ref.grad(dy, ids, V, 2.0, old if mode == "add" else None)
        for ids_dtype in ("i32", "i64"):
            got, _, _, _ = _run_grad(ctx, dy, ids, V, 2.0, "bf16", "f32", mode, old, ids_dtype=ids_dtype)
            assert np.array_equal(got, want.astype(np.float32)), (mode, ids_dtype)
    assert ctx.status() == 0


@pytest.mark.parametrize("offset,dy_ld,dw_ld", [(0, 40, 48), (1, 33, 41), (8, 64, 32), (3, 32, 40)])
def test_gradient_strides_leave_the_gaps_alone(ctx, offset, dy_ld, dw_ld):
    T, V, D = 900, 25, 32
    rng = np.random.default_rng(offset)
    ids = _ids(rng, T, V, "padded")
    ids[ids == 7] = 8
    for mode in ("write", "add"):
        flat = rng.integers(-8, 9, T * dy_ld + 16).astype(np.float32)
        old = rng.integers(-8, 9, V * dw_ld + 16).astype(np.float32)
        d_dy, d_dw, di = anc.DBuf(flat, ctx), anc.DBuf(old, ctx), anc.DBuf(ids, ctx)
        work = anc.DBuf.empty((kernels.embedding_grad_workspace(T, V, D),), np.uint8, ctx)
        kernels.embedding_grad(d_dy.ptr + 4 * offset, di, d_dw.ptr + 4 * offset, T, V, D, work, dy_dtype="f32",
                               dw_dtype="f32", mode=mode, dy_ld=dy_ld, dw_ld=dw_ld, ctx=ctx)
        ctx.sync()
        view = lambda a, n, ld: np.lib.stride_tricks.as_strided(a[offset:], (n, D), (4 * ld, 4))  # noqa: E731
        want = old.copy()
        ov = view(want, V, dw_ld)
        ov[:] = embed_ref.grad(view(flat, T, dy_ld), ids, V, 1.0, ov if mode == "add" else None)[0]
        assert np.array_equal(d_dw.to_numpy(), want), mode
        for b in (d_dy, d_dw, di, work):
            b.free()


def test_gradient_is_the_derivative_of_the_lookup(ctx):
    """<c, lookup(W)> is linear in W: its central difference along E equals <dW, E> up to the roundings of the
    lookup (u relative to each output) and of the gradient."""
    rng = np.random.default_rng(5)
    T, V, D, scale = 500, 60, 40, 3.0
    ids = _ids(rng, T, V, "padded")
    W, E, c = (rng.standard_normal(s).astype(np.float32) for s in ((V, D), (V, D), (T, D)))

    def outputs(w):
        dw, di, out = anc.DBuf(w, ctx), anc.DBuf(ids, ctx), anc.DBuf.zeros((T, D), np.float32, ctx)
        kernels.embedding_lookup(dw, di, out, T, V, D, scale=scale, table_dtype="f32", out_dtype="f32", ctx=ctx)
        ctx.sync()
        o = out.to_numpy().astype(np.float64)
        for b in (dw, di, out):
            b.free()
        return o
    Wp, Wm = W + E, W - E                                  # float32 tables; the step is what they differ by
    op, om = outputs(Wp), outputs(Wm)
    diff = float((c * (op - om)).sum())
    got, _, dyv, oldv = _run_grad(ctx, c, ids, V, scale, "f32", "f32", "write", np.zeros((V, D)))
    step = Wp.astype(np.float64) - Wm
    _, count, mag = embed_ref.grad(c, ids, V, scale)
    tol = (U * np.abs(c) * (np.abs(op) + np.abs(om))).sum() + ((count[:, None] + 3) * U * mag * np.abs(step)).sum()
    assert abs(diff - float((got * step).sum())) <= tol


def test_captured_and_replayed_with_new_tokens(ctx):
    """One captured gradient replays with other ids and gradients in the same buffers; two workspaces let two
    streams run at once."""
    rng = np.random.default_rng(9)
    T, V, D = 9000, 800, 72
    d_dy, d_ids = anc.DBuf.zeros((T, D), np.float32, ctx), anc.DBuf.zeros((T,), np.int64, ctx)
    nb = kernels.embedding_grad_workspace(T, V, D)
    works = [anc.DBuf.empty((nb,), np.uint8, ctx) for _ in range(2)]
    dws = [anc.DBuf.zeros((V, D), np.float32, ctx) for _ in range(2)]
    s2 = C.c_void_p()
    L.check(L.lib().anc_stream_create(ctx.handle, C.byref(s2)))
    call = lambda k, st: kernels.embedding_grad(d_dy, d_ids, dws[k], T, V, D, works[k], dy_dtype="f32",  # noqa: E731
                                                dw_dtype="f32", mode="write", stream=st, ctx=ctx)
    L.check(L.lib().anc_graph_begin(ctx.handle, ctx.stream))
    call(0, ctx.stream)
    g = C.c_void_p()
    L.check(L.lib().anc_graph_end(ctx.handle, ctx.stream, C.byref(g)))
    for k in range(3):
        ids = _ids(rng, T, V, "padded" if k else "one row")
        dy = rng.integers(-4, 5, (T, D)).astype(np.float32)
        d_dy.upload(dy)
        d_ids.upload(ids)
        L.check(L.lib().anc_graph_launch(ctx.handle, g, ctx.stream))
        call(1, s2.value)
        ctx.sync()
        ctx.sync(s2.value)
        want = embed_ref.grad(dy, ids, V, 1.0)[0]
        for dw in dws:
            assert np.array_equal(dw.to_numpy(), want)
    L.check(L.lib().anc_graph_destroy(g))
    L.check(L.lib().anc_stream_destroy(ctx.handle, s2))
    for b in [d_dy, d_ids] + works + dws:
        b.free()
    assert ctx.status() == 0


def test_offsets_past_32_bits(ctx):
    """Rows whose byte and element offsets pass 2^31 and 2^32, in the table, the gradient table and dy."""
    V, D, T = 300_000, 8192, 290_000
    rng = np.random.default_rng(2)
    table = anc.DBuf.zeros((V, D), np.uint16, ctx)                 # 4.9 GB
    rows = np.array([0, 1, 131071, 131072, 262143, 262144, 262145, V - 2, V - 1])
    vals = obf.rne_bits(rng.standard_normal((len(rows), D)))
    for r, v in zip(rows, vals):
        table.slice_elems(int(r) * D, D).upload(v)
    out, di = anc.DBuf.zeros((len(rows), D), np.uint16, ctx), anc.DBuf(rows, ctx)
    kernels.embedding_lookup(table, di, out, len(rows), V, D, ctx=ctx)
    ctx.sync()
    assert np.array_equal(out.to_numpy(), vals)
    # dy: the same memory as T rows, zero but for those; every token of the nonzero rows names a far row
    ids = np.full(T, -1, np.int64)
    ids[::2] = 7
    ids[rows[:-2]] = V - 1 - np.arange(len(rows) - 2) // 2
    dw, d_ids = anc.DBuf.zeros((V, D), np.float32, ctx), anc.DBuf(ids, ctx)      # 9.8 GB
    work = anc.DBuf.empty((kernels.embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    kernels.embedding_grad(table, d_ids, dw, T, V, D, work, dw_dtype="f32", mode="add", ctx=ctx)
    ctx.sync()
    want = np.zeros((8, D))
    for k, v in enumerate(vals[:-2]):
        want[k // 2] += obf.bits_f32(v)
    for k in range(8):
        got = dw.slice_elems((V - 1 - k) * D, D).to_numpy()
        assert np.abs(got - want[k]).max() <= 4 * U * 8, k                       # sums of at most two terms below 8
    assert not dw.slice_elems(7 * D, D).to_numpy().any()
    assert ctx.status() == 0
    for b in (table, out, di, dw, d_ids, work):
        b.free()


def test_table_of_many_short_rows(ctx):
    """Four sort passes (ids of 28 bits)."""
    V, D, T = 150_000_001, 1, 5000
    rng = np.random.default_rng(4)
    ids = rng.integers(0, V, T)
    ids[:1000] = ids[1000:2000]
    ids[2000:2500] = V - 1
    dy = rng.integers(-8, 9, (T, D)).astype(np.float32)
    dw, d_ids, d_dy = anc.DBuf.zeros((V,), np.float32, ctx), anc.DBuf(ids, ctx), anc.DBuf(dy, ctx)
    work = anc.DBuf.empty((kernels.embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    kernels.embedding_grad(d_dy, d_ids, dw, T, V, D, work, dy_dtype="f32", dw_dtype="f32", mode="add", ctx=ctx)
    ctx.sync()
    got = dw.to_numpy()
    want = np.zeros(V, np.float32)
    np.add.at(want, ids, dy[:, 0])
    assert np.array_equal(got, want)
    for b in (dw, d_ids, d_dy, work):
        b.free()
