"""GPU: the optimizer step that clips inside its own sweeps, and the chain lookup -> embedding gradient ->
accumulation -> norm -> clipped step on the engine's arenas.

The factor is one float32 product ahead of arithmetic that is checked elsewhere, so a clipped step on bf16 gradients
equals, bit for bit, an unclipped step on float32 gradients that hold those products."""
import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import kernels, shapes as S
from oracle import adamw_ref, bf16 as obf, clip_ref, embed_ref, grad_ref

pytestmark = pytest.mark.gpu
AKW = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, wd=0.1)
U = 2.0 ** -24


def _shapes():
    return S.qwen3_0_6b_shapes(n_layers=2, hidden=128, q_heads=2, kv_heads=1, head_dim=128, ffn=384, vocab=1001)


def _routing(shp):
    mu = [n for n, s in shp.items() if anc.default_is_muon(n, np.empty((0,) * len(s)))]
    return mu, tuple(n for n, s in shp.items() if len(s) == 1)


def _engine(ctx, params, mu, nd, **kw):
    kw = dict(dict(adamw_kw=AKW, grad_dtype="bf16", rounding="sr", seed=7, schedule=anc.PE_SCHEDULE, ctx=ctx), **kw)
    return anc.ResidentHybrid(params, mu, nd, **kw)


def _state(eng):
    sd = eng.state_dict()
    return {k: sd[k] for k in ("a_p32", "a_m", "a_v", "m_p32", "m_buf", "a_p16", "m_p16")}


def _same(a, b):
    for k in a:
        assert np.array_equal(a[k].view(np.uint8), b[k].view(np.uint8)), k


@pytest.mark.parametrize("scale", [None, 0.37])
@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rounding", ["rne", "sr"])
def test_adamw_scales_the_gradients_it_loads(ctx, rounding, g_dtype, scale):
    """Against the oracle on the scaled gradients, bit for bit; sizes with ragged and unaligned chunks."""
    rng = np.random.default_rng(3)
    sizes, off, arena = [5000, 2048, 13], [8, 5016, 7072], 7200
    f = lambda: rng.standard_normal(arena).astype(np.float32)  # noqa: E731
    p, m, v, g = f(), f() * 1e-2, f() ** 2 * 1e-3, f()
    g = obf.rne_f32(g) if g_dtype == "bf16" else g
    dp, dm, dv = (anc.DBuf(x, ctx) for x in (p, m, v))
    dg, d16 = anc.DBuf(obf.rne_bits(g) if g_dtype == "bf16" else g, ctx), anc.DBuf.zeros((arena,), np.uint16, ctx)
    it = 2 if g_dtype == "bf16" else 4
    opt = anc.ResidentAdamW([dict(g=dg.ptr + o * it, p32=dp.ptr + 4 * o, m=dm.ptr + 4 * o, v=dv.ptr + 4 * o,
                                  p16=d16.ptr + 2 * o, numel=n, elem_offset=o, wd=0.1)
                             for o, n in zip(off, sizes)], grad_dtype=g_dtype, rounding=rounding, seed=5, ctx=ctx)
    ds = anc.DBuf(np.array([9.0, scale or 1.0], np.float32), ctx)
    opt.set_grad_scale(ds.ptr + 4)
    if scale is None:
        opt.set_grad_scale(None)
        ds.upload(np.array([np.nan, np.nan], np.float32))
    opt.step(ctx.stream, 1e-3, 0.9, 0.95, 1e-8, t=4)
    ctx.sync()
    s = adamw_ref.adamw_scalars(1e-3, 0.9, 0.95, 1e-8, 4)
    gs = g * np.float32(scale) if scale is not None else g
    got = [x.to_numpy() for x in (dp, dm, dv, d16)]
    for o, n in zip(off, sizes):
        z = slice(o, o + n)
        want = adamw_ref.adamw_step(p[z].copy(), m[z].copy(), v[z].copy(), gs[z], s, 0.1, rounding, 5, 4, o)
        for a, b in zip(got, want):
            assert np.array_equal(a[z], b)
    opt.free()
    for b in (dp, dm, dv, dg, d16, ds):
        b.free()


@pytest.mark.parametrize("max_norm", [1e-3, 1e9])
def test_clipped_step_equals_a_step_on_the_scaled_gradients(ctx, max_norm):
    shp = _shapes()
    params = S.synthetic_params(shp, seed=0)
    mu, nd = _routing(shp)
    bits = [S.synthetic_grads_bf16(shp, seed=k) for k in (1, 2)]
    eng = _engine(ctx, params, mu, nd, max_grad_norm=max_norm)
    ref = _engine(ctx, params, mu, nd, grad_dtype="f32")
    for g in bits:
        vals = {n: obf.bits_f32(b) for n, b in g.items()}
        eng.upload_grads(g, ctx.stream)
        eng.step(ctx.stream)
        norm, f = eng.grad_norm()
        wn, wf = clip_ref.norm_and_factor(vals.values(), max_norm)
        assert abs(norm - wn) <= 6 * U * wn and abs(f - wf) <= 6 * U * wf
        assert (f == 1.0) == (max_norm > 1)
        ref.upload_grads({n: x * np.float32(f) for n, x in vals.items()}, ctx.stream)
        ref.step(ctx.stream)
        ctx.sync()
    _same(_state(eng), _state(ref))
    eng.free()
    ref.free()
    assert ctx.status() == 0


def test_gaps_of_the_arena_do_not_enter_the_norm(ctx):
    shp = {"embed": (7, 3), "a_norm": (5,), "w": (128, 128)}
    params = S.synthetic_params(shp, seed=0)
    eng = _engine(ctx, params, ["w"], (), max_grad_norm=1.0)
    eng.a_g.upload(np.full(eng.a_padded, 0x7FC0, np.uint16))           # NaN wherever nothing is written
    g = S.synthetic_grads_bf16(shp, seed=1)
    for n in shp:
        eng.grad_view(n).upload(g[n])
    eng.step(ctx.stream)
    norm, _ = eng.grad_norm()
    want, _ = clip_ref.norm_and_factor([obf.bits_f32(x) for x in g.values()], 1.0)
    assert abs(norm - want) <= 6 * U * want
    eng.free()


def test_clipped_step_by_graph_and_by_host_round_trip(ctx):
    """Eager, replayed and pipelined host steps give the same state; changed settings refuse the old graph."""
    shp = _shapes()
    params = S.synthetic_params(shp, seed=2)
    mu, nd = _routing(shp)
    grads = [S.synthetic_grads_bf16(shp, seed=10 + k, std=10.0 ** (-k)) for k in range(4)]
    eager, graph, host = (_engine(ctx, params, mu, nd, max_grad_norm=0.5) for _ in range(3))
    host.host_chunk_elems = 40000                                        # several units
    norms = []
    for k, g in enumerate(grads):
        eager.upload_grads(g, ctx.stream)
        eager.step(ctx.stream)
        norms.append(eager.grad_norm())
        graph.upload_grads(g, ctx.stream)
        if k == 0:
            graph.step(ctx.stream)
            graph.capture_step(ctx.stream, horizon=16)
        else:
            graph.replay_step(ctx.stream)
        assert graph.grad_norm() == norms[-1]
        host.step_host(g, ctx.stream)
        assert host.grad_norm() == norms[-1]
    for g, got in zip(grads, norms):                                     # each of the four is above 0.5
        want = clip_ref.norm_and_factor([obf.bits_f32(b) for b in g.values()], 0.5)
        assert abs(got[0] - want[0]) <= 6 * U * want[0] and abs(got[1] - want[1]) <= 6 * U * want[1]
    ctx.sync()
    _same(_state(eager), _state(graph))
    _same(_state(eager), _state(host))
    graph.max_grad_norm = 0.25
    with pytest.raises(RuntimeError, match="capture again"):
        graph.replay_step(ctx.stream)
    graph.max_grad_norm = None
    with pytest.raises(RuntimeError, match="capture again"):
        graph.replay_step(ctx.stream)
    # and without clipping the engine is what it was
    plain = _engine(ctx, params, mu, nd)
    plain.load_state_dict(graph.state_dict())
    for e in (plain, graph):
        e.upload_grads(grads[0], ctx.stream)
        e.step(ctx.stream)
    ctx.sync()
    _same(_state(plain), _state(graph))
    for e in (eager, graph, host, plain):
        e.free()
    assert ctx.status() == 0


def test_hybrid_optimizer_clips_and_refuses_half_steps(ctx):
    shp = _shapes()
    params = S.synthetic_params(shp, seed=4)
    rng = np.random.default_rng(5)
    grads = {n: rng.standard_normal(s).astype(np.float32) for n, s in shp.items()}
    opt = anc.HybridOptimizer(params, adamw_kw=AKW, max_grad_norm=1.0, ctx=ctx)
    opt.step(grads)
    norm, f = opt.grad_norm()
    wn, wf = clip_ref.norm_and_factor(grads.values(), 1.0)
    assert abs(norm - wn) <= 6 * U * wn and abs(f - wf) <= 6 * U * wf
    ref = anc.HybridOptimizer(params, adamw_kw=AKW, ctx=ctx)
    ref.step({n: g * np.float32(f) for n, g in grads.items()})
    a, b = opt.master(), ref.master()
    for n in shp:
        assert np.array_equal(a[n], b[n]), n
    with pytest.raises(RuntimeError, match="norm of all gradients"):
        opt.adamw.step({n: grads[n] for n in opt.adamw_names})
    opt.max_grad_norm = None
    opt.muon.step({n: grads[n] for n in opt.muon_names})
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            opt.max_grad_norm = bad
    assert opt.max_grad_norm is None
    opt.free()
    ref.free()


def test_sharded_engine_without_a_communicator_is_refused(ctx):
    shp = _shapes()
    params = S.synthetic_params(shp, seed=0)
    mu, nd = _routing(shp)
    with pytest.raises(ValueError, match="communicator"):
        _engine(ctx, params, mu, nd, rank=1, world=2, max_grad_norm=1.0)


def test_nccl_sum_of_squares_over_one_rank(ctx):
    """The sharded path's calls (sum of squares, all-reduce, finish) on a communicator of one rank."""
    from ancora_cutile_b200.zero1 import Comm, nccl_unique_id
    host = np.random.default_rng(0).standard_normal(5000).astype(np.float32)
    d = anc.DBuf(host, ctx)
    clip = anc.GradClip([dict(g=d, numel=5000)], grad_dtype="f32", ctx=ctx)
    comm = Comm(ctx, nccl_unique_id(), 0, 1)
    clip.sumsq(ctx.stream)
    comm.allreduce_f64(clip.sumsq_ptr, 1, ctx.stream)
    clip.finish(2.0, stream=ctx.stream)
    got = clip.read(ctx.stream)
    clip.norm(2.0, stream=ctx.stream)
    assert got == clip.read(ctx.stream)
    comm.destroy()
    clip.free()
    d.free()


def test_lookup_to_clipped_step(ctx):
    """Two micro-batches of a tied embedding: the lookup reads the step's bf16 rows; the head's gradient lies in the
    gradient arena, the embedding's is added straight into the float32 accumulator; the sum is rounded, its
    norm clips, the step runs.  Everything is compared with the oracle from the same inputs."""
    shp = _shapes()
    V, D = shp["embed"]
    params = S.synthetic_params(shp, seed=6)
    mu, nd = _routing(shp)
    eng = _engine(ctx, params, mu, nd, rounding="rne", max_grad_norm=0.05)
    eng.enable_grad_accumulation()
    rng = np.random.default_rng(7)
    T, scale = 700, float(np.float32(D ** 0.5))
    acc = {n: np.zeros(int(np.prod(s)), np.float32) for n, s in shp.items()}
    w16 = obf.bits_f32(obf.rne_bits(params["embed"]))
    d_out = anc.DBuf.zeros((T, D), np.uint16, ctx)
    for k in range(2):
        ids = rng.integers(-1, V, T)
        ids[:300] = 11                                             # one frequent token
        di = anc.DBuf(ids, ctx)
        eng.embedding_lookup("embed", di, d_out, T, scale=scale)
        ctx.sync()
        assert np.array_equal(d_out.to_numpy(), embed_ref.lookup(w16, ids, scale, "bf16"))
        # gradients of the same few magnitudes, whole multiples of 2^-14: every float32 sum is exact
        grads = {n: obf.rne_bits(rng.integers(-8, 9, s) * 2.0 ** -14) for n, s in shp.items()}
        dy = (rng.integers(-8, 9, (T, D)) * 2.0 ** -14).astype(np.float32)
        d_dy = anc.DBuf(obf.rne_bits(dy), ctx)
        eng.embedding_grad("embed", d_dy, di, T, scale=0.5, mode="add", into="acc")
        eng.upload_grads(grads, ctx.stream)
        acc["embed"] += embed_ref.grad(dy, ids, V, 0.5)[0].astype(np.float32).reshape(-1)
        for n in shp:
            acc[n] = grad_ref.grad_accumulate(acc[n], grads[n].reshape(-1), want_g16=False)[0]
        if k == 0:
            eng.accumulate_grads(ctx.stream)
        else:
            eng.finalize_grads(ctx.stream, rounding="rne")
        ctx.sync()
        di.free()
        d_dy.free()
    g16 = {n: grad_ref.grad_accumulate(acc[n], None, scale=0.5)[1].reshape(shp[n]) for n in shp}
    for n in shp:
        assert np.array_equal(eng.grad_view(n).to_numpy(), g16[n]), n
    eng.step(ctx.stream)
    norm, f = eng.grad_norm()
    vals = {n: obf.bits_f32(b) for n, b in g16.items()}
    wn, wf = clip_ref.norm_and_factor(vals.values(), 0.05)
    assert abs(norm - wn) <= 6 * U * wn and abs(f - wf) <= 6 * U * wf and f < 1.0
    s = adamw_ref.adamw_scalars(AKW["lr"], *AKW["betas"], AKW["eps"], 1)
    master = eng.master()
    for n in eng.adamw_names:
        p = params[n].reshape(-1)
        z = np.zeros_like(p)
        want = adamw_ref.adamw_step(p, z, z, vals[n].reshape(-1) * np.float32(f), s, 0.0 if n in nd else AKW["wd"],
                                    "rne", 7, 1, eng.a_off[n])
        assert np.array_equal(master[n][2], want[0]), n
    # the next lookup reads the rows the step wrote
    w16 = obf.bits_f32(obf.rne_bits(master["embed"][2].reshape(V, D)))
    di = anc.DBuf(np.arange(T, dtype=np.int32), ctx)
    eng.embedding_lookup("embed", di, d_out, T, ids_dtype="i32")
    ctx.sync()
    assert np.array_equal(d_out.to_numpy(), embed_ref.lookup(w16, np.arange(T), 1.0, "bf16"))
    with pytest.raises(ValueError):
        eng.embedding_grad("embed", d_out, di, T, ids_dtype="i32", into="acc")
    with pytest.raises(ValueError):
        eng.embedding_lookup("final_norm", di, d_out, T)
    di.free()
    d_out.free()
    eng.free()
    assert ctx.status() == 0
