"""CPU: what the gradient norm, clipping and embedding entry points refuse (every check comes before the first
CUDA call and before the context is read), workspace sizes, and the float64 oracles against plain formulas."""
import ctypes as C
import math

import numpy as np
import pytest

from ancora_cutile_b200 import _lib as L, kernels
from oracle import clip_ref, embed_ref

FAKE = C.c_void_p(4096)        # stands for a context or a device buffer; never read


def _clip_plan(tensors, grad=L.GRAD_BF16, out=L.GRAD_BF16, result=None, ctx=FAKE):
    arr = (L.ClipTensor * max(len(tensors), 1))(*[L.ClipTensor(*t) for t in tensors])
    h = C.c_void_p()
    return L.lib().anc_clip_plan_create(ctx, arr, len(tensors), grad, out, result, C.byref(h)), h


@pytest.mark.parametrize("tensors,kw,msg", [
    ([(None, None, 8)], {}, b"NULL pointer"),
    ([(4097, None, 8)], {}, b"aligned"),
    ([(4098, None, 8)], dict(grad=L.GRAD_F32, out=L.GRAD_F32), b"aligned"),
    ([(4096, 8193, 8)], {}, b"aligned"),
    ([(4096, None, 8)], dict(grad=L.GRAD_F32), b"in place"),
    ([(4096, None, 8)], dict(grad=2), b"grad_dtype"),
    ([(4096, 8192, 8)], dict(out=-1), b"out_dtype"),
    ([(4096, None, 8)], dict(result=4098), b"result"),
    ([(4096, None, 8)], dict(ctx=None), b"NULL"),
    # an output that lies partly over its own or another tensor's gradient would change the norm's input
    ([(4096, 4112, 64)], {}, b"overlap"),
    ([(4096, 8192, 64), (8200, 16384, 64)], {}, b"overlap"),
    ([(4096, 8192, 64), (16384, 8256, 64)], {}, b"overlap"),
    ([(4096, None, 64), (4160, None, 64)], {}, b"overlap"),
    ([(4096, 8192, 64)], dict(result=8192), b"overlap"),
    ([(4096, 8192, 64)], dict(result=4220), b"overlap"),
    ([(4096, None, (1 << 63))], {}, b"numel"),
])
def test_clip_plan_refusals(tensors, kw, msg):
    rc, h = _clip_plan(tensors, **kw)
    assert rc == L.E_INVALID and h.value is None
    assert msg in L.lib().anc_last_error(), L.lib().anc_last_error()


def test_clip_calls_refuse_a_missing_plan():
    l = L.lib()
    assert l.anc_grad_norm(None, 1.0, 1.0, 1e-6, None) == L.E_INVALID
    assert l.anc_grad_clip(None, 1.0, 1.0, 1e-6, None) == L.E_INVALID
    assert l.anc_grad_sumsq(None, None) == L.E_INVALID
    assert l.anc_grad_norm_finish(None, 1.0, 1.0, 1e-6, None) == L.E_INVALID
    assert l.anc_grad_apply(None, None) == L.E_INVALID
    assert l.anc_clip_plan_result(None, None, None) == L.E_INVALID
    assert l.anc_clip_plan_destroy(None) == 0


@pytest.mark.parametrize("scale,max_norm,eps", [
    (0.0, 1.0, 1e-6), (-1.0, 1.0, 1e-6), (math.nan, 1.0, 1e-6), (math.inf, 1.0, 1e-6),
    (1.0, -0.5, 1e-6), (1.0, math.nan, 1e-6), (1.0, 1.0, -1e-6), (1.0, 1.0, math.nan), (1.0, 1.0, math.inf)])
def test_clip_scalars_refused(scale, max_norm, eps):
    # the scalars are looked at before the plan's contents
    l = L.lib()
    for f in (l.anc_grad_norm, l.anc_grad_clip, l.anc_grad_norm_finish):
        assert f(FAKE, scale, max_norm, eps, None) == L.E_INVALID


def _lookup(ctx=FAKE, table=4096, td=0, tld=0, ids=1 << 20, idt=L.IDS_I64, out=1 << 21, od=0, old=0, T=4, V=10, D=8,
            scale=1.0):
    return L.lib().anc_embedding_lookup(ctx, table, td, tld, ids, idt, out, od, old, T, V, D, scale, None)


@pytest.mark.parametrize("kw", [
    dict(out=4096), dict(out=4098), dict(out=1 << 21, ids=(1 << 21) + 8),
    dict(ctx=None), dict(table=None), dict(ids=None), dict(out=None), dict(td=3), dict(od=-1), dict(idt=2),
    dict(table=4097), dict(out=4098, od=1), dict(ids=4100), dict(ids=4098, idt=L.IDS_I32), dict(tld=7), dict(old=7),
    dict(T=-1), dict(T=1 << 31), dict(V=0), dict(V=(1 << 31) - 1), dict(D=0), dict(D=(1 << 24) + 1),
    dict(scale=math.nan), dict(scale=math.inf)])
def test_lookup_refusals(kw):
    assert _lookup(**kw) == L.E_INVALID


def test_lookup_of_no_tokens_is_nothing():
    assert _lookup(T=0, table=None, ids=None, out=None) == 0


def _grad(ctx=FAKE, dy=4096, yd=0, yld=0, ids=1 << 21, idt=L.IDS_I64, dw=1 << 20, wd=0, wld=0, T=4, V=10, D=8, scale=1.0,
          mode=L.EMBED_ADD, pad=-1, work=1 << 24, wb=1 << 30):
    return L.lib().anc_embedding_grad(ctx, dy, yd, yld, ids, idt, dw, wd, wld, T, V, D, scale, mode, pad, work, wb, None)


@pytest.mark.parametrize("kw", [
    dict(dw=4096), dict(dw=8192, dy=8240), dict(dw=8192, ids=8248), dict(dw=1 << 20, work=(1 << 20) - 256),
    dict(dy=1 << 20, work=(1 << 20) - 256), dict(work=(1 << 21) - 256), dict(work=1 << 21),
    dict(ctx=None), dict(dy=None), dict(ids=None), dict(dw=None), dict(work=None), dict(work=(1 << 24) + 8), dict(yd=3),
    dict(wd=-1), dict(idt=2), dict(mode=2), dict(dy=4097), dict(dw=4098, wd=1), dict(ids=4100), dict(yld=7),
    dict(wld=7), dict(T=-1), dict(T=1 << 31), dict(V=0), dict(V=(1 << 31) - 1), dict(D=0), dict(D=(1 << 24) + 1),
    dict(wb=16), dict(scale=math.nan), dict(scale=-math.inf)])
def test_embedding_grad_refusals(kw):
    assert _grad(**kw) == L.E_INVALID


def test_buffers_that_know_their_size_are_held_to_it():
    class Buf:
        def __init__(self, nbytes):
            self.ptr, self.nbytes = 4096, nbytes

    class Ctx:
        handle = FAKE
    ok = dict(table=Buf(10 * 16), ids=Buf(32), out=Buf(64), T=4, V=10, D=8, ctx=Ctx)
    for k, n in (("table", 159), ("ids", 31), ("out", 63)):
        with pytest.raises(ValueError, match=k):
            kernels.embedding_lookup(**dict(ok, **{k: Buf(n)}))
    with pytest.raises(ValueError, match="ids"):               # 32-bit ids taken for 64-bit ones
        kernels.embedding_lookup(**dict(ok, ids=Buf(16)))
    ok = dict(dy=Buf(64), ids=Buf(32), dw=Buf(160), work=4096, T=4, V=10, D=8, ctx=Ctx)
    for k, n in (("dy", 63), ("ids", 31), ("dw", 159)):
        with pytest.raises(ValueError, match=k):
            kernels.embedding_grad(**dict(ok, **{k: Buf(n)}))
    with pytest.raises(ValueError, match="dw"):
        kernels.embedding_grad(**dict(ok, dw_ld=9))


def test_clip_buffers_that_know_their_size_are_held_to_it():
    class Buf:
        def __init__(self, nbytes, ptr):
            self.ptr, self.nbytes = ptr, nbytes

    class Ctx:
        handle = None                       # refused by the library, after the sizes were looked at
    from ancora_cutile_b200 import AncoraError, GradClip
    for g, out, result, what in ((15, 32, 8, "g"), (16, 31, 8, "out"), (16, 32, 7, "result")):
        with pytest.raises(ValueError, match=what):
            GradClip([dict(g=Buf(g, 4096), out=Buf(out, 8192), numel=8)], out_dtype="f32", result=Buf(result, 1 << 14),
                     ctx=Ctx)
    with pytest.raises(AncoraError):
        GradClip([dict(g=Buf(16, 4096), out=Buf(32, 8192), numel=8)], out_dtype="f32", result=Buf(8, 1 << 14), ctx=Ctx)
    with pytest.raises(ValueError, match="numel"):
        GradClip([dict(g=4096, numel=-1)], ctx=Ctx)


def test_default_context_follows_the_selected_device(monkeypatch):
    from ancora_cutile_b200 import buffers
    monkeypatch.setattr(buffers, "_contexts", {d: f"context {d}" for d in range(3)})
    monkeypatch.setattr(buffers, "_default_device", None)
    monkeypatch.delenv("LOCAL_RANK", raising=False)
    assert buffers.get_context() == "context 0"
    monkeypatch.setenv("LOCAL_RANK", "2")
    assert buffers.get_context() == "context 2"
    buffers.set_device(1)
    assert buffers.get_context() == "context 1" and buffers.get_context(0) == "context 0"


def test_adding_no_tokens_is_nothing():
    assert _grad(T=0, dy=None, ids=None, work=None, wb=0) == 0


def test_workspace_sizes_grow_with_the_tokens_and_cover_every_size():
    last = 0
    for T in (0, 1, 31, 255, 256, 257, 4096, 4097, 100001, 1 << 20):
        n = kernels.embedding_grad_workspace(T, 1000, 1024)
        assert n >= max(last, 16 * T) and n > 0
        last = n
    assert L.lib().anc_embedding_grad_workspace(4, 10, 8, None) == L.E_INVALID
    with pytest.raises(RuntimeError):
        kernels.embedding_grad_workspace(4, 0, 8)


def test_clip_oracle():
    g = [np.array([3.0, 0.0]), np.array([4.0])]
    assert clip_ref.norm_and_factor(g, 1.0, eps=0.0) == (5.0, 0.2)
    assert clip_ref.norm_and_factor(g, 10.0, scale=0.5, eps=0.0) == (2.5, 0.5)
    n, f = clip_ref.norm_and_factor([np.array([np.inf])], 1.0)
    assert n == math.inf and f == 0.0
    n, f = clip_ref.norm_and_factor([np.array([np.nan])], 1.0)
    assert math.isnan(n) and math.isnan(f)
    assert clip_ref.norm_and_factor([np.array([np.nan])], math.inf)[1] == 1.0
    assert clip_ref.norm_and_factor([], 1.0) == (0.0, 1.0)


def test_embedding_oracle_gradient_is_the_derivative_of_the_lookup():
    """<c, lookup(W)> is linear in W, so its difference quotient along E is <dW, E> up to rounding of the sums."""
    rng = np.random.default_rng(0)
    V, D, ids = 7, 3, np.array([2, 6, 2, -1, 0, 2])
    c = rng.standard_normal((len(ids), D))
    W, E = (rng.integers(-8, 9, (V, D)).astype(np.float32) for _ in range(2))
    f = lambda w: float((c * embed_ref.lookup(w, ids, 0.5, "f32")).sum())  # noqa: E731
    dw, count, _ = embed_ref.grad(c, ids, V, 0.5)
    assert list(count) == [1, 0, 3, 0, 0, 0, 1]
    assert abs((f(W + E) - f(W - E)) / 2 - float((dw * E).sum())) < 1e-12 * 100


@pytest.mark.parametrize("family", ["dense", "moe"])
@pytest.mark.parametrize("world", [1, 2, 4, 8])
def test_ranks_norm_spans_cover_every_element_once(monkeypatch, world, family):
    """What each rank's norm plan reads: over all ranks every parameter element exactly once, no arena gap."""
    from types import SimpleNamespace

    from ancora_cutile_b200 import resident, shapes as S
    from ancora_cutile_b200.hybrid import muon_names_for
    from ancora_cutile_b200.layout import ArenaLayout
    shp = (S.qwen3_0_6b_shapes(n_layers=5, hidden=256, ffn=768, vocab=1001) if family == "dense" else
           S.moe_family_shapes(n_layers=4, hidden=256, ffn=768, experts=3, expert_ffn=128, vocab=777))
    shp["odd_norm"] = (13,)
    monkeypatch.setattr(resident, "GradClip", lambda ts, **kw: ts)
    a_base, m_base, it = 1 << 20, 1 << 40, 2
    seen = {}
    for rank in range(world):
        lay = ArenaLayout(shp, muon_names_for(shp), rank, world)
        eng = SimpleNamespace(_gdt=np.dtype(np.uint16), adamw_names=lay.adamw_names, owned_range=lay.owned_range,
                              a_off=lay.a_off, a_g=SimpleNamespace(ptr=a_base), m_g=SimpleNamespace(ptr=m_base),
                              groups=lay.groups, rank=rank, grad_dtype="bf16", ctx=None)
        for t in resident.ResidentHybrid._make_clip(eng):
            base = m_base if t["g"] >= m_base else a_base
            lo = (t["g"] - base) // it
            seen.setdefault(base, []).append((lo, lo + t["numel"]))
    offs = {n: (a_base if n in lay.a_off else m_base, lay.a_off.get(n, lay.m_off.get(n, 0))) for n in shp}
    for base in (a_base, m_base):
        got = np.zeros(max(lay.a_padded, lay.m_total), np.int8)
        for lo, hi in seen[base]:
            got[lo:hi] += 1
        want = np.zeros_like(got)
        for n, (b, o) in offs.items():
            if b == base:
                want[o:o + int(np.prod(shp[n]))] += 1
        assert np.array_equal(got, want)
