"""GPU: global gradient norm and clipping against the float64 oracle.

Tolerances.  u = 2^-24 is half a float32 step.  A group of eight squares is summed in float32: every term passes
at most eight roundings, all terms are positive, so the group is off by at most 8u relative; the float64 sums above
add nothing visible at this scale; the square root halves that, the result is rounded to float32 once (u): the
norm is within 5u, asserted with 6u.  factor = scale * max_norm / (norm + eps) is computed in float64 from
the unrounded norm and rounded once: the same 5u.  The clipped gradient is one float32 product by the factor
and one rounding, so it equals numpy's float32 evaluation with the device's own factor bit for bit."""
import ctypes as C
import math

import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import _lib as L
from oracle import bf16 as obf, clip_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _dev(ctx, x, dtype):
    """float32 values -> device buffer of the type, and the values it holds."""
    if dtype == "bf16":
        b = obf.rne_bits(x)
        return anc.DBuf(b, ctx), obf.bits_f32(b)
    return anc.DBuf(x.astype(np.float32), ctx), x.astype(np.float32)


def _check_norm(got, want, what=""):
    for g, w in zip(got, want):
        if math.isnan(w):
            assert math.isnan(g), (what, g, w)
        elif math.isinf(w) or w == 0:
            assert g == w, (what, g, w)
        else:
            assert abs(g - w) <= 6 * U * abs(w) + 2.0 ** -149, (what, g, w)


# sizes around the vector (8), the chunk (8192) and several chunks per block; offsets that break 16-byte alignment
SIZES = {
    "one element": [1],
    "below a vector": [7, 3, 1],
    "odd": [8191, 8192, 8193, 17],
    "empty among others": [0, 5, 0, 100000, 0],
    "only empty": [0, 0],
    "none": [],
    "many": [1 + 37 * i for i in range(300)],
    "large": [20_000_003],
}


@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("gap", [1, 64])
@pytest.mark.parametrize("sizes", SIZES)
def test_norm_and_clip(ctx, sizes, gap, g_dtype):
    ns = SIZES[sizes]
    rng = np.random.default_rng(len(sizes) + gap)
    offs, at = [], 3 if gap == 1 else 0
    for n in ns:
        offs.append(at)
        at = -(-(at + n) // gap) * gap
    total = at + 16
    host = (rng.standard_normal(total) * np.exp(rng.uniform(-8, 2))).astype(np.float32)
    d, vals = _dev(ctx, host, g_dtype)
    it = 2 if g_dtype == "bf16" else 4
    parts = [vals[o:o + n] for o, n in zip(offs, ns)]
    for out_dtype in ("bf16", "f32"):
        ot = 2 if out_dtype == "bf16" else 4
        fill = 0x7ABC if out_dtype == "bf16" else np.float32(7.5)
        out = anc.DBuf(np.full(total, fill, np.uint16 if ot == 2 else np.float32), ctx)
        clip = anc.GradClip([dict(g=d.ptr + o * it, numel=n, out=out.ptr + o * ot) for o, n in zip(offs, ns)],
                            grad_dtype=g_dtype, out_dtype=out_dtype, ctx=ctx)
        for max_norm, scale in ((0.5, 1.0), (1e30, 0.25), (math.inf, 1.0), (0.0, 1.0)):
            clip.clip(max_norm, scale=scale)
            got = clip.read()
            _check_norm(got, clip_ref.norm_and_factor(parts, max_norm, scale), (sizes, max_norm))
            want = np.full(total, fill, out.dtype)
            f = np.float32(got[1])
            for o, n, p in zip(offs, ns, parts):
                want[o:o + n] = obf.rne_bits(p * f) if ot == 2 else p * f
            assert np.array_equal(out.to_numpy().view(np.uint16), want.view(np.uint16)), (max_norm, scale)
        first = clip.read()
        clip.clip(0.0)
        assert clip.read()[0] == first[0]                    # the same bits again
        clip.free()
        out.free()
    assert ctx.status() == 0
    d.free()


@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
def test_in_place(ctx, g_dtype):
    rng = np.random.default_rng(2)
    host = rng.standard_normal(70001).astype(np.float32)
    d, vals = _dev(ctx, host, g_dtype)
    it = 2 if g_dtype == "bf16" else 4
    spans = [(5, 40000), (40009, 29990)]
    clip = anc.GradClip([dict(g=d.ptr + o * it, numel=n) for o, n in spans], grad_dtype=g_dtype, ctx=ctx)
    clip.clip(1e9)                                           # above the norm: nothing changes
    assert clip.read()[1] == 1.0
    cur = d.to_numpy()
    assert np.array_equal(cur, obf.rne_bits(host) if it == 2 else host)
    clip.clip(3.0)
    norm, f = clip.read()
    _check_norm((norm, f), clip_ref.norm_and_factor([vals[o:o + n] for o, n in spans], 3.0))
    want = vals.copy()
    for o, n in spans:
        want[o:o + n] *= np.float32(f)
    got = d.to_numpy()
    assert np.array_equal(got, obf.rne_bits(want) if it == 2 else want)
    clip.free()
    d.free()


@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("magnitude", [1e-38, 1e-30, 1e-22, 1e-18, 1e18, 1e30, 2e37])
def test_norm_where_float32_squares_leave_their_range(ctx, magnitude, g_dtype):
    rng = np.random.default_rng(4)
    host = (rng.uniform(0.5, 1.0, 3000) * magnitude).astype(np.float32)
    host[::7] = 0
    host[1::7] *= np.float32(1e-4)
    d, vals = _dev(ctx, host, g_dtype)
    clip = anc.GradClip([dict(g=d, numel=3000)], grad_dtype=g_dtype, ctx=ctx)
    # a float32 tolerance relative to the norm; a norm below the normal range is off by half a denormal step
    clip.norm(math.inf)
    norm, _ = clip.read()
    want, _ = clip_ref.norm_and_factor([vals], math.inf)
    if want >= 2.0 ** 128 * (1 - U / 2):       # half a step above the largest float32: rounds to infinity
        assert norm == math.inf
    else:
        assert abs(norm - want) <= 6 * U * want + 2.0 ** -149
    clip.norm(1.0)                             # the factor comes from the unrounded norm
    _, f = clip.read()
    want_f = clip_ref.norm_and_factor([vals], 1.0)[1]
    assert abs(f - want_f) <= 6 * U * want_f + 2.0 ** -149
    clip.free()
    d.free()


@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", [0, 9, 4096, 99999])
def test_infinities_and_nan(ctx, where, bad, g_dtype):
    host = np.full(100000, 1e-3, np.float32)
    host[where] = bad
    d, vals = _dev(ctx, host, g_dtype)
    o = anc.DBuf.zeros((100000,), np.float32, ctx)
    clip = anc.GradClip([dict(g=d, numel=100000, out=o)], grad_dtype=g_dtype, out_dtype="f32", ctx=ctx)
    clip.clip(1.0)
    norm, f = clip.read()
    got = o.to_numpy()
    if np.isnan(bad):
        assert math.isnan(norm) and math.isnan(f) and np.isnan(got).all()
    else:
        assert norm == math.inf and f == 0.0
        assert np.isnan(got[where]) and not np.delete(got, where).any()
    clip.norm(math.inf, scale=0.5)                           # never clips
    assert clip.read()[1] == 0.5
    clip.free()
    o.free()
    d.free()


def test_halves_add_up_over_shards(ctx):
    """Two shards' sums of squares added by the caller give the whole's norm: what ranks do."""
    rng = np.random.default_rng(6)
    host = rng.standard_normal(50000).astype(np.float32)
    d = anc.DBuf(host, ctx)
    cut = 12345
    a = anc.GradClip([dict(g=d.ptr, numel=cut)], grad_dtype="f32", ctx=ctx)
    b = anc.GradClip([dict(g=d.ptr + 4 * cut, numel=50000 - cut)], grad_dtype="f32", ctx=ctx)
    a.sumsq()
    b.sumsq()
    s = [np.empty(1), np.empty(1)]
    for p, x in zip((a, b), s):
        L.check(L.lib().anc_d2h(ctx.handle, x.ctypes.data, p.sumsq_ptr, 8, None, 1))
    tot = s[0] + s[1]
    for p in (a, b):
        L.check(L.lib().anc_h2d(ctx.handle, p.sumsq_ptr, tot.ctypes.data, 8, None, 1))
        p.finish(2.0, scale=0.5)
    assert a.read() == b.read()
    _check_norm(a.read(), clip_ref.norm_and_factor([host], 2.0, 0.5))
    b.apply()
    f = np.float32(b.read()[1])
    got = d.to_numpy()
    assert np.array_equal(got[cut:], host[cut:] * f) and np.array_equal(got[:cut], host[:cut])
    a.free()
    b.free()
    d.free()


def test_caller_owned_result_two_plans_two_streams_and_a_graph(ctx):
    """Plans on different streams do not share anything; a captured clip replays on new gradients."""
    rng = np.random.default_rng(8)
    n = 3_000_001
    hosts = [rng.standard_normal(n).astype(np.float32) * s for s in (1.0, 30.0)]
    ds = [anc.DBuf(h, ctx) for h in hosts]
    res = anc.DBuf.zeros((4,), np.float32, ctx)
    outs = [anc.DBuf.zeros((n,), np.float32, ctx) for _ in range(2)]
    plans = [anc.GradClip([dict(g=ds[k], numel=n, out=outs[k])], grad_dtype="f32", result=res.ptr + 8 * k, ctx=ctx)
             for k in range(2)]
    s2 = C.c_void_p()
    L.check(L.lib().anc_stream_create(ctx.handle, C.byref(s2)))
    for _ in range(20):
        plans[0].clip(1.0, stream=ctx.stream)
        plans[1].clip(5.0, stream=s2.value)
    ctx.sync()
    ctx.sync(s2.value)
    got = res.to_numpy()
    for k, mx in ((0, 1.0), (1, 5.0)):
        _check_norm(got[2 * k:2 * k + 2].astype(np.float64), clip_ref.norm_and_factor([hosts[k]], mx))
        assert np.array_equal(outs[k].to_numpy(), hosts[k] * got[2 * k + 1])
    L.check(L.lib().anc_graph_begin(ctx.handle, ctx.stream))
    plans[0].clip(1.0, stream=ctx.stream)
    g = C.c_void_p()
    L.check(L.lib().anc_graph_end(ctx.handle, ctx.stream, C.byref(g)))
    for k in range(3):
        h = rng.standard_normal(n).astype(np.float32) * np.float32(10.0 ** (-k))
        ds[0].upload(h)
        L.check(L.lib().anc_graph_launch(ctx.handle, g, ctx.stream))
        ctx.sync()
        r = res.to_numpy()[:2]
        _check_norm(r.astype(np.float64), clip_ref.norm_and_factor([h], 1.0))
        assert np.array_equal(outs[0].to_numpy(), h * r[1])
    L.check(L.lib().anc_graph_destroy(g))
    for p in plans:
        p.free()
    L.check(L.lib().anc_stream_destroy(ctx.handle, s2))
    for b in ds + outs + [res]:
        b.free()
    assert ctx.status() == 0


def _tile(pattern, start, n):
    """n values of the endlessly repeated pattern from place ``start``."""
    i = start % len(pattern)
    return np.resize(np.concatenate([pattern[i:], pattern[:i]]), n)


@pytest.mark.parametrize("g_dtype,in_place", [("bf16", False), ("bf16", True), ("f32", False)])
def test_gradients_larger_than_the_sweep_backwards_starts_at(ctx, g_dtype, in_place):
    """From 400 MiB of gradients on the scaling sweep goes backwards and the norm has more blocks: every element
    scaled once, elements between the tensors untouched, norm and clip agreeing on the result."""
    it = 2 if g_dtype == "bf16" else 4
    sizes = [5, 60_000_011, 1, (440 << 20) // it - 60_100_000, 8192, 100_003]
    offs, at = [], 3
    for n in sizes:
        offs.append(at)
        at += n + 1
    total = at + 16
    pattern = (np.random.default_rng(6).standard_normal(999_983) * 1e-3).astype(np.float32)
    small, vals = _dev(ctx, pattern, g_dtype)
    bits = small.to_numpy()
    small.free()
    d = anc.DBuf(np.resize(bits, total), ctx)
    out = d if in_place else anc.DBuf.zeros((total,), bits.dtype, ctx)
    clip = anc.GradClip([dict(g=d.ptr + o * it, numel=n, out=out.ptr + o * it) for o, n in zip(offs, sizes)],
                        grad_dtype=g_dtype, ctx=ctx)
    sq = 0.0
    one = np.square(vals.astype(np.float64))
    for o, n in zip(offs, sizes):
        whole, rest = divmod(n, len(vals))
        sq += whole * math.fsum(one) + math.fsum(_tile(one, o + whole * len(vals), rest))
    want = math.sqrt(sq)
    clip.norm(0.25)
    first = clip.read()
    clip.clip(0.25)
    got = clip.read()
    for norm, factor in (first, got):
        _check_norm((norm, factor), (want, 0.25 / (want + 1e-6)))
    scaled = vals * np.float32(got[1])
    scaled = obf.rne_bits(scaled) if g_dtype == "bf16" else scaled
    result = out.to_numpy()
    for o, n in zip(offs, sizes):
        assert np.array_equal(result[o:o + n], _tile(scaled, o, n)), (o, n)
        assert result[o - 1] == (bits[(o - 1) % len(bits)] if in_place else 0), o
    clip.free()
    if not in_place:
        out.free()
    d.free()


@pytest.mark.parametrize("captured", [False, True])
def test_chained_clips_in_two_launches(ctx, captured):
    """The sweep that starts beside its norm: a plan's output is the next plan's gradient, back to back on one
    stream, also captured; every pass sees the gradients written just before it."""
    rng = np.random.default_rng(12)
    n = 12_000_005
    a, b, c = (anc.DBuf.zeros((n,), t, ctx) for t in (np.float32, np.float32, np.uint16))
    first = anc.GradClip([dict(g=a, numel=n, out=b)], grad_dtype="f32", ctx=ctx)
    second = anc.GradClip([dict(g=b, numel=n, out=c)], grad_dtype="f32", out_dtype="bf16", ctx=ctx)
    hosts = [(rng.standard_normal(n) * s).astype(np.float32) for s in (1e-3, 7.0, 0.5)]
    dev = [anc.DBuf(h, ctx) for h in hosts]

    def pair():
        first.clip(3.0, scale=0.5, stream=ctx.stream)
        second.clip(2.0, stream=ctx.stream)
    g = C.c_void_p()
    if captured:
        L.check(L.lib().anc_graph_begin(ctx.handle, ctx.stream))
        pair()
        L.check(L.lib().anc_graph_end(ctx.handle, ctx.stream, C.byref(g)))
    for k in (0, 1, 2, 1, 0, 2):
        for j in (2, k):                     # two passes without a wait between them: the second one counts
            L.check(L.lib().anc_d2d(ctx.handle, a.ptr, dev[j].ptr, 4 * n, ctx.stream))
            if captured:
                L.check(L.lib().anc_graph_launch(ctx.handle, g, ctx.stream))
            else:
                pair()
        ctx.sync()
        r1, r2 = first.read(), second.read()
        _check_norm(r1, clip_ref.norm_and_factor([hosts[k]], 3.0, scale=0.5))
        mid = hosts[k] * np.float32(r1[1])
        assert np.array_equal(b.to_numpy(), mid)
        _check_norm(r2, clip_ref.norm_and_factor([mid], 2.0))
        assert np.array_equal(c.to_numpy(), obf.rne_bits(mid * np.float32(r2[1])))
    if captured:
        L.check(L.lib().anc_graph_destroy(g))
    for x in (first, second, a, b, c, *dev):
        x.free()


@pytest.mark.parametrize("mode", ["in place", "mixed"])
def test_clips_in_place_in_two_launches(ctx, mode):
    """Tensors in place beside tensors with an output of their own, repeated without waits: a second clip finds the
    first one's gradients."""
    rng = np.random.default_rng(13)
    n = 9_000_001
    ha, hb = ((rng.standard_normal(n) * 0.1).astype(np.float32) for _ in range(2))
    a, b, out = anc.DBuf(ha, ctx), anc.DBuf(hb, ctx), anc.DBuf.zeros((n,), np.float32, ctx)
    clip = anc.GradClip([dict(g=a, numel=n), dict(g=b, numel=n, out=b if mode == "in place" else out)],
                        grad_dtype="f32", ctx=ctx)
    limits = (100.0, 50.0, 20.0, 1e9)
    for mx in limits:
        clip.clip(mx, stream=ctx.stream)
    ctx.sync()
    va, vb, vo = ha, hb, None
    for mx in limits:
        _, f = clip_ref.norm_and_factor([va, vb], mx)
        f = np.float32(f)
        vo = vb * f
        va, vb = va * f, (vo if mode == "in place" else vb)
    # the last factor is 1: the gradients are those its norm saw
    _check_norm(clip.read(), clip_ref.norm_and_factor([a.to_numpy(), b.to_numpy()], 1e9))
    # each of the four factors is within 6u of the oracle's and each product within u: 28u in all
    assert np.allclose(a.to_numpy(), va, rtol=30 * U, atol=0)
    assert np.allclose((b if mode == "in place" else out).to_numpy(), vo, rtol=30 * U, atol=0)
    if mode == "mixed":
        assert np.array_equal(b.to_numpy(), hb)
    clip.free()
    for x in (a, b, out):
        x.free()
