"""GPU: ways through the clip that depend on where gradients and outputs lie and on how many there are: no common
alignment of the two, tensors in place beside others, infinities and NaN, on one launch and on two.

Each clipped element is one float32 product by the device's own factor and one rounding: equal to numpy's bit for
bit.  The norm's tolerance of 6 * 2^-24: eight float32 roundings at most in a group of eight positive terms, halved by
the root, and one of the result."""
import math

import numpy as np
import pytest

import ancora_cutile_b200 as anc
from oracle import bf16 as obf, clip_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SIZE = {"bf16": 2, "f32": 4}
ONE_LAUNCH, TWO_LAUNCHES = 100_000, 9_000_000      # elements; the second is more than the resident blocks hold


def _dev(ctx, x, dtype):
    if dtype == "bf16":
        b = obf.rne_bits(x)
        return anc.DBuf(b, ctx), obf.bits_f32(b)
    return anc.DBuf(x, ctx), x


def _check(got, want):
    for g, w in zip(got, want):
        assert abs(g - w) <= 6 * U * abs(w), (got, want)


@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [(0, 1), (3, 0), (5, 6)])
@pytest.mark.parametrize("sizes", [[7, 8, 9, 8191, 8193, 40_001, 1], [TWO_LAUNCHES, 8200]])
def test_no_common_alignment(ctx, sizes, shift, g_dtype, out_dtype):
    """Gradient and output start at different elements of their vectors of eight; a tensor with a common alignment
    and an empty one between them."""
    rng = np.random.default_rng(len(sizes))
    sizes = sizes[:1] + [0, 4000] + sizes[1:]
    go, oo, ag, ao = [], [], 16, 16
    for k, n in enumerate(sizes):
        s = (2, 2) if k == 2 else shift                            # elements past a multiple of 8
        go.append(ag + s[0])
        oo.append(ao + s[1])
        ag += (n + 23) // 8 * 8
        ao += (n + 23) // 8 * 8
    host = (rng.standard_normal(ag + 16) * 0.01).astype(np.float32)
    d, vals = _dev(ctx, host, g_dtype)
    fill = np.full(ao + 16, 0x7ABC, np.uint16) if out_dtype == "bf16" else np.full(ao + 16, 7.5, np.float32)
    out = anc.DBuf(fill, ctx)
    clip = anc.GradClip([dict(g=d.ptr + o * SIZE[g_dtype], numel=n, out=out.ptr + p * SIZE[out_dtype])
                         for o, p, n in zip(go, oo, sizes)], grad_dtype=g_dtype, out_dtype=out_dtype, ctx=ctx)
    parts = [vals[o:o + n] for o, n in zip(go, sizes)]
    for max_norm in (0.25, 1e9):
        clip.clip(max_norm, scale=0.5)
        got = clip.read()
        _check(got, clip_ref.norm_and_factor(parts, max_norm, 0.5))
        want = fill.copy()
        for p, n, x in zip(oo, sizes, parts):
            y = x * np.float32(got[1])
            want[p:p + n] = obf.rne_bits(y) if out_dtype == "bf16" else y
        assert np.array_equal(out.to_numpy(), want)
    assert np.array_equal(d.to_numpy(), obf.rne_bits(host) if g_dtype == "bf16" else host)
    clip.free()
    d.free()
    out.free()
    assert ctx.status() == 0


@pytest.mark.parametrize("n", [ONE_LAUNCH, TWO_LAUNCHES])
@pytest.mark.parametrize("where", ["own output", "in place"])
@pytest.mark.parametrize("g_dtype,out_dtype", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_infinities_and_nan(ctx, bad, g_dtype, out_dtype, where, n):
    """In a vector, and in the elements before and behind the vectors."""
    if where == "in place" and g_dtype != out_dtype:
        with pytest.raises(anc.AncoraError, match="in place"):
            anc.GradClip([dict(g=4096, numel=n, out=4096)], grad_dtype=g_dtype, out_dtype=out_dtype, ctx=ctx)
        return
    o = 3
    for at in (0, n // 2, n - 1):
        host = np.full(n + 8, 2.0 ** -10, np.float32)
        host[o + at] = bad
        d, vals = _dev(ctx, host, g_dtype)
        out = d if where == "in place" else anc.DBuf.zeros((n + 8,), np.uint16 if out_dtype == "bf16" else np.float32, ctx)
        clip = anc.GradClip([dict(g=d.ptr + o * SIZE[g_dtype], numel=n, out=out.ptr + o * SIZE[out_dtype])],
                            grad_dtype=g_dtype, out_dtype=out_dtype, ctx=ctx)
        clip.clip(math.inf)                                        # never clips: as it was
        assert clip.read()[1] == 1.0
        got = out.to_numpy()[o:o + n]
        got = obf.bits_f32(got) if out_dtype == "bf16" else got
        assert np.array_equal(got, vals[o:o + n], equal_nan=True)
        clip.clip(1.0)
        norm, f = clip.read()
        got = out.to_numpy()
        got = obf.bits_f32(got) if out_dtype == "bf16" else got
        if math.isnan(bad):
            assert math.isnan(norm) and math.isnan(f) and np.isnan(got[o:o + n]).all()
        else:
            assert norm == math.inf and f == 0.0
            assert np.isnan(got[o + at]) and not np.delete(got[o:o + n], at).any()
        edge = np.concatenate([got[:o], got[o + n:]])
        assert np.array_equal(edge, np.full(8, 2.0 ** -10 if where == "in place" else 0.0))
        clip.free()
        d.free()
        if out is not d:
            out.free()
    assert ctx.status() == 0
