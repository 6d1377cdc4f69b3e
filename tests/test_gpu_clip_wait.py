"""GPU: the wait between the blocks of the one-launch clip, made to run out: one block comes only after another has
given up.  No block may then take the count for complete: norm and factor are NaN, every gradient and every output is
as it was, status bit 0x10 is set, and the next call on the plan is right."""
import ctypes as C
import math

import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import _lib as L
from oracle import bf16 as obf, clip_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _run_out(clip, late, polls=200, max_norm=0.5):
    return L.lib().anc_clip_wait_selftest(clip.handle, max_norm, polls, late, None)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("g_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [9000, 500_003])
def test_blocks_decide_together_when_the_wait_runs_out(ctx, n, g_dtype, in_place):
    rng = np.random.default_rng(n)
    host = rng.standard_normal(n).astype(np.float32)
    bits = obf.rne_bits(host) if g_dtype == "bf16" else host
    vals = obf.bits_f32(bits) if g_dtype == "bf16" else host
    d = anc.DBuf(bits, ctx)
    out = d if in_place else anc.DBuf.zeros((n,), np.uint16, ctx)
    clip = anc.GradClip([dict(g=d, numel=n, out=None if in_place else out)], grad_dtype=g_dtype,
                        out_dtype=g_dtype if in_place else "bf16", ctx=ctx)
    blocks = -(-n // 8192)
    ctx.sync()
    assert ctx.status() == 0
    before = out.to_numpy()
    for late in sorted({0, blocks // 2, blocks - 1}):
        for _ in range(2):
            L.check(_run_out(clip, late))
            ctx.sync()
            assert ctx.status() == 0x10
            assert all(math.isnan(x) for x in clip.read())
            assert np.array_equal(d.to_numpy(), bits)
            assert np.array_equal(out.to_numpy(), before)
    assert ctx.status() == 0                                       # reading clears it
    clip.clip(0.5)
    norm, f = clip.read()
    want = clip_ref.norm_and_factor([vals], 0.5)
    assert abs(norm - want[0]) <= 6 * U * want[0] and abs(f - want[1]) <= 6 * U * want[1]
    scaled = vals * np.float32(f)
    got = out.to_numpy()
    assert np.array_equal(got, scaled if got.dtype == np.float32 else obf.rne_bits(scaled))
    assert ctx.status() == 0
    clip.free()
    d.free()
    if not in_place:
        out.free()


def test_refusals(ctx):
    d = anc.DBuf.zeros((20000,), np.float32, ctx)
    one, three = (anc.GradClip([dict(g=d, numel=n)], grad_dtype="f32", ctx=ctx) for n in (100, 20000))
    assert _run_out(one, 0) == L.E_INVALID                         # a single block waits for nobody
    for kw in (dict(late=3), dict(late=0, polls=0), dict(late=0, polls=(1 << 14) + 1), dict(late=0, max_norm=-1.0)):
        assert _run_out(three, **kw) == L.E_INVALID
    assert L.lib().anc_clip_wait_selftest(None, 1.0, 10, C.c_uint32(0), None) == L.E_INVALID
    for x in (one, three, d):
        x.free()
