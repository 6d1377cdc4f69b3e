"""GPU: the embedding's gradient added straight into the engine's float32 accumulator, over several optimizer steps.

All gradients are whole multiples of 2^-14 of a few magnitudes, so every float32 sum is exact and the sums
are compared bit for bit."""
import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200 import shapes as S
from oracle import bf16 as obf, embed_ref, grad_ref

pytestmark = pytest.mark.gpu
AKW = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, wd=0.1)
SHP = dict(S.qwen3_0_6b_shapes(n_layers=1, hidden=128, q_heads=2, kv_heads=1, head_dim=128, ffn=384, vocab=301))
V, D = SHP["embed"]
T = 400


class Window:
    """One optimizer step's micro-batches on an engine, and their sums in the oracle."""

    def __init__(self, ctx, seed=0, **kw):
        params = S.synthetic_params(SHP, seed=1)
        mu = [n for n, s in SHP.items() if anc.default_is_muon(n, np.empty((0,) * len(s)))]
        nd = tuple(n for n, s in SHP.items() if len(s) == 1)
        kw = dict(dict(adamw_kw=AKW, grad_dtype="bf16", rounding="rne", schedule=anc.PE_SCHEDULE, ctx=ctx), **kw)
        self.ctx, self.eng = ctx, anc.ResidentHybrid(params, mu, nd, **kw)
        self.rng = np.random.default_rng(seed)
        self.bufs = []

    def grad(self, shape):
        return (self.rng.integers(-8, 9, shape) * 2.0 ** -14).astype(np.float32)

    def write(self, names):
        """What a backward pass leaves in the gradient arena; returns it."""
        out = {n: self.grad(SHP[n]) for n in names}
        for n, g in out.items():
            self.eng.grad_view(n).upload(obf.rne_bits(g))
        return out

    def embed(self, **kw):
        """The embedding's gradient of one micro-batch into the accumulator; returns its sums."""
        ids = self.rng.integers(-1, V, T)
        dy = self.grad((T, D))
        di, dd = anc.DBuf(ids, self.ctx), anc.DBuf(obf.rne_bits(dy), self.ctx)
        self.bufs += [di, dd]
        self.eng.embedding_grad("embed", dd, di, T, mode="add", into="acc", **kw)
        return embed_ref.grad(dy, ids, V, 1.0)[0].astype(np.float32)

    def run(self, micro=2, tied=False, head_first=True, say=False, untied=False):
        """A whole window up to ``finalize_grads``; checks the finished gradients.  say, untied: the calls name it."""
        kw = dict(tied=True) if say else dict(tied=False) if untied else {}
        acc = {n: np.zeros(s, np.float32) for n, s in SHP.items()}
        for k in range(micro):
            if tied and head_first:
                acc["embed"] += self.write(["embed"])["embed"]
            acc["embed"] += self.embed(**kw)
            for n, g in self.write([n for n in SHP if n != "embed" or (tied and not head_first)]).items():
                acc[n] += g
            if k < micro - 1:
                self.eng.accumulate_grads(self.ctx.stream)
            else:
                self.eng.finalize_grads(self.ctx.stream, rounding="rne")
        self.check(acc, micro)

    def check(self, acc, micro):
        self.ctx.sync()
        for n in SHP:
            _, bits = grad_ref.grad_accumulate(acc[n].reshape(-1), None, scale=1.0 / micro)
            assert np.array_equal(self.eng.grad_view(n).to_numpy().reshape(-1), bits), n

    def free(self):
        self.eng.free()
        for b in self.bufs:
            b.free()
        assert self.ctx.status() == 0


@pytest.fixture
def win(ctx):
    w = Window(ctx)
    w.eng.enable_grad_accumulation()
    yield w
    w.free()


@pytest.mark.parametrize("micro", [1, 3])
def test_untied_table_over_several_steps(win, micro):
    """Nothing but the embedding writes the table's gradient: the finished gradient of one step is not part of
    the next one's sum."""
    for _ in range(3):
        win.run(micro)
        win.eng.step(win.ctx.stream)


@pytest.mark.parametrize("head_first", [True, False])
def test_tied_table_over_several_steps(win, head_first):
    for _ in range(3):
        win.run(2, tied=True, head_first=head_first)
        win.eng.step(win.ctx.stream)


def test_untied_table_over_replayed_half_and_host_steps(win):
    eng, st = win.eng, win.ctx.stream
    win.run()
    eng.step(st)
    eng.capture_step(st, horizon=8)
    for how in ("replay", "replay", "parts", "host", "step"):
        win.run()
        if how == "replay":
            eng.replay_step(st)
        elif how == "parts":
            eng.step_part("muon", st)
            eng.step_part("adamw", st)
        elif how == "host":
            grads = {n: obf.rne_bits(win.grad(s)) for n, s in SHP.items()}
            eng.step_host(grads, st)
        else:
            eng.step(st)
    win.run()


def test_untied_table_with_clipping(ctx):
    w = Window(ctx, max_grad_norm=0.01)
    w.eng.enable_grad_accumulation()
    for _ in range(3):
        w.run()
        w.eng.step(ctx.stream)
        assert w.eng.grad_norm()[1] < 1.0
    w.free()


@pytest.mark.parametrize("tied", [False, True])
def test_where_an_earlier_gradient_may_lie_in_the_arena(win, tied):
    """A step before the first call for the table: refused until the caller says whose the region is."""
    eng, st = win.eng, win.ctx.stream
    win.write(SHP)
    eng.step(st)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="tied"):
            win.embed()
    assert not eng.acc_a.to_numpy().any()                          # nothing was added
    acc = {n: np.zeros(s, np.float32) for n, s in SHP.items()}
    for k in range(2):
        for n, g in win.write([n for n in SHP if tied or n != "embed"]).items():
            acc[n] += g
        acc["embed"] += win.embed(tied=tied if k == 0 else None)   # said once, holds from then on
        (eng.accumulate_grads, lambda s: eng.finalize_grads(s, rounding="rne"))[k](st)
    win.check(acc, 2)
    eng.step(st)


def test_finished_gradients_that_no_step_took(win):
    """A step left out (a norm that is not finite, say): the next window may not add the finished gradient."""
    eng, st = win.eng, win.ctx.stream
    win.run()
    with pytest.raises(RuntimeError, match="tied"):
        win.embed()
    with pytest.raises(RuntimeError, match="tied"):
        eng.accumulate_grads(st)
    eng.step(st)                                                   # taken after all
    win.run()


def test_windows_without_steps_of_a_table_that_is_said_to_be_untied(win):
    for k in range(3):
        win.run(untied=True)
    win.eng.step(win.ctx.stream)
    win.run()


def test_windows_without_steps_of_a_table_that_is_said_to_be_tied(win):
    for k in range(3):
        win.run(tied=True, say=True)
    win.eng.step(win.ctx.stream)
    win.run(tied=True)


def test_tied_belongs_to_the_accumulator(win):
    ids, dy = anc.DBuf(np.zeros(4, np.int64), win.ctx), anc.DBuf(np.zeros((4, D), np.uint16), win.ctx)
    win.bufs += [ids, dy]
    with pytest.raises(ValueError, match="tied"):
        win.eng.embedding_grad("embed", dy, ids, 4, tied=True)
    win.eng.embedding_grad("embed", dy, ids, 4)                    # "write": the region is a fresh gradient
    assert not win.eng.grad_view("embed").to_numpy().any()


@pytest.mark.parametrize("full", [False, True])
def test_an_upload_of_all_gradients_leaves_nothing_to_say(win, full):
    """The table's region then holds what the caller put there, whatever came before."""
    eng, st = win.eng, win.ctx.stream
    win.write(SHP)
    eng.step(st)
    for k in range(2):                                             # after a step; after a window that was not stepped on
        up = {n: win.grad(s) for n, s in SHP.items()}
        (eng.upload_full_grads if full else eng.upload_grads)({n: obf.rne_bits(g) for n, g in up.items()}, st)
        up["embed"] = up["embed"] + win.embed()
        eng.finalize_grads(st, rounding="rne")
        win.check(up, 1)
