"""CPU: the engine's scratch for embedding gradients grows by a factor.  Earlier scratch is kept for graphs that may hold
it, so growing by what each call needs would keep about the square of it."""
from types import SimpleNamespace

import numpy as np

from ancora_cutile_b200 import kernels, resident


def test_token_counts_that_creep_upwards(monkeypatch):
    made, used = [], []

    class Buf:
        def __init__(self, nbytes):
            self.nbytes = nbytes
            made.append(nbytes)

    monkeypatch.setattr(resident, "DBuf", SimpleNamespace(empty=lambda shape, dtype, ctx: Buf(int(np.prod(shape)))))
    monkeypatch.setattr(resident.kernels, "embedding_grad",
                        lambda dy, ids, dw, T, V, D, work, **kw: used.append((T, work.nbytes)))
    eng = resident.ResidentHybrid.__new__(resident.ResidentHybrid)
    eng.shapes, eng.ctx, eng.grad_dtype, eng._embed_work = {"embed": (1000, 256)}, SimpleNamespace(stream=5), "bf16", []
    eng.grad_view, eng._acc_stale = lambda name: 4096, set()
    counts = list(range(1, 9000, 3)) + [100, 8000, 1]
    for T in counts:
        eng.embedding_grad("embed", 4096, 4096, T)
    need = [kernels.embedding_grad_workspace(T, 1000, 256) for T in counts]
    assert [t for t, _ in used] == counts
    assert all(n >= w for (_, n), w in zip(used, need))            # every call had what it needs
    assert sum(made) <= 4 * max(need)                              # in all, and each no more than twice the largest
    assert max(made) <= 2 * max(need)
    assert len(made) <= 20


def test_one_large_call_takes_no_more_than_it_needs(monkeypatch):
    made = []
    monkeypatch.setattr(resident, "DBuf", SimpleNamespace(
        empty=lambda shape, dtype, ctx: made.append(int(np.prod(shape))) or SimpleNamespace(nbytes=made[-1])))
    monkeypatch.setattr(resident.kernels, "embedding_grad", lambda *a, **kw: None)
    eng = resident.ResidentHybrid.__new__(resident.ResidentHybrid)
    eng.shapes, eng.ctx, eng.grad_dtype, eng._embed_work = {"embed": (1000, 256)}, SimpleNamespace(stream=5), "bf16", []
    eng.grad_view, eng._acc_stale = lambda name: 4096, set()
    eng.embedding_grad("embed", 4096, 4096, 65536)
    assert made == [kernels.embedding_grad_workspace(65536, 1000, 256)]
