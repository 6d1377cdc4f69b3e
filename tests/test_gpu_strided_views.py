"""GPU: views of another library whose rows lie apart, given as they are with their row strides."""
import numpy as np
import pytest

import ancora_cutile_b200 as anc
from ancora_cutile_b200.kernels import embedding_grad, embedding_grad_workspace, embedding_lookup
from oracle import bf16 as obf, embed_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,gap", [(8, 8), (77, 3), (256, 64)])
def test_torch_views(ctx, D, gap, dtype):
    torch = pytest.importorskip("torch")
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    rng = np.random.default_rng(D)
    T, V, ld = 50, 20, D + gap
    ids = rng.integers(-1, V, T)
    vals = lambda *s: obf.rne_f32((rng.integers(-8, 9, s) / 8).astype(np.float32))  # noqa: E731
    host = dict(table=vals(V, ld), out=vals(T, ld), dy=vals(T, ld), dw=vals(V, ld))
    dev = {k: torch.tensor(v, device=f"cuda:{ctx.device}", dtype=dt) for k, v in host.items()}
    d_ids = torch.tensor(ids, device=f"cuda:{ctx.device}")
    work = anc.DBuf.empty((embedding_grad_workspace(T, V, D),), np.uint8, ctx)
    torch.cuda.synchronize()
    view = {k: x[:, :D] for k, x in dev.items()}
    assert view["table"].nbytes < ((V - 1) * ld + D) * view["table"].element_size()
    embedding_lookup(view["table"], d_ids, view["out"], T, V, D, scale=0.5, table_dtype=dtype, out_dtype=dtype,
                     table_ld=ld, out_ld=ld, ctx=ctx)
    embedding_grad(view["dy"], d_ids, view["dw"], T, V, D, work, scale=2.0, dy_dtype=dtype, dw_dtype=dtype, mode="add",
                   dy_ld=ld, dw_ld=ld, ctx=ctx)
    ctx.sync()
    want = dict(host)
    want["out"] = host["out"].copy()
    want["out"][:, :D] = embed_ref.lookup(host["table"][:, :D], ids, 0.5, "f32")
    want["dw"] = host["dw"].copy()
    want["dw"][:, :D] = embed_ref.grad(host["dy"][:, :D], ids, V, 2.0, host["dw"][:, :D])[0]
    for k, w in want.items():                                      # eighths of small integers: exact, also in bf16
        assert np.array_equal(dev[k].float().cpu().numpy(), obf.rne_f32(w) if dtype == "bf16" else w), k
    work.free()
    assert ctx.status() == 0
