"""Timed cases of the gradient-side operators next to the optimizer step: the global gradient norm, gradient
clipping, the embedding lookup and the embedding's gradient by sorted tokens.

``run`` computes an operator in elementary torch operations, or, where ``own`` is true, through this package.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4, "i32": 4, "i64": 8}
_EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the norm every step logs and clips by, for the gradients of a two-layer test model: launch latency
        dict(name="norm small model", op="norm", set="model", layers=2, hidden=256, ffn=768, vocab=2048, gap=64,
             g="bf16", scale=1.0, max_norm=1.0),
        # the same for all 310 tensors of the benchmark model, 1.19 GB of bf16 gradients
        dict(name="norm benchmark model", op="norm", set="model", layers=28, hidden=1024, ffn=3072, vocab=151936,
             gap=64, g="bf16", scale=1.0, max_norm=1.0),
        # float32 gradients of a checkpoint-like bag of tensors packed with no alignment
        dict(name="norm ragged f32", op="norm", set="ragged", count=61, total=40000003, gap=1, g="f32", scale=0.5,
             max_norm=0.25),
        # clipping for the test model
        dict(name="clip small model", op="clip", set="model", layers=2, hidden=256, ffn=768, vocab=2048, gap=64,
             g="bf16", out="bf16", scale=1.0, max_norm=1.0),
        # float32 accumulators of four micro-batches -> clipped bf16 gradients, four layers and the embedding
        dict(name="clip accumulators", op="clip", set="model", layers=4, hidden=1024, ffn=3072, vocab=151936, gap=64,
             g="f32", out="bf16", scale=0.25, max_norm=1.0),
        # the benchmark model's bf16 gradients
        dict(name="clip benchmark model", op="clip", set="model", layers=28, hidden=1024, ffn=3072, vocab=151936,
             gap=64, g="bf16", out="bf16", scale=1.0, max_norm=1.0),
        # one decoding step of a few sequences
        dict(name="lookup decode", op="lookup", T=4, V=151936, D=1024, w="bf16", out="bf16", ids="i64", scale=1.0,
             pad=0.0),
        # a training micro-batch of 16 sequences of 2048 tokens, a twentieth of it padding
        dict(name="lookup micro-batch", op="lookup", T=32768, V=151936, D=1024, w="bf16", out="bf16", ids="i32",
             scale=32.0, pad=0.05),
        # a few tokens, odd row length: the unaligned path
        dict(name="embedding grad small odd", op="grad", T=37, V=1000, D=131, dy="f32", dw="f32", ids="i64",
             scale=1.0, pad=0.1, mode="add"),
        # the test model's micro-batch, whole table written
        dict(name="embedding grad test model", op="grad", T=2048, V=2048, D=256, dy="bf16", dw="bf16", ids="i64",
             scale=1.0, pad=0.0, mode="write"),
        # benchmark model, 8 sequences of 2048 tokens: the whole bf16 gradient table is written
        dict(name="embedding grad write", op="grad", T=16384, V=151936, D=1024, dy="bf16", dw="bf16", ids="i64",
             scale=1.0, pad=0.0, mode="write"),
        # benchmark model, 32 sequences of 2048 tokens added into the float32 accumulator
        dict(name="embedding grad accumulate", op="grad", T=65536, V=151936, D=1024, dy="bf16", dw="f32", ids="i32",
             scale=32.0, pad=0.05, mode="add"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "lookup", "grad"])
    if op in ("norm", "clip"):
        if rng.random() < 0.4:
            hidden = 128 * rng.randint(1, 8)
            c = dict(set="model", layers=_log(rng, 1, 28), hidden=hidden, ffn=hidden * 3, vocab=_log(rng, 500, 151936))
        else:
            count = _log(rng, 1, 200)
            c = dict(set="ragged", count=count, total=max(count, _log(rng, 1000, 300000000)))
        c.update(op=op, gap=rng.choice([1, 64]), g=rng.choice(["bf16", "f32"]), scale=rng.choice([1.0, 0.5, 0.125]),
                 max_norm=rng.choice([0.01, 0.25, 1.0, 100.0]))
        if op == "clip":
            c["out"] = rng.choice(["bf16", "f32"])
            if c["set"] == "model" and c["layers"] > 14:
                c["layers"] = 14
        return c
    D = _log(rng, 8, 4096)
    if rng.random() < 0.6:
        D = max(8, D // 8 * 8)
    V = min(_log(rng, 100, 262144), (1 << 28) // D)
    T = min(_log(rng, 1, 131072), (1 << 27) // D)
    c = dict(op=op, T=T, V=V, D=D, ids=rng.choice(["i32", "i64"]), scale=rng.choice([1.0, 0.5, math.sqrt(D)]),
             pad=rng.choice([0.0, 0.0, 0.05, 0.3]))
    if op == "lookup":
        c.update(w=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
    else:
        c.update(dy=rng.choice(["bf16", "f32"]), dw=rng.choice(["bf16", "f32"]), mode=rng.choice(["write", "add"]))
    return c


def _sizes(case):
    """Element counts of the gradient tensors of a case."""
    if case["set"] == "model":
        H, F = case["hidden"], case["ffn"]
        layer = [H, 2 * H * H, H * H, H * H, 128, 128, 2 * H * H, H, H * F, H * F, F * H]
        return [case["vocab"] * H] + layer * case["layers"] + [H]
    r = np.random.RandomState(case["count"])
    share = r.lognormal(0.0, 2.0, case["count"])
    sizes = np.maximum(1, (share / share.sum() * case["total"]).astype(np.int64))
    return [int(x) for x in sizes]


def _offsets(sizes, gap):
    offs, at = [], 0
    for n in sizes:
        offs.append(at)
        at = -(-(at + n) // gap) * gap
    return offs, max(at, 1)


def _distinct(case):
    """Expected number of table rows that the tokens of a case name (ids follow a 1 / rank law)."""
    T, V = case["T"] * (1.0 - case["pad"]), case["V"]
    rank = np.arange(V, dtype=np.float64)
    p = np.log((rank + 2) / (rank + 1)) / math.log(V + 1)
    return float(np.sum(1.0 - np.exp(T * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def work(case):
    op = case["op"]
    if op in ("norm", "clip"):
        n = sum(_sizes(case))
        b = n * _BYTES[case["g"]] + 8
        return {"bytes": b + (n * _BYTES[case["out"]] if op == "clip" else 0), "flops": (2 if op == "norm" else 3) * n}
    T, V, D = case["T"], case["V"], case["D"]
    used, rows = T * (1.0 - case["pad"]), _distinct(case)
    if op == "lookup":
        return {"bytes": T * _BYTES[case["ids"]] + rows * D * _BYTES[case["w"]] + T * D * _BYTES[case["out"]],
                "flops": T * D}
    table = V * D * _BYTES[case["dw"]] if case["mode"] == "write" else 2 * rows * D * _BYTES[case["dw"]]
    return {"bytes": T * _BYTES[case["ids"]] + used * D * _BYTES[case["dy"]] + table, "flops": used * D + rows * D}


# ------------------------------------------------------------------ inputs
def _token_ids(case, gen):
    """Token ids with the 1 / rank law of text, spread over the table; the padded tail is -1."""
    T, V = case["T"], case["V"]
    u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
    ids = (rank * 1000003 + 12345) % V
    n_pad = int(case["pad"] * T)
    if n_pad:
        ids[T - n_pad:] = -1
    return ids.to(torch.int32) if case["ids"] == "i32" else ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=case)
    if op in ("norm", "clip"):
        sizes = _sizes(case)
        offs, total = _offsets(sizes, case["gap"])
        arena = torch.empty(total, device="cuda", dtype=_DT[case["g"]]).normal_(0.0, 1e-3, generator=gen)
        arena[:sizes[0] // 2].zero_()                  # embedding rows that no token of the step named
        s["grads"] = [arena[o:o + n] for o, n in zip(offs, sizes)]
        s["result"] = torch.zeros(2, device="cuda")
        if op == "clip":
            s["out"] = torch.zeros(total, device="cuda", dtype=_DT[case["out"]])
            s["outs"] = [s["out"][o:o + n] for o, n in zip(offs, sizes)]
        if own:
            from ancora_cutile_b200 import GradClip
            s["plan"] = GradClip(
                [dict(g=g.data_ptr(), numel=g.numel(), out=s["outs"][i].data_ptr() if op == "clip" else None)
                 for i, g in enumerate(s["grads"])],
                grad_dtype=case["g"], out_dtype=case.get("out"), result=s["result"].data_ptr())
        return s
    T, V, D = case["T"], case["V"], case["D"]
    s["ids"] = _token_ids(case, gen)
    if op == "lookup":
        s["table"] = torch.empty(V, D, device="cuda", dtype=_DT[case["w"]]).normal_(0.0, 0.02, generator=gen)
        s["out"] = torch.zeros(T, D, device="cuda", dtype=_DT[case["out"]])
    else:
        s["dy"] = torch.empty(T, D, device="cuda", dtype=_DT[case["dy"]]).normal_(0.0, 1e-3, generator=gen)
        s["dw"] = torch.empty(V, D, device="cuda", dtype=_DT[case["dw"]]).normal_(0.0, 1e-3, generator=gen)
        if own:
            from ancora_cutile_b200 import kernels
            s["work"] = torch.empty(kernels.embedding_grad_workspace(T, V, D), device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------ the operators
def _stream():
    return torch.cuda.current_stream().cuda_stream or 1     # 1: the legacy default stream's own handle


def _run_own(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        s["plan"].norm(case["max_norm"], scale=case["scale"], eps=_EPS, stream=_stream())
        return s["result"]
    if op == "clip":
        s["plan"].clip(case["max_norm"], scale=case["scale"], eps=_EPS, stream=_stream())
        return {"result": s["result"], "out": s["out"]}
    from ancora_cutile_b200 import kernels
    if op == "lookup":
        kernels.embedding_lookup(s["table"].data_ptr(), s["ids"].data_ptr(), s["out"].data_ptr(), case["T"], case["V"],
                                 case["D"], scale=case["scale"], table_dtype=case["w"], out_dtype=case["out"],
                                 ids_dtype=case["ids"], stream=_stream())
        return s["out"]
    kernels.embedding_grad(s["dy"].data_ptr(), s["ids"].data_ptr(), s["dw"].data_ptr(), case["T"], case["V"],
                           case["D"], s["work"].data_ptr(), scale=case["scale"], dy_dtype=case["dy"],
                           dw_dtype=case["dw"], ids_dtype=case["ids"], mode=case["mode"], stream=_stream())
    return s["dw"]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op in ("norm", "clip"):
        # squares in 32 bits, their sum in 64: one number from up to 600 million
        sq = torch.stack([g.float().square().sum(dtype=torch.float64) for g in state["grads"]])
        norm = sq.sum().sqrt() * case["scale"]
        factor = case["scale"] * torch.clamp(case["max_norm"] / (norm + _EPS), max=1.0)
        result = torch.stack([norm, factor]).float()
        if op == "norm":
            return result
        [o.copy_(g.float() * result[1]) for o, g in zip(state["outs"], state["grads"])]
        return {"result": result, "out": state["out"]}
    ids = state["ids"].long()
    live = (ids >= 0)[:, None]
    if op == "lookup":
        rows = state["table"][ids.clamp(min=0)].float() * case["scale"]
        return torch.where(live, rows, 0.0).to(_DT[case["out"]])
    dy = torch.where(live, state["dy"].float(), 0.0)
    total = torch.zeros(case["V"], case["D"], device=dy.device).index_add_(0, ids.clamp(min=0), dy) * case["scale"]
    dw = state["dw"]
    return dw.copy_(total if case["mode"] == "write" else dw.float() + total)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "clip"):
        sq = math.fsum(float(torch.dot(p, p)) for g in s["grads"] for c in g.split(1 << 26) for p in (c.double(),))
        norm = case["scale"] * math.sqrt(sq)
        factor = case["scale"] * min(1.0, case["max_norm"] / (norm + _EPS))
        result = torch.tensor([norm, factor], dtype=torch.float64)
        if op == "norm":
            return result
        out = torch.zeros(s["out"].shape, device="cuda", dtype=torch.float64)
        at = 0
        for g in s["grads"]:
            out[at:at + g.numel()] = g.double() * factor
            at = -(-(at + g.numel()) // case["gap"]) * case["gap"]
        return {"result": result, "out": out}
    ids = s["ids"].long()
    keep = torch.nonzero(ids >= 0).flatten()
    if op == "lookup":
        out = torch.zeros(case["T"], case["D"], device="cuda", dtype=torch.float64)
        out[keep] = s["table"].double()[ids[keep]] * case["scale"]
        return out
    out = torch.zeros(case["V"], case["D"], device="cuda", dtype=torch.float64)
    if case["mode"] == "add":
        out += s["dw"].double()
    if keep.numel():
        # sums of runs of equal ids as differences of a running sum over the sorted tokens
        order = keep[torch.argsort(ids[keep], stable=True)]
        run_sum = s["dy"][order].double().cumsum(0)
        last = torch.nonzero(torch.diff(ids[order], append=ids.new_tensor([-2]))).flatten()
        upto = run_sum[last]
        out[ids[order][last]] += case["scale"] * torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))
    return out
