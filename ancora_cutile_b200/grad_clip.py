"""Global gradient norm over many device tensors, and clipping by it.

The reference steps on its gradients as they are; training loops put a clip in front.  Everything stays on
the device: ``norm`` leaves {norm, factor} in two floats of device memory, ``clip`` multiplies the gradients by
the factor, and the optimizer sweeps can apply the factor themselves as they load the gradients
(``ResidentAdamW.set_grad_scale``, ``MuonPlan.set_grad_scale``, ``ResidentHybrid(max_grad_norm=...)``).
"""
import ctypes as C

import numpy as np

from . import _lib as L
from .buffers import dev_ptr, get_context

_GRAD = {"bf16": L.GRAD_BF16, "f32": L.GRAD_F32}
_SIZE = {"bf16": 2, "f32": 4}


def _buf(obj, numel, dtype, what):
    """Address of ``obj``; a buffer that knows its size must hold ``numel`` elements."""
    n = getattr(obj, "nbytes", None)
    if n is not None and n < numel * _SIZE[dtype]:
        raise ValueError(f"{what} holds {n} bytes: too few for {numel} {dtype}")
    return dev_ptr(obj)


class GradClip:
    """tensors: list of dicts {g, numel[, out]}: device buffers (anything ``dev_ptr`` accepts) of ``grad_dtype``,
    with ``out`` of ``out_dtype`` (default: the same type), or absent or ``g`` itself to clip in place.  ``result``: a caller's
    device buffer of two float32 {norm, factor}; by default the plan holds them.

      norm   = scale * sqrt(sum of squares over all tensors)
      factor = scale * min(1, max_norm / (norm + eps))

    Calls are asynchronous on ``stream`` and must be ordered among themselves."""

    def __init__(self, tensors, grad_dtype="bf16", out_dtype=None, result=None, ctx=None):
        self.ctx = ctx or get_context()
        self.grad_dtype, self.out_dtype = grad_dtype, out_dtype or grad_dtype
        arr = (L.ClipTensor * max(len(tensors), 1))()
        for i, t in enumerate(tensors):
            n = int(t["numel"])
            if n < 0:
                raise ValueError(f"tensor {i}: numel {n}")
            arr[i] = L.ClipTensor(_buf(t["g"], n, self.grad_dtype, f"tensor {i}: g"),
                                  _buf(t.get("out"), n, self.out_dtype, f"tensor {i}: out"), n)
        h = C.c_void_p()
        L.check(L.lib().anc_clip_plan_create(self.ctx.handle, arr, len(tensors), _GRAD[self.grad_dtype],
                                             _GRAD[self.out_dtype], _buf(result, 2, "f32", "result"), C.byref(h)))
        self.handle = h
        r, s = C.c_void_p(), C.c_void_p()
        L.check(L.lib().anc_clip_plan_result(self.handle, C.byref(r), C.byref(s)))
        self.result_ptr, self.sumsq_ptr = r.value, s.value

    @property
    def factor_ptr(self):
        """Device address of the float32 factor (what ``set_grad_scale`` takes)."""
        return self.result_ptr + 4

    def norm(self, max_norm=float("inf"), scale=1.0, eps=1e-6, stream=None):
        """{norm, factor} of the gradients as they are now."""
        rc = L.lib().anc_grad_norm(self.handle, scale, max_norm, eps, stream or None)
        if rc:
            L.check(rc)

    def clip(self, max_norm, scale=1.0, eps=1e-6, stream=None):
        """``norm``, then out = round(g * factor) for every tensor."""
        rc = L.lib().anc_grad_clip(self.handle, scale, max_norm, eps, stream or None)
        if rc:
            L.check(rc)

    def sumsq(self, stream=None):
        """This rank's sum of squares alone (``sumsq_ptr``); add the ranks' sums, then ``finish``."""
        L.check(L.lib().anc_grad_sumsq(self.handle, stream or None))

    def finish(self, max_norm=float("inf"), scale=1.0, eps=1e-6, stream=None):
        """{norm, factor} from the sum of squares at ``sumsq_ptr``."""
        L.check(L.lib().anc_grad_norm_finish(self.handle, scale, max_norm, eps, stream or None))

    def apply(self, stream=None):
        """out = round(g * factor) with the factor the last ``norm`` / ``finish`` left."""
        L.check(L.lib().anc_grad_apply(self.handle, stream or None))

    def read(self, stream=None):
        """(norm, factor) as Python floats; waits for ``stream``."""
        out = np.empty(2, np.float32)
        L.check(L.lib().anc_d2h(self.ctx.handle, out.ctypes.data, self.result_ptr, 8, stream or None, 1))
        return float(out[0]), float(out[1])

    def free(self):
        if self.handle:
            L.check(L.lib().anc_clip_plan_destroy(self.handle))
            self.handle = None
