"""CPU: a tensor clipped in place keeps its type, however the caller says that it is in place: a wider output would run
past the gradient, a narrower one would lie over gradients that are still to be read."""
import ctypes as C

import pytest

from ancora_cutile_b200 import AncoraError, GradClip, _lib as L

FAKE = C.c_void_p(4096)        # stands for a context; never read


@pytest.mark.parametrize("grad,out", [(L.GRAD_F32, L.GRAD_BF16), (L.GRAD_BF16, L.GRAD_F32)])
@pytest.mark.parametrize("tensors", [
    [(4096, 4096, 64)],
    [(4096, 4096, 1)],
    [(8192, 16384, 64), (4096, 4096, 64)],
    [(4096, None, 64)],
])
def test_in_place_with_unequal_types_is_refused(tensors, grad, out):
    arr = (L.ClipTensor * len(tensors))(*[L.ClipTensor(*t) for t in tensors])
    h = C.c_void_p()
    assert L.lib().anc_clip_plan_create(FAKE, arr, len(tensors), grad, out, None, C.byref(h)) == L.E_INVALID
    assert h.value is None
    assert b"in place" in L.lib().anc_last_error()


def test_python_plans_refuse_it_too():
    class Ctx:
        handle = FAKE
    for kw in (dict(grad_dtype="f32", out_dtype="bf16"), dict(grad_dtype="bf16", out_dtype="f32")):
        with pytest.raises(AncoraError, match="in place"):
            GradClip([dict(g=4096, numel=64, out=4096)], ctx=Ctx, **kw)
