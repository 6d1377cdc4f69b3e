"""CPU: the size check on the embedding calls' buffers goes by what a view spans, not by how many elements it has: a
view whose rows lie apart counts fewer bytes than lie between its first and last element."""
import ctypes as C

import numpy as np
import pytest

from ancora_cutile_b200 import AncoraError, kernels


class Ctx:
    handle = None                       # refused by the library, after the sizes were looked at


class View:
    """What array libraries report of a device array of ``shape`` whose strides are in elements."""

    def __init__(self, shape, strides, dtype, ptr=4096):
        it = np.dtype(dtype).itemsize
        self.nbytes = int(np.prod(shape)) * it
        self.__cuda_array_interface__ = dict(shape=shape, typestr=np.dtype(dtype).str, data=(ptr, False), version=3,
                                             strides=None if strides is None else tuple(s * it for s in strides))


def _lookup(**kw):
    kw = dict(dict(table=View((10, 8), (16, 1), np.uint16), ids=1 << 20, out=View((4, 8), None, np.uint16), T=4, V=10, D=8,
                   table_ld=16, ctx=Ctx), **kw)
    return kernels.embedding_lookup(**kw)


def _grad(**kw):
    kw = dict(dict(dy=View((4, 8), (24, 1), np.float32), ids=1 << 20, dw=View((10, 8), (9, 1), np.float32), work=1 << 24,
                   T=4, V=10, D=8, dy_dtype="f32", dw_dtype="f32", dy_ld=24, dw_ld=9, ctx=Ctx), **kw)
    return kernels.embedding_grad(**kw)


def test_views_with_rows_apart_reach_the_library():
    with pytest.raises(AncoraError, match="ctx"):
        _lookup()
    with pytest.raises(AncoraError, match="ctx"):
        _lookup(out=View((4, 8), (40, 1), np.uint16), out_ld=40)
    with pytest.raises(AncoraError, match="NULL"):
        _grad()


@pytest.mark.parametrize("call,kw,what", [
    (_lookup, dict(table_ld=17), "table"),                                     # rows further apart than the view's
    (_lookup, dict(V=11), "table"),
    (_lookup, dict(D=9), "table"),
    (_lookup, dict(table=View((10, 8), None, np.uint16)), "table"),            # contiguous: its bytes are its span
    (_lookup, dict(table=View((10, 8), (8, 1), np.uint16)), "table"),
    (_lookup, dict(table=View((0, 8), (16, 1), np.uint16)), "table"),          # spans nothing
    (_lookup, dict(table=View((10, 8), (-16, 1), np.uint16)), "table"),        # rows before its address
    (_lookup, dict(out_ld=9), "out"),
    (_grad, dict(dy_ld=25), "dy"),
    (_grad, dict(dw_ld=10), "dw"),
    (_grad, dict(dw=View((10, 8), (8, 1), np.float32)), "dw"),
])
def test_views_that_span_too_little_are_still_refused(call, kw, what):
    with pytest.raises(ValueError, match=what):
        call(**kw)


def test_last_row_need_not_be_a_whole_stride():
    with pytest.raises(AncoraError, match="ctx"):
        _lookup(table=View((10, 8), (16, 1), np.uint16), table_ld=16, V=10)    # 9 * 16 + 8 elements
