"""Embedding lookup and its gradient (TEST INFRASTRUCTURE): the lookup in numpy float32, bit for bit what the
kernel computes; the gradient in float64 with the size of the terms, for error bounds.  The reference has no
counterpart."""
import numpy as np

from . import bf16


def lookup(table, ids, scale, out_dtype):
    """table: float32 values.  Returns float32 values or bf16 bits; rows of negative or too large ids are zero."""
    ids = np.asarray(ids, np.int64)
    live = (ids >= 0) & (ids < table.shape[0])
    rows = np.where(live[:, None], table[np.where(live, ids, 0)] * np.float32(scale), np.float32(0))
    rows = rows.astype(np.float32)
    return bf16.rne_bits(rows) if out_dtype == "bf16" else rows


def grad(dy, ids, V, scale, base=None, padding_idx=None):
    """(dW, count, magnitude) in float64: scale * sum of dy over the tokens of each row, plus ``base`` when
    given; tokens per row; scale * sum of |dy|."""
    ids = np.asarray(ids, np.int64)
    live = (ids >= 0) & (ids < V)
    if padding_idx is not None and padding_idx >= 0:
        live &= ids != padding_idx
    D = dy.shape[1]
    total, mag = np.zeros((V, D)), np.zeros((V, D))
    x = np.asarray(dy, np.float64)[live]
    np.add.at(total, ids[live], x)
    np.add.at(mag, ids[live], np.abs(x))
    s = float(np.float32(scale))
    total *= s
    if base is not None:
        total += np.asarray(base, np.float64)
    return total, np.bincount(ids[live], minlength=V), abs(s) * mag
