"""Global gradient norm and clipping factor in float64 (TEST INFRASTRUCTURE).

norm = scale * sqrt(sum of squares), factor = scale * min(1, max_norm / (norm + eps)); max_norm = inf never
clips.  The reference has no counterpart."""
import math

import numpy as np


def norm_and_factor(grads, max_norm, scale=1.0, eps=1e-6):
    """grads: arrays whose values are exact in float64."""
    with np.errstate(over="ignore", invalid="ignore"):
        parts = [float(np.dot(x, x)) for x in (np.asarray(g, np.float64).reshape(-1) for g in grads)]
    sq = math.fsum(parts) if all(math.isfinite(p) for p in parts) else float(np.sum(parts))
    norm = scale * math.sqrt(sq) if sq == sq else math.nan
    den = norm + eps
    if math.isinf(max_norm) or den == 0.0:
        c = 1.0
    elif math.isnan(den):
        c = math.nan
    else:
        c = min(1.0, max_norm / den)
    return norm, scale * c
