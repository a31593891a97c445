"""Log probabilities, entropy and best alternatives of class rows in fp64 (the oracle of lmi_class_logprobs)."""
import numpy as np


def evidence(x, labels=None, top=0, activation="softmax"):
    """x (..., C) any float array, labels (...) integers.  Returns dict(logprob, entropy, top_logprob, top_index)."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        if activation == "softmax":
            m = x.max(-1, keepdims=True)                       # NaN if any value is
            empty = m == -np.inf
            z = x - np.where(empty, 0.0, m)                    # +inf - +inf = NaN, as the formula says
            e = np.exp(z)
            s = e.sum(-1, keepdims=True)
            lp = np.where(empty, -np.inf, z - np.log(s))
            p = np.where(empty, 0.0, e / s)
            entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), np.where(np.isnan(p), np.nan, 0.0)).sum(-1)
        else:
            if activation == "sigmoid":
                lp, ln = -np.logaddexp(0.0, -x), -np.logaddexp(0.0, x)
                p, q = np.exp(lp), np.exp(ln)
            else:
                p, q = x, 1.0 - x
                lp, ln = np.log(p), np.log1p(-p)
            h = -np.where(p == 0, 0.0, p * lp) - np.where(q == 0, 0.0, q * ln)
            entropy = h.sum(-1)
    out = {"entropy": entropy}
    if labels is not None:
        labels = np.asarray(labels)
        ok = (labels >= 0) & (labels < x.shape[-1])
        at = np.where(ok, labels, 0).astype(np.int64)
        out["logprob"] = np.where(ok, np.take_along_axis(lp, at[..., None], -1)[..., 0], np.nan)
    if top:
        # NaN first, then by value, equal values by class
        key = np.where(np.isnan(x), np.inf, x)
        order = np.lexsort((np.broadcast_to(np.arange(x.shape[-1]), x.shape), -key, ~np.isnan(x)), axis=-1)[..., :top]
        out["top_index"] = order
        out["top_logprob"] = np.take_along_axis(lp, order, -1)
    return out
