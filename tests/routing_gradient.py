"""The router's gradient in float64 by sums of terms that do not cancel, for logits whose scores are far apart or far below
1 (tests/routing.py's differences lose in float64 what one expert leaves of a softmax). tests/test_routing_gradient.py
holds it to the definition in many digits."""
import numpy as np

LEAST_LOG = -745.14  # e to this and less is 0 in 64 bits: no score


def log_scores(x, scoring):
    """log p, and log (1 - p) for sigmoids."""
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if scoring == "sigmoid":
            rest = np.log1p(np.exp(-np.abs(x)))
            p, q = np.minimum(x, 0.0) - rest, np.minimum(-x, 0.0) - rest
        else:
            top = np.where(x.max(axis=1, keepdims=True) == -np.inf, 0.0, x.max(axis=1, keepdims=True))
            total = np.exp(x - top).sum(axis=1, keepdims=True)
            p = x - top - np.log(np.where(total == 0.0, 1.0, total))
            q = np.zeros_like(p)
    return np.where(p < LEAST_LOG, -np.inf, p), q


def grad(x, scoring, ids, dw, renorm, scale=1.0):
    """(the gradient, the sum of the magnitudes of its terms):
    renormalised      w_s (1 - p_s, of sigmoids) sum_r w_r (d_s - d_r)
    softmax, chosen   p_s (sum_r p_r (d_s - d_r) + d_s (the sum of the scores that were not chosen))
    softmax, others  -p_e sum_r p_r d_r
    sigmoid           d_s p_s (1 - p_s)
    with an expert's slots added up."""
    lp, lq = log_scores(x, scoring)
    p, q = np.exp(lp), np.exp(lq)
    out, size = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(len(x)):
        slots = [(int(e), float(d)) for e, d in zip(ids[t], dw[t]) if 0 <= e < x.shape[1]]
        if not slots:
            continue
        e = np.array([s[0] for s in slots])
        d = np.array([s[1] for s in slots])
        if renorm:
            top = lp[t, e].max()
            w = np.exp(lp[t, e] - (0.0 if top == -np.inf else top))
            w = w / (w.sum() or 1.0)
            terms = (w[:, None] * w[None, :]) * (d[:, None] - d[None, :])
            for i, s in enumerate(e):
                out[t, s] += q[t, s] * terms[i].sum()
                size[t, s] += q[t, s] * np.abs(terms[i]).sum()
        elif scoring == "sigmoid":
            for s, v in slots:
                out[t, s] += v * p[t, s] * q[t, s]
                size[t, s] += abs(v) * p[t, s] * q[t, s]
        else:
            once = np.unique(e)
            back = np.array([d[e == s].sum() for s in once])
            rest = np.delete(p[t], once).sum()
            terms = p[t, once][None, :] * (back[:, None] - back[None, :])
            out[t] = -p[t] * (p[t, once] * back).sum()
            size[t] = p[t] * (p[t, once] * np.abs(back)).sum()
            out[t, once] = p[t, once] * (terms.sum(1) + back * rest)
            size[t, once] = p[t, once] * (np.abs(terms).sum(1) + np.abs(back) * rest)
    return out * scale, size * scale
