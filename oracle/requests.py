"""The operators around a batch's projections in plain numpy and 64 bits: the RMS norm with its 8-bit codes, low-rank
adapters, log-probabilities.  Written from their definitions; what a definition rounds to fp32 is rounded there."""
import numpy as np

GROUP = 128


def norm(x, delta, weight, eps):
    """(h, p, r): the sum and the products as they are rounded, and the row's factor."""
    x, weight = np.asarray(x, np.float32), np.asarray(weight, np.float32)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        h = x if delta is None else x + np.asarray(delta, np.float32)
        p = h * weight
        r = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    return h, p, np.where(np.isfinite(h).all(-1, keepdims=True), r, np.nan)


def codes(p, r):
    """(q, s) of one row's products: s in 64 bits, q exactly, by whole numbers."""
    q, s = np.zeros(p.shape, np.int8), []
    for at in range(0, p.size, GROUP):
        part = p[at:at + GROUP].astype(np.float64)
        top = np.abs(part).max()
        if not np.isfinite(top) or not np.isfinite(r):
            s.append(np.nan)
        elif top * r < 1e-10:
            s.append(1e-10)
        else:
            s.append(top * r / 127)
            # 2 * 127 |p| against the odd multiples of max|p|, both as whole numbers of 2^-149 / 2^104: no rounding
            m = int(np.ldexp(top, 149))
            for i, v in enumerate(part):
                c = (254 * int(np.ldexp(abs(v), 149)) + m) // (2 * m)
                q[at + i] = -c if v < 0 else c
    return q, np.array(s)


def lora(base, x, a, b, ids, scales=None, ranks=None):
    """(out, size): out in 64 bits and the sum of the absolute products that went into it."""
    x, a, b = (np.asarray(t, np.float64) for t in (x, a, b))
    out = np.zeros((x.shape[0], b.shape[1])) if base is None else np.asarray(base, np.float64).copy()
    size = np.zeros_like(out)
    for i, k in enumerate(ids):
        if k < 0:
            continue
        r = a.shape[1] if ranks is None else ranks[k]
        if k >= a.shape[0] or r < 0 or r > a.shape[1]:
            out[i] = np.nan
            continue
        s = 1.0 if scales is None else float(scales[k])
        out[i] += b[k, :, :r] @ (a[k, :r] @ x[i]) * s
        size[i] = np.abs(b[k, :, :r]) @ (np.abs(a[k, :r]) @ np.abs(x[i])) * abs(s)
    return out, size


def logprobs(z, tokens, k):
    """(log-probabilities of tokens [B, n], entropy, ids, their log-probabilities, log sum exp(z - max)), which is taken
    off z - max and not added to max: 64 bits of a logit of -3.4e38 hold no logarithm beside it."""
    z = np.asarray(z, np.float64)
    B, V = z.shape
    tokens = np.asarray(tokens).reshape(B, -1)
    lp, ent = np.full(tokens.shape, np.nan), np.full(B, np.nan)
    ids, top, logs = np.full((B, k), -1, np.int32), np.full((B, k), np.nan), np.full(B, np.nan)
    for i in range(B):
        if np.isnan(z[i]).any() or (z[i] == np.inf).any():
            continue
        inside = (tokens[i] >= 0) & (tokens[i] < V)
        m = z[i].max()
        top[i] = -np.inf
        if m == -np.inf:
            lp[i, inside], ent[i] = -np.inf, 0
            continue
        d = z[i] - m
        e = np.exp(d)
        logs[i] = np.log(e.sum())
        held = e > 0
        ent[i] = logs[i] - (e[held] * d[held]).sum() / e.sum()
        lp[i, inside] = d[tokens[i][inside]] - logs[i]
        order = np.argsort(-z[i], kind="stable")[:k]
        order = order[z[i][order] > -np.inf]
        ids[i, :order.size], top[i, :order.size] = order, d[order] - logs[i]
    return lp, ent, ids, top, logs
