"""The paged 4-bit KV cache in 64 bits (numpy): what ibh_kv4_* (include/ibhip.h)
compute, written from the format's definition.  No counterpart in the reference."""
from __future__ import annotations

import numpy as np

PAGE = 64


def places(hd):
    """Byte and shift of every (position, dim) of a head's part of a page, for keys and values, and the halfword of
    its (scale, mid) pair."""
    t, d = np.meshgrid(np.arange(PAGE), np.arange(hd), indexing="ij")
    e, slot = d % 16, 4 * (t % 16) + t // 16
    f = slot % 16
    k = (t // 32 * (hd // 64) + d // 64) * 1024 + (d % 64 // 16 * 16 + t % 16) * 16 + t // 16 % 2 * 8 + e // 8 * 4 + e % 4
    v = 36 * hd + d // 32 * 1024 + (slot // 16 * 16 + d % 16) * 16 + d % 32 // 16 * 8 + f // 8 * 4 + f % 4
    pair = (d // 64 * 64 + slot) * 2
    return (k, 4 * (e // 4 % 2), 16 * hd + pair), (v, 4 * (f // 4 % 2), 34 * hd + pair)


def quantise(x):
    """(codes 0..15, scale, mid) of groups of 64 along the last axis; the format's own roundings, the rest in 64 bits."""
    g = np.clip(np.asarray(x, np.float32), -65504, 65504).reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    scale = ((hi - lo) / np.float32(15)).astype(np.float16)
    mid = (lo + np.float32(8) * scale.astype(np.float32)).astype(np.float16)
    s, m = scale.astype(np.float64), mid.astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint((g.astype(np.float64) - m) / s), -8, 7), 0)
    return (np.nan_to_num(c) + 8).astype(np.uint8), scale[..., 0], mid[..., 0]


def held(x):
    """What x is held as."""
    c, s, m = quantise(x)
    return (m[..., None].astype(np.float64) + s[..., None].astype(np.float64) * (c.astype(np.float64) - 8)).reshape(x.shape)


def store(pool, pages, n_kv, hd, k, v, first):
    """Writes rows k, v [n, n_kv * hd] at positions first .. into a sequence's pages (pool [n_pages, bytes], in place)."""
    P = places(hd)
    for i in range(k.shape[0]):
        pos = first + i
        if pos < 0:
            continue
        for h in range(n_kv):
            part = pool[pages[pos // PAGE]].reshape(n_kv, -1)[h]
            t = pos % PAGE
            for (at, shift, pair), x in zip(P, (k, v)):
                c, s, m = quantise(x[i, h * hd:(h + 1) * hd])
                np.bitwise_and.at(part, at[t], (0xF0 >> shift[t]).astype(np.uint8))
                np.bitwise_or.at(part, at[t], (c.reshape(-1) << shift[t]).astype(np.uint8))
                half = part.view(np.uint16)
                half[pair[t][::64]] = s.view(np.uint16)
                half[pair[t][::64] + 1] = m.view(np.uint16)


def load(pool, pages, n_kv, hd, n):
    """K, V [n_kv, n, hd] in 64 bits, the values of a sequence's first n positions."""
    out = []
    for at, shift, pair in places(hd):
        x = pool[np.asarray(pages[:(n + PAGE - 1) // PAGE], int)].reshape(-1, n_kv, 72 * hd)
        c = (x[:, :, at] >> shift.astype(np.uint8)) & 15
        half = x.view(np.float16).astype(np.float64)
        y = half[:, :, pair + 1] + half[:, :, pair] * (c.astype(np.float64) - 8)
        out.append(y.transpose(1, 0, 2, 3).reshape(n_kv, -1, hd)[:, :n])
    return out


def attend(q, K, V, n_q):
    """(out [n_q, heads * hd], probabilities summed over the rows [n_kv, n], largest sum |q k| / sqrt(hd))."""
    n_kv, n, hd = K.shape
    q = np.asarray(q, np.float64).reshape(n_q, n_kv, -1, hd)
    out, w, top = np.zeros(q.shape), np.zeros((n_kv, n)), 0.0
    for i in range(n_q):
        m = n - n_q + i + 1
        if m <= 0:
            continue
        for h in range(n_kv):
            s = q[i, h] @ K[h, :m].T / np.sqrt(hd)
            e = np.exp(s - s.max(-1, keepdims=True))
            p = e / e.sum(-1, keepdims=True)
            out[i, h] = p @ V[h, :m]
            w[h, :m] += p.sum(0)
            a = np.abs(q[i, h]) @ np.abs(K[h, :m]).T / np.sqrt(hd)
            if np.isfinite(a).any():
                top = max(top, float(a[np.isfinite(a)].max()))
    return out.reshape(n_q, -1), w, top


def keep(w, n, budget, sink, recent):
    """The positions kept of a head whose first n weights are w[:n]."""
    if n <= budget:
        return np.arange(n)
    c = np.arange(sink, n - recent)
    r = np.where(np.isnan(w[c]), -np.inf, w[c].astype(np.float64))
    nan = np.isnan(w[c])
    order = c[np.lexsort((c, nan, -r))][:budget - sink - recent]
    return np.concatenate([np.arange(sink), np.sort(order), np.arange(n - recent, n)])
