"""Accuracy of the paged 4-bit cache's attention where its inputs are uneven, and
what its weights add up to.  Bounds are written with each test; e = 2^-24 is a
rounding of fp32."""
import numpy as np
import pytest
import torch

from oracle import kv4 as R
from test_kv4_gpu import Made, device_errors, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# ── accumulated weights ──────────────────────────────────────────────────────
@pytest.mark.parametrize("n_q,t", [(1, 150), (1, 1100), (2, 1100), (6, 150), (6, 1100), (9, 150), (9, 1100), (70, 1100)])
@pytest.mark.parametrize("size", [4e3, 2.0 ** 23, 2.0 ** 26, 1e20])
def test_weights_of_tied_scores(ops, n_q, t, size):
    """Every score of a row is the same large number, so each of the c positions that a query sees has the weight 1 / c
    exactly.  c is summed without rounding; its reciprocal and product (2 e each) and the sum over the rows (an e a
    row) are rounded."""
    print(f"case ties n_q={n_q} t={t} size={size}", flush=True)
    rng = np.random.default_rng(61)
    n_heads, n_kv, hd = 8, 2, 64
    m = Made(ops, rng, [t], n_kv, hd)
    m.k[0] = np.ones((t, n_kv * hd), np.float32)                  # constant groups: scale 0
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = torch.full((1, n_q, n_heads * hd), float(size), device="cuda")
    q[:, :, 5 * hd:6 * hd] *= -1
    out, w = torch.empty_like(q), torch.zeros(1, n_kv, m.table.shape[1] * 64, device="cuda")
    ops.kv4_attn(out, q, m.cache, n_heads, weights_in=w, weights_out=w)
    grp = n_heads // n_kv
    want = np.zeros(t)
    for i in range(n_q):
        want[:t - n_q + i + 1] += grp / (t - n_q + i + 1)
    got = w.cpu().numpy()[0]
    assert (np.abs(got[:, :t] - want) <= (4 + n_q * grp) * 2.0 ** -24 * want).all(), (got[:, 0], want[0])
    assert (got[:, t:] == 0).all()


# ── values of uneven size ────────────────────────────────────────────────────
def parts(m, i, q, n_q, n_heads):
    """Row by row (query, head): the output's 64-dim groups in 64 bits, the sums of p |v| over each group, the largest
    sum |q k| / sqrt(hd)."""
    K, V = m.loaded(i)
    hd, grp = m.hd, n_heads // m.n_kv
    q = np.asarray(q, np.float64).reshape(n_q, n_heads, hd)
    out, size, top = np.zeros((n_q, n_heads, hd // 64, 64)), np.zeros((n_q, n_heads, hd // 64)), 0.0
    for a in range(n_q):
        n = K.shape[1] - n_q + a + 1
        for h in range(n_heads):
            k, v = K[h // grp, :n], V[h // grp, :n].reshape(n, -1, 64)
            s = k @ q[a, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[a, h] = np.tensordot(p, v, 1)
            size[a, h] = p @ np.linalg.norm(v, axis=2)
            top = max(top, float((np.abs(k) @ np.abs(q[a, h])).max() / np.sqrt(hd)))
    return out, size, top


@pytest.mark.parametrize("groups", [slice(0, 1), slice(0, None)])
@pytest.mark.parametrize("n_heads,n_kv,n_q,t,hd", [
    (8, 2, 1, 330, 64), (8, 2, 12, 330, 64), (8, 2, 12, 330, 128), (8, 2, 70, 1500, 128), (8, 2, 12, 330, 192),
    (64, 64, 40, 130, 64), (64, 64, 40, 1600, 128), (64, 64, 34, 700, 256)])   # blocks of several pages: one split, and more
def test_large_values_behind_small_ones(ops, n_heads, n_kv, n_q, t, hd, groups):
    """The first page holds only values of 2^-14, which every query looks at; from the second page on there are others
    of 2^10 (in the first 64 dims, or in all) that none looks at, with probabilities below 2^-60.  A score is off by
    8 e S (S = sum |q k| / sqrt(hd)) and moves its probability by that share, and the normaliser by as much: 16 e
    max(1, S) of sum p |v| of each 64 dims on their own."""
    print(f"case behind {n_heads}/{n_kv} n_q={n_q} t={t} hd={hd} {groups}", flush=True)
    rng = np.random.default_rng(43 + hd)
    m = Made(ops, rng, [t], n_kv, hd)
    u = rng.choice([-1.0, 1.0], hd)
    seen = (np.arange(t) % 64 < 23) & (np.arange(t) < 250)
    seen[:64] = True
    k = rng.standard_normal((t, n_kv, hd)) * 0.1 + np.where(seen, 3.0, -3.0)[:, None, None] * u
    v = rng.standard_normal((t, n_kv, hd)) * 2.0 ** -14
    v.reshape(t, n_kv, -1, 64)[~seen, :, groups] *= 2.0 ** 24
    m.k[0], m.v[0] = (x.reshape(t, -1).astype(np.float32) for x in (k, v))
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = rng.standard_normal((1, n_q, n_heads, hd)) * 0.1 + 10 / np.sqrt(hd) * u
    q = torch.from_numpy(q.reshape(1, n_q, n_heads * hd).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    ops.kv4_attn(out, q, m.cache, n_heads)
    want, size, top = parts(m, 0, q[0].cpu().numpy(), n_q, n_heads)
    err = np.linalg.norm(out.cpu().numpy().reshape(want.shape) - want, axis=-1)
    tol = 16 * 2.0 ** -24 * max(1.0, top)
    print("err / size", (err / size).max(), "tol", tol, flush=True)
    assert (err <= tol * size).all()


def test_maxima_that_creep_up(ops):
    """Scores of a row rise by 0.9 bits a page, while other rows of its wavefront jump by 8.7 bits on a page of their own;
    the first 64 dims' values are 2^10 on the first page, all but out of sight at the end, and 2^-14 behind it.  One
    split.  Bound as above."""
    rng = np.random.default_rng(44)
    n, n_kv, hd, n_q, pages = 64, 8, 128, 40, 32
    t = pages * 64
    m = Made(ops, rng, [t] + [1] * (n - 1), n_kv, hd)
    page = np.arange(t) // 64
    k = rng.integers(-8, 8, (t, n_kv, hd)).astype(np.float32)        # held exactly: scale 1, mid 0
    for i in range(n_q):                                             # query i: a jump on pages 1 + i % 15 and 15 behind
        k[:, :, i] = ((page >= 1 + i % 15) * 1 + (page >= 16 + i % 15) * 1)[:, None]
    k[:, :, 15], k[:, :, 31] = 0, 0                                  # two rows that do not jump
    k[:, :, 62], k[:, :, 63], k[:, :, 126], k[:, :, 127] = -8, 7, -8, 7
    k[:, :, 64], k[:, :, 65] = (page % 16 - 8)[:, None], (page // 16)[:, None]
    v = rng.standard_normal((t, n_kv, 2, 64))
    v[:, :, 0] *= np.where(page == 0, 2.0 ** 10, 2.0 ** -14)[:, None, None]
    m.k[0], m.v[0] = k.reshape(t, -1), v.reshape(t, -1).astype(np.float32)
    one = ops.Kv4Cache(m.dpool, m.dtable[:1], m.dlens[:1], n_kv, hd)
    ops.kv4_append(one, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = np.zeros((n, n_q, n_kv, hd), np.float32)
    for i in range(n_q):
        q[:, i, :, i] = 6 * np.sqrt(hd)
    q[..., 64], q[..., 65] = 0.62 * np.sqrt(hd), 16 * 0.62 * np.sqrt(hd)
    out = torch.empty(n, n_q, n_kv * hd, device="cuda")
    ops.kv4_attn(out, torch.from_numpy(q.reshape(n, n_q, -1)).cuda(), m.cache, n_kv)
    assert (m.loaded(0)[0] == k.transpose(1, 0, 2)).all()
    want, size, top = parts(m, 0, q[0], n_q, n_kv)
    err = np.linalg.norm(out[0].cpu().numpy().reshape(want.shape) - want, axis=-1)
    tol = 12 * 2.0 ** -24 * max(1.0, top)
    print("err / size", (err / size).max((1, 2)), "tol", tol, flush=True)
    assert (err <= tol * size).all()


@pytest.mark.parametrize("n_heads,n_kv,n_q", [(64, 16, 1), (16, 4, 6), (16, 4, 64)])
def test_probabilities_are_not_cut_short(ops, n_heads, n_kv, n_q):
    """All positions hold one value vector, -2 in one dim of each 64 and 7/4 (scale 1/4, mid 0) in the others, so the
    output is that vector whatever the probabilities are, and what it lacks is what p * scale lost.  Roundings to
    nearest leave no mean: at most 4 e a row from its sums, and less than e in the mean over 64 rows and more."""
    rng = np.random.default_rng(71)
    hd, t = 64, 128
    m = Made(ops, rng, [t], n_kv, hd)
    v = np.where(np.arange(n_kv * hd) % 64 == 9, -2.0, 1.75)
    m.v[0] = np.tile(v, (t, 1)).astype(np.float32)
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = torch.from_numpy(rng.standard_normal((1, n_q, n_heads * hd)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    ops.kv4_attn(out, q, m.cache, n_heads)
    r = out.cpu().numpy().astype(np.float64).reshape(-1, 64) / v[:64] - 1
    print("mean", r.mean(), "largest", np.abs(r).max(), flush=True)
    assert abs(r.mean()) <= 2.0 ** -24


# ── queries with one large channel ───────────────────────────────────────────
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n_heads,n_kv,hd,n_q,t", [(8, 2, 128, 1, 700), (8, 2, 128, 1, 4096), (8, 2, 64, 2, 1100), (8, 2, 128, 6, 700),
                                                   (6, 2, 192, 5, 300), (4, 2, 256, 8, 300), (8, 2, 128, 9, 700)])
@pytest.mark.parametrize("size", [30.0, 300.0, 3000.0])
def test_query_with_an_outlier_channel(ops, n_heads, n_kv, hd, n_q, t, size, weights):
    """One channel of the query is large, and the keys hold 0 there (scale 1/4, mid 0), so the others make the score.
    A score is off by 8 e S (S = sum |q k| / sqrt(hd)): 16 e max(1, S) of sum p |v|."""
    print(f"case outlier {n_heads}/{n_kv} hd={hd} n_q={n_q} t={t} size={size} weights={weights}", flush=True)
    rng = np.random.default_rng(hd + n_q)
    m = Made(ops, rng, [t], n_kv, hd)
    k = np.clip(rng.standard_normal((t, n_kv, hd // 64, 64)), -2, 1.75)
    k[..., 0], k[..., 1] = -2, 1.75
    k[:, :, 0, 7] = 0
    m.k[0] = k.reshape(t, -1).astype(np.float32)
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = rng.standard_normal((1, n_q, n_heads, hd))
    q[..., 7] = size * rng.uniform(0.7, 1.4, q.shape[:-1])
    q = torch.from_numpy(q.reshape(1, n_q, n_heads * hd).astype(np.float32)).cuda()
    out, w = torch.empty_like(q), torch.zeros(1, n_kv, m.table.shape[1] * 64, device="cuda")
    ops.kv4_attn(out, q, m.cache, n_heads, **(dict(weights_in=w, weights_out=w) if weights else {}))
    want, size, top = parts(m, 0, q[0].cpu().numpy(), n_q, n_heads)
    assert (m.loaded(0)[0][:, :, 7] == 0).all()
    err = np.linalg.norm(out.cpu().numpy().reshape(want.shape) - want, axis=-1)
    tol = 16 * 2.0 ** -24 * max(1.0, top)
    print("err / size", (err / size).max(), "tol", tol, flush=True)
    assert (err <= tol * size).all()
    if weights:
        p = R.attend(q[0].cpu().numpy(), *m.loaded(0), n_q)[1]
        assert (np.abs(w[0, :, :t].cpu().numpy() - p) <= (tol + 2.0 ** -22) * p + 2.0 ** -120).all()


@pytest.mark.parametrize("n_heads,n_kv,hd,n_q,t", [(8, 2, 128, 1, 700), (8, 2, 64, 6, 300), (8, 2, 128, 9, 700)])
@pytest.mark.parametrize("size", [30.0, 3000.0])
def test_query_with_an_outlier_channel_beside_middles(ops, n_heads, n_kv, hd, n_q, t, size):
    """The same where the keys' other channels lie around 3/2, so that 0 is -8 steps from a middle: a score is the sum
    over its 64-dim groups of mid * sum q and scale * sum q (code - 8), which cancel.  Each is off by 8 e of its own
    absolute sum, A = sum (|mid| sum |q| + scale sum |q (code - 8)|) / sqrt(hd): 16 e max(1, A) of sum p |v|."""
    print(f"case beside middles {n_heads}/{n_kv} hd={hd} n_q={n_q} t={t} size={size}", flush=True)
    rng = np.random.default_rng(hd + n_q)
    m = Made(ops, rng, [t], n_kv, hd)
    k = np.clip(rng.standard_normal((t, n_kv, hd)) * 0.5 + 1.5, 0.01, 3)
    k[:, :, 7] = 0
    m.k[0] = k.reshape(t, -1).astype(np.float32)
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = rng.standard_normal((1, n_q, n_heads, hd))
    q[..., 7] = size * rng.uniform(0.7, 1.4, q.shape[:-1])
    q = torch.from_numpy(q.reshape(1, n_q, n_heads * hd).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    ops.kv4_attn(out, q, m.cache, n_heads)
    want, sums, _ = parts(m, 0, q[0].cpu().numpy(), n_q, n_heads)
    c, s, mid = (x.astype(np.float64) for x in R.quantise(m.k[0]))
    aq = np.abs(q[0].cpu().numpy().astype(np.float64)).reshape(n_q, n_kv, -1, hd // 64, 64)
    c, s, mid = c.reshape(t, n_kv, hd // 64, 64), s.reshape(t, n_kv, -1), mid.reshape(t, n_kv, -1)
    top = 0.0
    for h in range(n_kv):
        a = np.einsum("tg,qrg->tqr", np.abs(mid[:, h]), aq[:, h].sum(-1)) + np.einsum("tg,tgd,qrgd->tqr", s[:, h], np.abs(c[:, h] - 8), aq[:, h])
        top = max(top, a.max() / np.sqrt(hd))
    err = np.linalg.norm(out.cpu().numpy().reshape(want.shape) - want, axis=-1)
    tol = 16 * 2.0 ** -24 * max(1.0, top)
    print("err / size", (err / sums).max(), "tol", tol, flush=True)
    assert (err <= tol * sums).all()
