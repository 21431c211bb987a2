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
