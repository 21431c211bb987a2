"""The norm's codes beside those that the activations' quantizer makes of the norm's fp32 output."""
import numpy as np
import pytest
import torch

from libinferbit_amd import ops
from oracle import requests as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("N", [1, 100, 128, 130, 1000, 4096, 5632, 14336, 17000])
def test_codes_beside_the_quantizers(N):
    """The quantizer takes y (its own two roundings, and two of the largest of 128) over a scale and its inverse, a product
    and a sum, one rounding each: 7 half steps of a code up to 127 and one of 128, 1017 U in all."""
    B, eps = 6, 1e-5
    rng = np.random.default_rng(N)
    x = (rng.standard_normal((B, N)) * np.exp(rng.standard_normal(N))).astype(np.float32)
    d, w = (rng.standard_normal((B, N)) * 0.3).astype(np.float32), (rng.random(N) + 0.5).astype(np.float32)
    x[1], d[1] = 0, 0                                    # codes 0 and 1e-10
    x[2, :128], d[2, :128] = x[2, :128] * np.float32(1e-12), 0      # such a group beside others
    x[3] = rng.integers(-127, 128, N) * np.float32(0.5)  # borders, where y's own rounding decides
    x[3, ::128], d[3] = 127, 0
    gpu = lambda t: torch.from_numpy(t).cuda()
    G = (N + 127) // 128
    y, q, s = torch.empty(B, N, device="cuda"), torch.empty(B, N, dtype=torch.int8, device="cuda"), torch.empty(B, G, device="cuda")
    ops.add_rmsnorm(y, gpu(x), gpu(w), eps, delta=gpu(d), q=q, s=s)
    q2, s2 = torch.empty(B, N, dtype=torch.int8, device="cuda"), torch.empty(B, G, device="cuda")
    for i in range(B):
        assert ops.quantize_input_int8_g128(y[i], q2[i], s2[i], N) == G
    q, s, q2, s2 = (t.cpu().numpy() for t in (q, s, q2, s2))
    # s is rounded once and within a hair, the quantizer's from y's two roundings and its own
    np.testing.assert_allclose(s, s2, rtol=4.1 * U)
    _, p, r = R.norm(x, d, w, eps)
    p = np.pad(p.astype(np.float64), ((0, 0), (0, G * 128 - N))).reshape(B, G, 128)
    top = np.abs(p).max(-1, keepdims=True)
    part = np.abs(127 * p / np.where(top == 0, 1, top)).reshape(B, -1)[:, :N]
    clear = np.abs(part - np.floor(part) - 0.5) > 1017 * U
    assert clear.mean() > 0.4
    np.testing.assert_array_equal(q[clear], q2[clear])
    assert (np.abs(q.astype(int) - q2) <= 1).all()
    zero = top[:, :, 0] * r < 1e-10                      # where both leave nothing, and 1e-10
    np.testing.assert_array_equal(s == np.float32(1e-10), zero)
    assert zero[1].all() and not q[np.repeat(zero, 128, 1)[:, :N]].any()
