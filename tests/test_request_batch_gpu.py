"""A batch through the operators around its projections as a model runs them: an adapter takes what its projection takes,
the normed row, so the norm gives fp32 beside the codes; the adapters add in place, with ranks of their own.  Each stage
is held against 64 bits of what it was given."""
import numpy as np
import pytest
import torch

import libinferbit_amd as L
from libinferbit_amd import ops
from oracle import pyoracle as O
from oracle import requests as R

pytestmark = pytest.mark.gpu
U, EPS = 2.0 ** -24, 1e-5
RANKS = [16, 3, 0, 9, 16, 1]


class Batch:
    """B rows of width N over a vocabulary V, six adapters.  Up to 32 rows are a step of requests through W4A8 and INT8
    columns, more are packed prompts through the INT8 GEMM."""

    def __init__(self, B, N, V, seed):
        L.ops.init(0)
        rng = np.random.default_rng(seed)
        self.B, self.N, self.V, self.rng, self.coded = B, N, V, rng, B <= 32
        self.w, ws = O.quantize(4 if self.coded else 8, (rng.standard_normal((N, N)) * 0.05).astype(np.float32))
        self.head, hs = O.quantize(8, (rng.standard_normal((V, N)) * 0.05).astype(np.float32))
        self.n1, self.n2 = (rng.random((2, N)) + 0.5).astype(np.float32)
        g = torch.Generator().manual_seed(seed)
        n = len(RANKS)
        self.a, self.b, self.scales = (torch.randn(n, 16, N, generator=g) / N ** 0.5).half(), (torch.randn(n, N, 16, generator=g) / 4).half(), torch.rand(n, generator=g) + 0.5
        gpu = lambda t: torch.from_numpy(t).cuda()
        self.d = dict(w=gpu(self.w), ws=gpu(ws.view(np.int16)), head=gpu(self.head), hs=gpu(hs.view(np.int16)), n1=gpu(self.n1),
                      n2=gpu(self.n2), a=self.a.cuda(), b=self.b.cuda(), scales=self.scales.cuda(), ranks=torch.tensor(RANKS, dtype=torch.int32, device="cuda"))
        # the weights in 64 bits
        codes = np.stack([self.w & 15, self.w >> 4], -1).reshape(N, N).astype(np.float64) - 8 if self.coded else self.w.reshape(N, N).view(np.int8).astype(np.float64)
        self.w64 = codes * ws.view(np.float16).astype(np.float64)[:, None]
        self.head64 = self.head.reshape(V, N).view(np.int8).astype(np.float64) * hs.view(np.float16).astype(np.float64)[:, None]
        f = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="cuda")
        self.t = dict(x=f(B, N), delta=f(B, N), ids=f(B, dtype=torch.int32), tok=f(B, 2, dtype=torch.int32), h1=f(B, N), y=f(B, N), q=f(B, N, dtype=torch.int8),
                      s=f(B, (N + 127) // 128), o=f(B, N), h2=f(B, N), z=f(B, N), logits=f(B, V), lp=f(B, 2), ent=f(B), top=f(B, 6, dtype=torch.int32), top_lp=f(B, 6))
        self.fill()

    def fill(self):
        B, N, rng, t = self.B, self.N, self.rng, self.t
        t["x"].copy_(torch.from_numpy(rng.standard_normal((B, N)).astype(np.float32) * 2))
        t["delta"].copy_(torch.from_numpy(rng.standard_normal((B, N)).astype(np.float32)))
        t["ids"].copy_(torch.from_numpy(rng.integers(-1, len(RANKS), B).astype(np.int32)))
        t["tok"].copy_(torch.from_numpy(rng.integers(0, self.V, (B, 2)).astype(np.int32)))

    def run(self):
        B, N, V, d, t = self.B, self.N, self.V, self.d, self.t
        product = ops.matmul_int8_batch if self.coded else ops.gemm_int8
        ops.add_rmsnorm(t["y"], t["x"], d["n1"], EPS, delta=t["delta"], h=t["h1"], **(dict(q=t["q"], s=t["s"]) if self.coded else {}))
        if self.coded:
            ops.matmul_w4a8_batch(t["o"], d["w"], d["ws"], t["q"], t["s"], N, N, B, N)
        else:
            product(t["o"], d["w"], d["ws"], t["y"], N, N, B, N)
        ops.lora(t["o"], t["y"], d["a"], d["b"], t["ids"], base=t["o"], scales=d["scales"], ranks=d["ranks"])
        ops.add_rmsnorm(t["z"], t["o"], d["n2"], EPS, delta=t["h1"], h=t["h2"])
        product(t["logits"], d["head"], d["hs"], t["z"], V, N, B, V)
        ops.logprobs(t["lp"], t["logits"], t["tok"], entropy=t["ent"], top_ids=t["top"], top_logprobs=t["top_lp"])

    def check(self):
        t = {k: v.cpu().numpy() for k, v in self.t.items()}
        h, p, r = R.norm(t["x"], t["delta"], self.n1, EPS)
        np.testing.assert_array_equal(t["h1"], h)
        np.testing.assert_allclose(t["y"], p.astype(np.float64) * r, rtol=2.01 * U)
        held = t["y"].astype(np.float64)
        if self.coded:
            for i in range(self.B):
                q, s = R.codes(p[i], r[i, 0])
                np.testing.assert_array_equal(t["q"][i], q)
                np.testing.assert_allclose(t["s"][i], s, rtol=3.01 * U)
            held = t["q"].astype(np.float64) * np.repeat(t["s"].astype(np.float64), 128, 1)[:, :self.N]
        # the projections hold 1e-4 of their largest; of the adapters' sums of 16 N products each is rounded in chains of
        # at most (N + 16) / 32 + 128 additions, the scale's and the base's
        y = held @ self.w64.T
        o, size = R.lora(y, t["y"], self.a.float().numpy(), self.b.float().numpy(), t["ids"], self.scales.numpy(), RANKS)
        assert (np.abs(t["o"] - o) <= 1e-4 * np.abs(y).max() + U * (((self.N + 16) / 32 + 132) * size + 2 * np.abs(o))).all()
        assert np.abs(o - y).max() > 0.01 * np.abs(y).max() or (t["ids"] < 0).all()        # the adapters do count
        h, p, r = R.norm(t["o"], t["h1"], self.n2, EPS)
        np.testing.assert_array_equal(t["h2"], h)
        np.testing.assert_allclose(t["z"], p.astype(np.float64) * r, rtol=2.01 * U)
        logits = t["z"].astype(np.float64) @ self.head64.T
        np.testing.assert_allclose(t["logits"], logits, atol=1e-4 * np.abs(logits).max())
        # (z - max) - log S of given logits: a rounding of each, a sum of V terms in chains of V / 1024 + 64
        lp, ent, ids, top, logs = R.logprobs(t["logits"], t["tok"], 6)
        far = (self.V / 1024 + 72 + 4 * np.abs(logs).max()) * U
        np.testing.assert_allclose(t["lp"], lp, rtol=4 * U, atol=far)
        np.testing.assert_allclose(t["top_lp"], top, rtol=4 * U, atol=far)
        np.testing.assert_allclose(t["ent"], ent, rtol=2 * (self.V / 1024 + 72) * U, atol=2 * far)
        np.testing.assert_array_equal(t["top"], ids)


@pytest.mark.parametrize("B,N,V", [(1, 256, 1000), (5, 512, 4001), (32, 1024, 9000), (70, 512, 4032), (300, 256, 2048)])
def test_a_batch(B, N, V):
    b = Batch(B, N, V, B)
    b.run()
    b.check()


@pytest.mark.parametrize("B", [9, 90])
def test_a_captured_batch(B):
    b = Batch(B, 512, 4992, B)
    b.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run()
    for _ in range(4):
        b.fill()
        g.replay()
        torch.cuda.synchronize()
        b.check()
        torch.empty(1 << 20, device="cuda").fill_(float("nan"))      # memory that the graph does not own
