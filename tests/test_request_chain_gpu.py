"""A step of a batch through the operators around its projections, as a server runs them: residual and norm to codes, the
W4A8 projection, each request's adapter beside it, the next residual and norm, the INT8 head, log-probabilities."""
import numpy as np
import pytest
import torch

import libinferbit_amd as L
from libinferbit_amd import ops
from oracle import pyoracle as O
from oracle import requests as R

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Step:
    """B requests, width N, vocabulary V, adapters of rank 16; the operands on the GPU and on the host."""

    def __init__(self, B, N, V, n, seed):
        L.ops.init(0)
        rng = np.random.default_rng(seed)
        self.B, self.N, self.V, self.rng = B, N, V, rng
        self.w, self.ws = O.quantize(4, (rng.standard_normal((N, N)) * 0.05).astype(np.float32))
        self.head, self.hs = O.quantize(8, (rng.standard_normal((V, N)) * 0.05).astype(np.float32))
        self.n1, self.n2 = (rng.random((2, N)) + 0.5).astype(np.float32)
        g = torch.Generator().manual_seed(seed)
        self.a = (torch.randn(n, 16, N, generator=g) / np.sqrt(N)).half()
        self.b = torch.randn(n, N, 16, generator=g).half() / 4
        self.scales = torch.rand(n, generator=g) + 0.5
        gpu = lambda t: torch.from_numpy(t).cuda()
        self.d = dict(w=gpu(self.w), ws=gpu(self.ws.view(np.int16)), head=gpu(self.head), hs=gpu(self.hs.view(np.int16)),
                      n1=gpu(self.n1), n2=gpu(self.n2), a=self.a.cuda(), b=self.b.cuda(), scales=self.scales.cuda())
        f = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="cuda")
        self.x, self.delta, self.ids, self.tok = f(B, N), f(B, N), f(B, dtype=torch.int32), f(B, dtype=torch.int32)
        self.h1, self.q, self.s, self.y, self.o, self.h2, self.z = f(B, N), f(B, N, dtype=torch.int8), f(B, (N + 127) // 128), f(B, N), f(B, N), f(B, N), f(B, N)
        self.logits, self.lp, self.ent, self.top, self.top_lp = f(B, V), f(B), f(B), f(B, 6, dtype=torch.int32), f(B, 6)
        self.fill()

    def fill(self):
        B, N, rng = self.B, self.N, self.rng
        self.x.copy_(torch.from_numpy(rng.standard_normal((B, N)).astype(np.float32) * 2))
        self.delta.copy_(torch.from_numpy(rng.standard_normal((B, N)).astype(np.float32)))
        self.ids.copy_(torch.from_numpy(rng.integers(-1, self.a.shape[0], B).astype(np.int32)))
        self.tok.copy_(torch.from_numpy(rng.integers(0, self.V, B).astype(np.int32)))

    def run(self):
        B, N, V, d = self.B, self.N, self.V, self.d
        ops.add_rmsnorm(None, self.x, d["n1"], EPS, delta=self.delta, h=self.h1, q=self.q, s=self.s)
        ops.matmul_w4a8_batch(self.y, d["w"], d["ws"], self.q, self.s, N, N, B, N)
        ops.lora(self.o, self.h1, d["a"], d["b"], self.ids, base=self.y, scales=d["scales"])
        ops.add_rmsnorm(self.z, self.o, d["n2"], EPS, delta=self.h1, h=self.h2)
        ops.matmul_int8_batch(self.logits, d["head"], d["hs"], self.z, V, N, B, V)
        ops.logprobs(self.lp, self.logits, self.tok, entropy=self.ent, top_ids=self.top, top_logprobs=self.top_lp)

    def check(self):
        host = {k: getattr(self, k).cpu().numpy() for k in ("x", "delta", "ids", "tok", "h1", "q", "s", "y", "o", "h2", "z", "logits", "lp", "ent", "top", "top_lp")}
        h, p, r = R.norm(host["x"], host["delta"], self.n1, EPS)
        np.testing.assert_array_equal(host["h1"], h)
        for i in range(self.B):
            q, s = R.codes(p[i], r[i, 0])
            np.testing.assert_array_equal(host["q"][i], q)
            np.testing.assert_allclose(host["s"][i], s, rtol=3.01 * 2.0 ** -24)
        # the projection of these codes in 64 bits
        nib = np.stack([self.w & 15, self.w >> 4], -1).reshape(self.N, self.N).astype(np.float64) - 8
        held = host["q"].astype(np.float64) * np.repeat(host["s"].astype(np.float64), 128, 1)[:, :self.N]
        y = held @ nib.T * self.ws.view(np.float16).astype(np.float64)
        np.testing.assert_allclose(host["y"], y, atol=1e-4 * np.abs(y).max())
        # from the codes on in 64 bits throughout; the parts hold 1e-4 of the products' largest (the two projections) and
        # far less (the others): 1e-3 of the logits' largest over both
        o, _ = R.lora(y, h, self.a.float().numpy(), self.b.float().numpy(), host["ids"], self.scales.numpy())
        np.testing.assert_allclose(host["o"], o, atol=2e-4 * np.abs(o).max())
        h2 = o + h
        z = h2 / np.sqrt((h2 ** 2).mean(-1, keepdims=True) + EPS) * self.n2
        logits = z @ (self.head.reshape(self.V, self.N).view(np.int8).astype(np.float64) * self.hs.view(np.float16).astype(np.float64)[:, None]).T
        far = 1e-3 * np.abs(logits).max()
        np.testing.assert_allclose(host["logits"], logits, atol=far)
        # the entropy moves by at most far * sum p |log p + entropy| <= 2 far log V, 18.3 far at 9000
        lp, ent, _, top, _ = R.logprobs(logits, host["tok"], 6)
        np.testing.assert_allclose(host["lp"], lp[:, 0], atol=2 * far + 1e-4)
        np.testing.assert_allclose(host["top_lp"], top, atol=2 * far + 1e-4)
        np.testing.assert_allclose(host["ent"], ent, atol=20 * far + 1e-3)
        _, _, ids, _, _ = R.logprobs(host["logits"], host["tok"], 6)
        np.testing.assert_array_equal(host["top"], ids)


@pytest.mark.parametrize("B,N,V", [(1, 256, 1000), (5, 512, 4001), (32, 1024, 9000)])
def test_a_step(B, N, V):
    s = Step(B, N, V, 6, B)
    s.run()
    s.check()


def test_a_captured_step():
    s = Step(9, 512, 5000, 4, 1)
    s.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run()
    for _ in range(4):
        s.fill()
        g.replay()
        torch.cuda.synchronize()
        s.check()
        torch.empty(1 << 20, device="cuda").fill_(float("nan"))      # memory that the graph does not own
