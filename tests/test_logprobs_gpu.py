"""Log-probabilities, entropy and alternatives on the GPU, against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from libinferbit_amd import _lib, ops
from oracle import requests as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def run(z, tokens, k, gap=0, entropy=True, flat=False):
    B, V = z.shape
    wide = torch.full((B, V + gap), float("nan"), device="cuda")
    wide[:, :V] = torch.from_numpy(z)
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device="cuda").view(B, -1)
    if flat:
        tok = tok.view(B)
    lp = None if tok is None else torch.full(tok.shape, 7.0, device="cuda")
    ent = torch.full((B,), 7.0, device="cuda") if entropy else None
    ids, top = (torch.full((B, k), 7, dtype=torch.int32, device="cuda"), torch.full((B, k), 7.0, device="cuda")) if k else (None, None)
    ops.logprobs(lp, wide[:, :V], tok, entropy=ent, top_ids=ids, top_logprobs=top)
    return tuple(None if t is None else t.cpu().numpy() for t in (lp, ent, ids, top))


def check(got, z, tokens, k):
    """A log-probability is (z - max) - log S.  The difference, the logarithm and their difference are rounded once each;
    S of terms whose exponentials are within 4 steps plus their argument's rounding (|x| e^x <= 1/e of a step in the sum)
    is summed in chains of at most V / 1024 + 64 additions.  The entropy is log S - sum e^d d / S: its second term is at
    most the entropy itself and, likewise summed, off by as much, relative to it."""
    lp, ent, ids, top, = got
    wlp, went, wids, wtop, logs = R.logprobs(z, np.zeros((z.shape[0], 0), int) if tokens is None else tokens, k)
    V = z.shape[1]
    chain = (V / 1024 + 64 + 8) * U
    logs = np.abs(np.where(np.isfinite(logs), logs, 0))[:, None]

    def near(x, want):
        np.testing.assert_array_equal(np.isnan(x), np.isnan(want))
        fine = np.isfinite(want)
        np.testing.assert_array_equal(x[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        off = np.abs(np.where(fine, x, 0) - np.where(fine, want, 0))
        allowed = chain + 2 * U * (logs + 2 * np.abs(np.where(fine, want, 0)) + logs)
        assert (off <= allowed).all(), (off / allowed).max()

    if lp is not None:
        near(lp.reshape(wlp.shape), wlp)
    if ent is not None:
        np.testing.assert_array_equal(np.isnan(ent), np.isnan(went))
        fine = ~np.isnan(went)
        assert (np.abs(ent - went) <= 2 * chain * (1 + np.abs(went)) + 4 * U * logs[:, 0])[fine].all()
    if k:
        np.testing.assert_array_equal(ids, wids)
        near(top, wtop)


def logits(B, V, seed, scale=3.0):
    return (np.random.default_rng(seed).standard_normal((B, V)) * scale).astype(np.float32)


def some(B, V, n, seed):
    return np.random.default_rng(seed + 99).integers(0, V, (B, n))


@pytest.mark.parametrize("V", [1, 2, 3, 5, 63, 64, 65, 255, 257, 1000, 1023, 1024, 1025, 2047, 4095, 4096, 4097, 8191, 8193,
                               12289, 16384, 32000, 32003, 50001, 128000, 260001])
def test_sizes(V):
    z = logits(3, V, V)
    for k in (0, 1, 5, 64):
        t = some(3, V, 2, V)
        check(run(z, t, k), z, t, k)


@pytest.mark.parametrize("B", [1, 2, 7, 64, 257, 300, 1500])
@pytest.mark.parametrize("k", [0, 3, 20])
def test_rows(B, k):
    for V in (777, 9001):
        z, t = logits(B, V, B), some(B, V, 1, B)
        check(run(z, t, k, flat=True), z, t, k)


@pytest.mark.parametrize("k", [1, 2, 7, 15, 16, 17, 31, 32, 33, 63, 64])
def test_numbers_of_alternatives(k):
    z, t = logits(5, 20011, k), some(5, 20011, 3, k)
    check(run(z, t, k), z, t, k)


@pytest.mark.parametrize("gap", [1, 2, 3, 4, 64])
def test_spaced_rows(gap):
    for B, V in ((3, 5000), (600, 5000), (9, 33)):
        z, t = logits(B, V, gap), some(B, V, 1, gap)
        check(run(z, t, 6, gap=gap), z, t, 6)


@pytest.mark.parametrize("B", [2, 700])
@pytest.mark.parametrize("V", [100, 5000, 40001])
def test_orders_that_are_hard_for_a_search(B, V):
    """Ascending and descending rows, all equal, few levels, the best side by side, alternating."""
    if B * V > 5_000_000:
        B = 130
    rng = np.random.default_rng(1)
    z = [np.arange(V), -np.arange(V), np.zeros(V), rng.integers(0, 3, V), np.where(np.arange(V) < 80, 5, rng.standard_normal(V)),
         np.where(np.arange(V) >= V - 90, 5 + np.arange(V) % 7, 0), np.arange(V) % 2 * 1.0, np.arange(V) // 64 * 0.25,
         np.where(np.arange(V) % 256 == 3, np.arange(V) % 1000, -1.0), -0.0 * (np.arange(V) % 2)]
    z = np.array([z[i % len(z)] for i in range(max(B, len(z)))], np.float32) * np.float32(0.01)
    for k in (1, 8, 64):
        check(run(z, some(z.shape[0], V, 1, V), k), z, some(z.shape[0], V, 1, V), k)


@pytest.mark.parametrize("V", [50, 3000, 70001])
@pytest.mark.parametrize("k", [0, 4, 40])
def test_masks(V, k):
    z = logits(12, V, V)
    inf = np.inf
    rng = np.random.default_rng(V)
    z[0] = -inf                                          # nothing is left
    z[1, :] = -inf
    z[1, V // 2] = 2.5                                   # one
    z[2, 3:] = -inf                                      # fewer than k
    z[3] = np.where(rng.random(V) < 0.95, -inf, z[3])
    z[4] = np.where(rng.random(V) < 0.95, np.finfo(np.float32).min, z[4])
    z[5] = np.finfo(np.float32).min                      # all alike
    z[6, V // 3] = np.nan
    z[7, V - 1] = inf
    z[8, V - 1], z[8, 0] = -inf, np.nan
    z[9] = np.finfo(np.float32).max
    z[10, :V - 1] = -inf
    z[11] *= np.float32(1e30)
    t = some(12, V, 3, V)
    t[:, 1] = [V // 2, V // 2, 1, 0, 0, V - 1, V // 3, V - 1, 0, 0, V - 1, 5]
    check(run(z, t, k), z, t, k)


def test_tokens_that_are_not_there():
    z = logits(4, 1000, 0)
    t = np.array([[-1, 1000], [999, 0], [2 ** 31 - 1, -2 ** 31], [5, 1001]])
    check(run(z, t, 2), z, t, 2)


@pytest.mark.parametrize("entropy,n,k", [(True, 0, 0), (False, 1, 0), (False, 0, 3), (False, 2, 5)])
def test_outputs_alone(entropy, n, k):
    for B in (2, 600):
        z = logits(B, 9000, n)
        t = some(B, 9000, n, 1) if n else None
        check(run(z, t, k, entropy=entropy), z, t, k)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 30.0, 1000.0])
def test_flat_and_sharp_rows(scale):
    z, t = logits(6, 32000, 4, scale), some(6, 32000, 2, 3)
    t[:, 0] = z.argmax(1)
    check(run(z, t, 5), z, t, 5)


def test_many_tokens_a_row():
    z, t = logits(3, 500, 1), some(3, 500, 2500, 1)
    check(run(z, t, 0), z, t, 0)


def test_no_rows():
    ops.logprobs(torch.empty(0, device="cuda"), torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("B,V", [(2, 60000), (700, 3000)])
def test_streams_and_replays(B, V):
    k = 10
    z = [torch.from_numpy(logits(B, V, s)).cuda() for s in range(2)]
    t = torch.from_numpy(some(B, V, 1, 0)).int().cuda()
    outs = [(torch.empty(B, 1, device="cuda"), torch.empty(B, device="cuda"), torch.empty(B, k, dtype=torch.int32, device="cuda"),
             torch.empty(B, k, device="cuda")) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for zz, o, st in zip(z, outs, streams):
            with torch.cuda.stream(st):
                ops.logprobs(o[0], zz, t, entropy=o[1], top_ids=o[2], top_logprobs=o[3])
    torch.cuda.synchronize()
    for s in range(2):
        check(tuple(x.cpu().numpy() for x in outs[s]), logits(B, V, s), t.cpu().numpy(), k)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for s in range(2):
        with torch.cuda.graph(graphs[s]):
            ops.logprobs(outs[s][0], z[s], t, entropy=outs[s][1], top_ids=outs[s][2], top_logprobs=outs[s][3])
    for seed in range(3):
        for s in range(2):
            z[s].copy_(torch.from_numpy(logits(B, V, 10 * seed + s)))
        for st, g in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in range(2):
            check(tuple(x.cpu().numpy() for x in outs[s]), logits(B, V, 10 * seed + s), t.cpu().numpy(), k)


def test_rows_beyond_4_gb():
    V = 150_000
    B = 2 ** 32 // (4 * V) + 3
    z = torch.zeros(B, V, device="cuda")
    z[-1] = torch.from_numpy(logits(1, V, 5)[0])
    z[-2, V - 1] = 20.0
    ids, top, ent = torch.empty(B, 4, dtype=torch.int32, device="cuda"), torch.empty(B, 4, device="cuda"), torch.empty(B, device="cuda")
    ops.logprobs(None, z, None, entropy=ent, top_ids=ids, top_logprobs=top)
    check((None, ent[-3:].cpu().numpy(), ids[-3:].cpu().numpy(), top[-3:].cpu().numpy()), z[-3:].cpu().numpy(), None, 4)


def test_wrappers_refuse():
    z, t = torch.zeros(3, 100, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    lp, ids, top = torch.empty(3, device="cuda"), torch.empty(3, 4, dtype=torch.int32, device="cuda"), torch.empty(3, 4, device="cuda")
    for err, args, kw in ((ValueError, (None, z, t), {}), (ValueError, (lp, z, None), {}), (TypeError, (lp, z, t.long()), {}),
                          (ValueError, (lp[:2], z, t), {}), (ValueError, (lp, z, t[:2]), {}), (TypeError, (lp, z.half(), t), {}),
                          (ValueError, (lp, z, t), dict(top_ids=ids)), (ValueError, (lp, z, t), dict(top_ids=ids, top_logprobs=top[:, :3])),
                          (TypeError, (lp, z, t), dict(top_ids=ids.long(), top_logprobs=top)), (ValueError, (lp, z, t), dict(entropy=lp[:2])),
                          (ValueError, (lp, z.cpu(), t), {}), (ValueError, (lp, z[:1].expand(3, 100), t), {}),
                          (_lib.IbhError, (None, z, None), {}), (_lib.IbhError, (lp, z, t), dict(entropy=lp))):
        with pytest.raises(err):
            ops.logprobs(*args, **kw)
    with pytest.raises(_lib.IbhError):
        ops.logprobs(None, z, None, top_ids=torch.empty(3, 65, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(3, 65, device="cuda"))
