"""Low-rank adapters of many requests on the GPU, against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from libinferbit_amd import _lib, ops
from oracle import requests as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def adapters(n, rank, N, M, kind, seed):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(n, rank, N, generator=g) / np.sqrt(N)).to(TYPES[kind])
    b = (torch.randn(n, M, rank, generator=g) / np.sqrt(rank)).to(TYPES[kind])
    return a, b, torch.rand(n, generator=g) * 2 + 0.1


def rows(t, gap, fill=float("nan")):
    wide = torch.full((t.shape[0], t.shape[1] + gap), fill, device="cuda")
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def check(out, base, x, a, b, ids, scales, ranks):
    """A sum of n products is held in chains of at most n / 32 + 64 fp32 additions, each half a step off at most; then come
    the scale's product and the base's addition."""
    want, size = R.lora(base, x, a.float().numpy(), b.float().numpy(), ids, scales, ranks)
    off = np.abs(out - want)
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(out), nan)
    chain = (a.shape[2] + a.shape[1]) / 32 + 128 + 4
    assert (off <= U * (chain * size + 2 * np.abs(want)))[~nan].all(), np.nanmax(off / (size + 1e-30)) / U
    # and the errors are no more than random ones: far below what the longest chain allows
    fine = ~nan & (size > 0)
    if fine.any():
        assert np.sqrt(np.mean(off[fine] ** 2)) <= 2.0 ** -20 * np.sqrt(np.mean((size + np.abs(want))[fine] ** 2))


def one(B, N, M, rank, n, kind, ids, seed=0, scales=True, ranks=None, base=True, gap=(0, 0, 0)):
    a, b, s = adapters(n, rank, N, M, kind, seed)
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(B, N, generator=g) * torch.exp(torch.randn(N, generator=g))
    y = torch.randn(B, M, generator=g) if base else None
    if ranks is not None:                                # what lies behind an adapter's rank is not used
        for i, r in enumerate(ranks):
            if 0 <= r < rank:
                a[i, r:], b[i, :, r:] = float("nan"), float("inf")
    out = rows(torch.full((B, M), 7.0), gap[0], 3.0)
    ops.lora(out, rows(x, gap[1]), a.cuda(), b.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda"),
             base=None if y is None else rows(y, gap[2]), scales=s.cuda() if scales else None,
             ranks=None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda"))
    if ranks is not None:
        for i, r in enumerate(ranks):
            if 0 <= r < rank:
                a[i, r:], b[i, :, r:] = 0, 0
    check(out.cpu().numpy().astype(np.float64), None if y is None else y.numpy(), x.numpy(), a, b, ids,
          s.numpy() if scales else None, ranks)
    if gap[0] and B > 1:
        assert (out.as_strided((B - 1, gap[0]), (M + gap[0], 1), M) == 3).all()


def spread(B, n, seed, none=0.1):
    rng = np.random.default_rng(seed)
    return np.where(rng.random(B) < none, -1 - rng.integers(0, 3, B), (rng.random(B) ** 2 * n).astype(int)).tolist()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("N,M", [(1, 1), (1, 300), (300, 1), (7, 5), (8, 8), (64, 128), (127, 129), (130, 70), (256, 512),
                                 (1000, 1001), (2048, 2048), (4096, 1024)])
@pytest.mark.parametrize("rank", [1, 16, 20])
def test_shapes(N, M, rank, kind):
    one(3, N, M, rank, 4, kind, [2, -1, 0], seed=N + M)
    one(70, N, M, rank, 4, kind, spread(70, 4, N), seed=N + M)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rank", [1, 2, 3, 7, 8, 9, 15, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129, 200, 255, 256])
def test_ranks(rank, kind):
    one(9, 256, 192, rank, 3, kind, [0, 2, 1, 2, 2, -1, 0, 1, 2], seed=rank)
    one(100, 192, 264, rank, 3, kind, spread(100, 3, rank), seed=rank)


@pytest.mark.parametrize("B", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 66, 127, 128, 129, 200, 500, 1030])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_rows(B, n):
    one(B, 256, 136, 16, n, "bf16", spread(B, n, B), seed=B)


@pytest.mark.parametrize("B,n", [(8191, 3), (8192, 40), (8193, 1), (9001, 300), (20000, 2), (70, 1022), (300, 1023), (1000, 1500), (8500, 4096)])
def test_many_rows_and_adapters(B, n):
    """More rows than the sorting block keeps in registers, more adapters than it has threads."""
    one(B, 64, 32, 8, n, "bf16", spread(B, n, B), seed=n)
    one(B, 36, 20, 3, n, "fp16", np.random.default_rng(B).integers(-1, n, B).tolist(), seed=n)
    one(B, 32, 32, 4, n, "bf16", sorted(spread(B, n, B + 1)), seed=n, ranks=np.random.default_rng(n).integers(-1, 6, n).tolist())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B", [1, 7, 64])
@pytest.mark.parametrize("rank,N", [(16, 4096), (16, 4104), (17, 4096), (128, 512), (128, 520), (1, 60000), (8, 9000), (64, 5000)])
def test_one_launch_and_two(rank, N, B, kind):
    one(B, N, 300, rank, 5, kind, spread(B, 5, rank), seed=rank + N)


@pytest.mark.parametrize("B", [20, 150])
def test_uneven_ranks(B):
    for kind in TYPES:
        one(B, 512, 200, 48, 6, kind, spread(B, 6, B), ranks=[0, 1, 17, 48, 33, 16], seed=B)
        one(B, 100, 77, 40, 6, kind, spread(B, 6, B), ranks=[40, 8, 0, 39, 32, 3], seed=B)


@pytest.mark.parametrize("B", [5, 80])
@pytest.mark.parametrize("gap", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (4, 4, 4), (3, 5, 7)])
def test_spaced_rows(B, gap):
    one(B, 256, 128, 16, 3, "fp16", spread(B, 3, 1), gap=gap)
    one(B, 250, 130, 10, 3, "bf16", spread(B, 3, 1), gap=gap)


@pytest.mark.parametrize("B", [1, 30, 90])
def test_without_base_and_scales(B):
    one(B, 256, 128, 16, 3, "fp16", spread(B, 3, 2), base=False)
    one(B, 256, 128, 16, 3, "bf16", spread(B, 3, 2), scales=False)
    one(B, 256, 128, 16, 3, "bf16", [-1] * B, base=False)


@pytest.mark.parametrize("B", [12, 140])
def test_rows_and_ranks_that_are_not_there(B):
    _lib.lib().ibh_device_errors(1)
    ids = spread(B, 5, B)
    one(B, 128, 96, 8, 5, "fp16", ids)
    assert _lib.lib().ibh_device_errors(0) == 0
    ids[3], ids[7] = 5, 2 ** 31 - 1
    one(B, 128, 96, 8, 5, "fp16", ids)
    assert _lib.lib().ibh_device_errors(1) == 8
    one(B, 128, 96, 8, 5, "bf16", spread(B, 5, B + 1, none=0), ranks=[3, 9, 8, -1, 0])
    assert _lib.lib().ibh_device_errors(1) == 8


@pytest.mark.parametrize("B,kind", [(1, "bf16"), (40, "fp16"), (300, "bf16")])
def test_in_place(B, kind):
    a, b, s = adapters(4, 16, 512, 384, kind, 3)
    x, y, ids = torch.randn(B, 512), torch.randn(B, 384), spread(B, 4, B)
    out = y.cuda()
    ops.lora(out, x.cuda(), a.cuda(), b.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda"), base=out, scales=s.cuda())
    check(out.cpu().numpy(), y.numpy(), x.numpy(), a, b, ids, s.numpy(), None)


@pytest.mark.parametrize("B", [4, 100])
@pytest.mark.parametrize("kind", TYPES)
def test_magnitudes(B, kind):
    """Elements across fp32's range beside each other, and the adapters' smallest and largest numbers."""
    a, b, s = adapters(3, 8, 320, 64, kind, 1)
    a[0], b[1] = a[0] * 2.0 ** -14, b[1] * 2.0 ** -14
    a[2] = a[2] * 2.0 ** 13
    x = torch.randn(B, 320) * torch.exp2(torch.randint(-40, 40, (B, 320)).float())
    x[0] *= 2.0 ** -60
    x[1] *= 2.0 ** 60
    ids = spread(B, 3, B, none=0)
    out = torch.empty(B, 64, device="cuda")
    ops.lora(out, x.cuda(), a.cuda(), b.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda"), scales=s.cuda())
    check(out.cpu().numpy().astype(np.float64), None, x.numpy(), a, b, ids, s.numpy(), None)


@pytest.mark.parametrize("B", [4, 100])
def test_a_bad_row_stays_alone(B):
    a, b, s = adapters(3, 16, 256, 128, "bf16", 1)
    x = torch.randn(B, 256)
    x[1, 100], x[3, 7] = float("nan"), float("inf")
    ids = [0] * B
    out = torch.empty(B, 128, device="cuda")
    ops.lora(out, x.cuda(), a.cuda(), b.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda"))
    out = out.cpu().numpy()
    assert not np.isfinite(out[[1, 3]]).any()
    good = [i for i in range(B) if i not in (1, 3)]
    check(out[good], None, x.numpy()[good], a, b, [ids[i] for i in good], None, None)


@pytest.mark.parametrize("B", [6, 130])
def test_the_same_bits_every_time_and_in_any_order(B):
    a, b, s = adapters(4, 24, 1024, 520, "fp16", 2)
    a, b, s, x = a.cuda(), b.cuda(), s.cuda(), torch.randn(B, 1024, device="cuda")
    ids = torch.tensor(spread(B, 4, 5), dtype=torch.int32, device="cuda")
    out = torch.empty(B, 520, device="cuda")
    ops.lora(out, x, a, b, ids, scales=s)
    for _ in range(5):
        again = torch.empty_like(out)
        ops.lora(again, x, a, b, ids, scales=s)
        assert torch.equal(out, again)
    turn = torch.randperm(B, device="cuda")
    ops.lora(again, x[turn], a, b, ids[turn], scales=s)
    assert torch.equal(out[turn], again)


@pytest.mark.parametrize("B", [8, 200])
def test_replays_follow_ids(B):
    a, b, s = adapters(5, 16, 256, 128, "bf16", 2)
    ad, bd, sd = a.cuda(), b.cuda(), s.cuda()
    x, out = torch.randn(B, 256), torch.empty(B, 128, device="cuda")
    xd, ids = x.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda")
    ops.lora(out, xd, ad, bd, ids, scales=sd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.lora(out, xd, ad, bd, ids, scales=sd)
    for seed in range(4):
        now = spread(B, 5, seed, none=0.2 * seed)
        ids.copy_(torch.tensor(now, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check(out.cpu().numpy(), None, x.numpy(), a, b, now, s.numpy(), None)


def test_two_streams_at_once():
    got = []
    sets = [(adapters(4, 16, 512, 256, "fp16", k), torch.randn(100, 512), spread(100, 4, k)) for k in range(2)]
    dev = [([t.cuda() for t in ab], x.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda")) for ab, x, ids in sets]
    outs = [torch.empty(100, 256, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for (ab, x, ids), out, st in zip(dev, outs, streams):
            with torch.cuda.stream(st):
                ops.lora(out, x, ab[0], ab[1], ids, scales=ab[2])
    torch.cuda.synchronize()
    for ((a, b, s), x, ids), out in zip(sets, outs):
        check(out.cpu().numpy(), None, x.numpy(), a, b, ids, s.numpy(), None)


@pytest.mark.parametrize("B,rank", [(6, 64), (90, 16)])
def test_two_graphs_at_once(B, rank):
    """Each with a workspace of its own, replayed side by side on two streams."""
    sets = [(adapters(4, rank, 2048, 256, "bf16", k), torch.randn(B, 2048), spread(B, 4, k)) for k in range(2)]
    dev = [([t.cuda() for t in ab], x.cuda(), torch.tensor(ids, dtype=torch.int32, device="cuda")) for ab, x, ids in sets]
    outs, graphs, streams = [torch.empty(B, 256, device="cuda") for _ in sets], [], [torch.cuda.Stream() for _ in sets]
    for (ab, x, ids), out in zip(dev, outs):
        ops.lora(out, x, ab[0], ab[1], ids, scales=ab[2])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.lora(out, x, ab[0], ab[1], ids, scales=ab[2])
        graphs.append(g)
    for _ in range(10):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for ((a, b, s), x, ids), out in zip(sets, outs):
            check(out.cpu().numpy(), None, x.numpy(), a, b, ids, s.numpy(), None)


def test_no_rows():
    a, b, s = (t.cuda() for t in adapters(2, 8, 64, 32, "fp16", 0))
    ops.lora(torch.empty(0, 32, device="cuda"), torch.empty(0, 64, device="cuda"), a, b,
             torch.empty(0, dtype=torch.int32, device="cuda"))


def test_a_large_pool():
    """Adapters beyond 4 GB: 64 bits of offset."""
    n, rank, N, M = 700, 64, 40000, 8
    a = torch.zeros(n, rank, N, dtype=torch.bfloat16, device="cuda")
    b = torch.randn(n, M, rank, device="cuda").to(torch.bfloat16)
    a[n - 1] = torch.randn(rank, N, device="cuda") / 200
    a[n - 2] = torch.randn(rank, N, device="cuda") / 200
    for B in (2, 70):
        x = torch.randn(B, N)
        ids = [n - 1 - i % 2 for i in range(B)]
        out = torch.empty(B, M, device="cuda")
        ops.lora(out, x.cuda(), a, b, torch.tensor(ids, dtype=torch.int32, device="cuda"))
        check(out.cpu().numpy(), None, x.numpy(), a[n - 2:].cpu(), b[n - 2:].cpu(), [i - n + 2 for i in ids], None, None)


def test_wrappers_refuse():
    a, b, s = (t.cuda() for t in adapters(2, 8, 64, 32, "fp16", 0))
    x, out, ids = torch.zeros(3, 64, device="cuda"), torch.zeros(3, 32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for err, args, kw in ((TypeError, (out, x, a, b.bfloat16(), ids), {}), (TypeError, (out, x, a, b, ids.long()), {}),
                          (ValueError, (out, x, a, b[:1], ids), {}), (ValueError, (out, x[:, :63], a, b, ids), {}),
                          (ValueError, (out[:2], x, a, b, ids), {}), (ValueError, (out, x, a, b, ids[:2]), {}),
                          (TypeError, (out, x.half(), a, b, ids), {}), (ValueError, (out, x, a, b, ids), dict(scales=s[:1])),
                          (ValueError, (out, x, a, b, ids), dict(base=out[:2])), (TypeError, (out, x, a, b, ids), dict(ranks=ids[:2].float())),
                          (ValueError, (out, x, a.cpu(), b, ids), {}), (ValueError, (out, x, a[:, ::2], b[:, :, ::2], ids), {}),
                          (ValueError, (out[:1].expand(3, 32), x, a, b, ids), {}), (_lib.IbhError, (x[:, :32], x, a, b, ids), {})):
        with pytest.raises(err):
            ops.lora(*args, **kw)
    a, b, s = (t.cuda() for t in adapters(2, 64, 4096, 32, "fp16", 0))
    with pytest.raises(_lib.IbhError):
        ops.lora(out, torch.zeros(3, 4096, device="cuda"), a, b, ids, ws=torch.empty(4, dtype=torch.uint8, device="cuda"))
