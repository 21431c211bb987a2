"""The residual's addition with the RMS norm and its 8-bit codes on the GPU, against the oracle."""
import numpy as np
import pytest
import torch

from libinferbit_amd import ops
from oracle import requests as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GROUP = R.GROUP


def spaced(a, gap):
    """a on the GPU as rows cut out of wider ones, NaN around them."""
    t = torch.full((a.shape[0], a.shape[1] + gap), float("nan"), device="cuda")
    t[:, :a.shape[1]] = torch.from_numpy(a)
    return t[:, :a.shape[1]]


def inputs(B, N, seed, delta=True):
    rng = np.random.default_rng(seed)
    chan = np.exp(rng.standard_normal(N))
    x = (rng.standard_normal((B, N)) * chan).astype(np.float32)
    d = (rng.standard_normal((B, N)) * chan * 0.3).astype(np.float32) if delta else None
    return x, d, (rng.random(N) + 0.5).astype(np.float32)


def run(x, d, w, eps, gap=0, y=True, q=True, h=True):
    B, N = x.shape
    new = lambda on, shape, dtype: torch.full(shape, 77, dtype=dtype, device="cuda") if on else None
    o = dict(y=new(y, (B, N), torch.float32), q=new(q, (B, N), torch.int8),
             s=new(q, (B, (N + GROUP - 1) // GROUP), torch.float32), h=new(h, (B, N), torch.float32))
    ops.add_rmsnorm(o["y"], spaced(x, gap), torch.from_numpy(w).cuda(), eps, delta=None if d is None else spaced(d, gap),
                    h=o["h"], q=o["q"], s=o["s"])
    return {k: None if t is None else t.cpu().numpy() for k, t in o.items()}


def check(o, x, d, w, eps):
    """h and codes are the definition's; y and s have two and three roundings behind p: the factor's (whose own error is
    far below), the product's, the division's."""
    h, p, r = R.norm(x, d, w, eps)
    if o["h"] is not None:
        np.testing.assert_array_equal(o["h"], h)
    if o["y"] is not None:
        want = p.astype(np.float64) * r
        np.testing.assert_array_equal(np.isnan(o["y"]), np.isnan(want))
        assert (np.abs(o["y"] - want) <= 2.01 * U * np.abs(want) + 2.0 ** -149)[~np.isnan(want)].all()
    if o["q"] is not None:
        for i in range(x.shape[0]):
            q, s = R.codes(p[i], r[i, 0])
            np.testing.assert_array_equal(o["q"][i], q)
            np.testing.assert_allclose(o["s"][i], s, rtol=3.01 * U, atol=2.0 ** -149)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 31, 127, 128, 129, 255, 260, 1000, 1024, 1025, 2047, 2048, 4096, 4097, 5632,
                               8192, 8195, 14336, 16384, 16385, 20002])
def test_sizes(N):
    x, d, w = inputs(3, N, N)
    check(run(x, d, w, 1e-5), x, d, w, 1e-5)
    check(run(x, None, w, 1e-6, h=False), x, None, w, 1e-6)


@pytest.mark.parametrize("gap", [1, 2, 4, 7])
@pytest.mark.parametrize("N", [130, 1024, 4099, 17000])
def test_spaced_rows(N, gap):
    x, d, w = inputs(5, N, N + gap)
    check(run(x, d, w, 1e-5, gap=gap), x, d, w, 1e-5)


@pytest.mark.parametrize("y,q,h", [(True, False, False), (True, False, True), (False, True, False), (False, True, True)])
@pytest.mark.parametrize("N", [300, 4096, 16400])
def test_outputs_alone(N, y, q, h):
    x, d, w = inputs(2, N, N)
    check(run(x, d, w, 1e-5, y=y, q=q, h=h), x, d, w, 1e-5)


@pytest.mark.parametrize("B", [1, 2, 64, 1000])
def test_many_rows(B):
    x, d, w = inputs(B, 384, B)
    check(run(x, d, w, 1e-5), x, d, w, 1e-5)


@pytest.mark.parametrize("N", [200, 1000, 1026, 2048, 2051, 4096, 4100, 8190])
def test_more_rows_than_wide_blocks_take(N):
    """The many rows of a call are a few, again and again: equal rows come out equal, the first ones are right."""
    x, d, w = inputs(3, N, N)
    o = run(np.tile(x, (350, 1)), np.tile(d, (350, 1)), w, 1e-5)
    check({k: v[:3] for k, v in o.items()}, x, d, w, 1e-5)
    for k, v in o.items():
        np.testing.assert_array_equal(v, np.tile(v[:3], (350, 1)), err_msg=k)


def test_codes_at_borders():
    """Quotients of 127 p / max|p| at halves, and as near to them as floats come."""
    rng = np.random.default_rng(5)
    rows = [np.concatenate([[127.0], np.arange(127) + 0.5]), np.concatenate([[254.0], -(np.arange(127) * 2.0 + 1)])]
    for _ in range(30):
        m = np.float32(rng.random() + 1)
        half = ((np.arange(127) + 0.5) * np.float64(m) / 127).astype(np.float32)
        for way in (-np.inf, np.inf, None):
            rows.append(np.concatenate([[m], half if way is None else np.nextafter(half, np.float32(way))]))
    x = np.array(rows, np.float32)
    check(run(x, None, np.ones(128, np.float32), 1e-5, h=False), x, None, np.ones(128, np.float32), 1e-5)


@pytest.mark.parametrize("N", [4096, 17000])
def test_values_at_the_ends_of_the_range(N):
    x, d, w = inputs(8, N, 9)
    x[0] *= np.float32(1e18)                             # squares beyond fp32
    x[1] *= np.float32(1e-25)                            # and below
    x[2], d[2] = 0, 0
    x[3] *= np.float32(1e-40)                            # subnormal numbers
    x[4, 5] = np.nan
    d[5, 7] = np.inf
    x[6, :128], d[6, :128] = 0, 0                        # a group of zeros in a row of others
    check(run(x, d, w, 1e-5), x, d, w, 1e-5)
    x, d = np.delete(x, 2, 0), np.delete(d, 2, 0)
    check(run(x, d, w, 0.0), x, d, w, 0.0)
    w[200], w[3] = np.nan, 3e38
    o = run(x, d, w, 1e-5)
    h, p, r = R.norm(x, d, w, 1e-5)
    for i in range(x.shape[0]):
        q, s = R.codes(p[i], r[i, 0])
        np.testing.assert_array_equal(o["q"][i], q)
        np.testing.assert_array_equal(np.isnan(o["s"][i]), np.isnan(s))


@pytest.mark.parametrize("N", [300, 4096, 17000])
def test_rows_of_subnormal_numbers(N):
    """Without eps the factor is beyond fp32, y and the scales are ordinary numbers."""
    x, _, w = inputs(3, N, 4)
    x[0] *= np.float32(1e-39)
    x[1] *= np.float32(1e-42)
    x[2] *= np.float32(1e-37)
    check(run(x, None, w, 0.0, h=False), x, None, w, 0.0)
    check(run(x, None, w, 1e-30, h=False), x, None, w, 1e-30)


def test_a_row_of_zeros_without_eps():
    x, w = np.zeros((1, 256), np.float32), np.ones(256, np.float32)
    o = run(x, None, w, 0.0, h=False)
    assert np.isnan(o["y"]).all() and np.isnan(o["s"]).all() and not o["q"].any()


@pytest.mark.parametrize("N", [1000, 4096, 16390])
@pytest.mark.parametrize("place", ["h=x", "h=delta", "y=x", "y=delta", "h=x,y=delta", "h=delta,y=x"])
def test_in_place(N, place):
    x, d, w = inputs(3, N, N)
    t = {"x": torch.from_numpy(x).cuda(), "delta": torch.from_numpy(d).cuda()}
    at = dict(p.split("=") for p in place.split(","))
    o = {k: t[at[k]] if k in at else torch.empty(3, N, device="cuda") for k in ("h", "y")}
    if place.startswith("y"):
        o["h"] = None
    q, s = torch.empty(3, N, dtype=torch.int8, device="cuda"), torch.empty(3, (N + 127) // 128, device="cuda")
    ops.add_rmsnorm(o["y"], t["x"], torch.from_numpy(w).cuda(), 1e-5, delta=t["delta"], h=o["h"], q=q, s=s)
    o |= {"q": q, "s": s}
    check({k: None if v is None else v.cpu().numpy() for k, v in o.items()}, x, d, w, 1e-5)


def test_nothing_beyond_the_outputs_is_written():
    x, d, w = inputs(3, 133, 1)
    big = torch.full((3 * 133 + 64,), 5, dtype=torch.int8, device="cuda")
    yb = torch.full((3 * 133 + 64,), 5.0, device="cuda")
    s = torch.empty(3, 2, device="cuda")
    ops.add_rmsnorm(yb[32:32 + 399].view(3, 133), spaced(x, 0), torch.from_numpy(w).cuda(), 1e-5, delta=spaced(d, 0),
                    q=big[32:32 + 399].view(3, 133), s=s)
    for t in (big, yb):
        assert (t[:32] == 5).all() and (t[431:] == 5).all()
    check(dict(y=yb[32:431].view(3, 133).cpu().numpy(), q=big[32:431].view(3, 133).cpu().numpy(), s=s.cpu().numpy(), h=None), x, d, w, 1e-5)


def test_no_rows():
    e = torch.empty(0, 128, device="cuda")
    ops.add_rmsnorm(e, e, torch.ones(128, device="cuda"), 1e-5)


def test_other_streams_and_replays():
    x, d, w = inputs(4, 4096, 3)
    xs, ds, wt = (torch.from_numpy(t).cuda() for t in (x, d, w))
    h, q, s = torch.empty_like(xs), torch.empty(4, 4096, dtype=torch.int8, device="cuda"), torch.empty(4, 32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.add_rmsnorm(None, xs, wt, 1e-5, delta=ds, h=h, q=q, s=s)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.add_rmsnorm(None, xs, wt, 1e-5, delta=ds, h=h, q=q, s=s)
    for seed in (11, 12, 13):
        x, d, _ = inputs(4, 4096, seed)
        xs.copy_(torch.from_numpy(x))
        ds.copy_(torch.from_numpy(d))
        g.replay()
        torch.cuda.synchronize()
        check(dict(y=None, h=h.cpu().numpy(), q=q.cpu().numpy(), s=s.cpu().numpy()), x, d, w, 1e-5)


def test_wrappers_refuse():
    x, w = torch.zeros(2, 256, device="cuda"), torch.ones(256, device="cuda")
    q, s = torch.zeros(2, 256, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, device="cuda")
    y = torch.empty_like(x)
    for err, args, kw in ((ValueError, (None, x, w, 1e-5), {}), (ValueError, (y, x, w, 1e-5), dict(q=q)),
                          (ValueError, (y, x, w[:255], 1e-5), {}), (ValueError, (y[:1], x, w, 1e-5), {}),
                          (ValueError, (y, x, w, 1e-5), dict(delta=x[:1])), (ValueError, (None, x, w, 1e-5), dict(q=q, s=s[:, :1])),
                          (ValueError, (y, x, w.cpu(), 1e-5), {}), (TypeError, (y, x.half(), w, 1e-5), {}),
                          (TypeError, (y, x, w.double(), 1e-5), {}), (TypeError, (None, x, w, 1e-5), dict(q=q.to(torch.uint8), s=s)),
                          (ValueError, (y, x[:1].expand(2, 256), w, 1e-5), {}), (ValueError, (y, x.T.contiguous().T, w, 1e-5), {}),
                          (ops_error(), (y, x, w, -1.0), {}), (ops_error(), (y, x, w, 1e-5), dict(h=y))):
        with pytest.raises(err):
            ops.add_rmsnorm(*args, **kw)


def ops_error():
    from libinferbit_amd import _lib
    return _lib.IbhError
