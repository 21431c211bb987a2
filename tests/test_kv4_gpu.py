"""The paged 4-bit KV cache on the GPU against oracle/kv4.py (64 bits).

Codes, scales and mids are those of the definition, so what is stored, read
back and moved is compared bit for bit.  Attention: a score of absolute sum S
(sum |q k| / sqrt(hd)) is summed in chains of up to 64 terms whose roundings of
2^-24 S add like their root, 8 * 2^-24 S; it moves its probability by that
share, and the normaliser by as much: 16 * 2^-24 max(1, S) of the output's
2-norm.  A weight is a sum of such probabilities, each of them at least
2^-126 or nothing: fp32 holds no smaller normal number."""
import numpy as np
import pytest
import torch

from oracle import kv4 as R

pytestmark = pytest.mark.gpu

PAGE = 64


@pytest.fixture(scope="module")
def ops():
    import libinferbit_amd as L
    L.ops.init(0)
    return L.ops


def device_errors(clear=1):
    import libinferbit_amd as L
    return L.lib().ibh_device_errors(clear)


class Made:
    """A cache with normally distributed keys and values, host and device."""

    def __init__(self, ops, rng, lens, n_kv, hd, max_pages=None, extra=3, scale=1.0):
        self.lens, self.n_kv, self.hd = np.asarray(lens, np.int32), n_kv, hd
        n = len(lens)
        need = max(1, max((t + PAGE - 1) // PAGE for t in lens))
        mp = max_pages or need
        self.n_pages = n * mp + extra
        self.table = rng.permutation(self.n_pages)[:n * mp].astype(np.int32).reshape(n, mp)
        self.pool = rng.integers(0, 256, (self.n_pages, n_kv * 72 * hd), dtype=np.uint8)
        # stale pairs that are no numbers lie behind every length
        self.pool.view(np.uint16).reshape(self.n_pages, n_kv, 36 * hd)[:, :, 16 * hd:18 * hd] = 0x7E00
        self.pool.view(np.uint16).reshape(self.n_pages, n_kv, 36 * hd)[:, :, 34 * hd:36 * hd] = 0x7C00
        self.k = [(rng.standard_normal((t, n_kv * hd)) * scale).astype(np.float32) for t in lens]
        self.v = [rng.standard_normal((t, n_kv * hd)).astype(np.float32) for t in lens]
        self.dpool = torch.from_numpy(self.pool.copy()).cuda()
        self.dtable, self.dlens = torch.from_numpy(self.table).cuda(), torch.from_numpy(self.lens).cuda()
        self.cache = ops.Kv4Cache(self.dpool, self.dtable, self.dlens, n_kv, hd)
        most = max(lens)
        if most:
            K, V = np.zeros((2, n, most, n_kv * hd), np.float32)
            for i, t in enumerate(lens):
                K[i, most - t:], V[i, most - t:] = self.k[i], self.v[i]
            ops.kv4_append(self.cache, torch.from_numpy(K).cuda(), torch.from_numpy(V).cuda())

    def loaded(self, i):
        h = lambda x: R.held(x).reshape(len(x), self.n_kv, self.hd).transpose(1, 0, 2)
        return h(self.k[i]), h(self.v[i])


def fill(pool, m):
    for i, t in enumerate(m.lens):
        R.store(pool, m.table[i], m.n_kv, m.hd, m.k[i], m.v[i], 0)


@pytest.mark.parametrize("lens,n_kv,hd", [([1], 1, 64), ([63, 64, 65], 2, 128), ([0, 5, 130], 1, 192), ([17, 200], 2, 256)])
def test_append_stores_the_defined_bytes(ops, lens, n_kv, hd):
    print(f"case append {lens} {n_kv} {hd}", flush=True)
    rng = np.random.default_rng(sum(lens) + hd)
    m = Made(ops, rng, lens, n_kv, hd)
    want = m.pool.copy()
    fill(want, m)
    np.testing.assert_array_equal(m.dpool.cpu().numpy(), want)
    assert device_errors() == 0


def test_append_one_by_one_strided_and_read_back(ops):
    rng = np.random.default_rng(5)
    n, n_kv, hd = 3, 2, 64
    m = Made(ops, rng, [62, 0, 127], n_kv, hd, max_pages=3)
    want = m.pool.copy()
    fill(want, m)
    rows = [[], [], []]
    for step in range(5):
        # k and v inside one wider row, not on 16 bytes
        both = torch.randn(n, 1, 2 * n_kv * hd + 3, generator=torch.Generator().manual_seed(step)).cuda()
        k, v = both[:, :, 1:1 + n_kv * hd], both[:, :, 2 + n_kv * hd:2 + 2 * n_kv * hd]
        m.dlens += 1
        ops.kv4_append(m.cache, k, v)
        for i in range(n):
            R.store(want, m.table[i], n_kv, hd, k[i].cpu().numpy(), v[i].cpu().numpy(), int(m.lens[i]) + step)
            rows[i].append((k[i, 0].cpu().numpy(), v[i, 0].cpu().numpy()))
    np.testing.assert_array_equal(m.dpool.cpu().numpy(), want)
    k, v = (torch.full((n, 7, n_kv * hd), 3.25, device="cuda") for _ in range(2))
    ops.kv4_read(m.cache, k, v)
    for i in range(n):
        have = int(m.lens[i]) + 5
        for j, x in enumerate((k, v)):
            got = x[i].cpu().numpy()
            assert (got[:max(0, 7 - have)] == 3.25).all()         # rows before position 0
            np.testing.assert_array_equal(got[2:], R.held(np.stack([r[j] for r in rows[i]])).astype(np.float32))


def test_append_borders_and_odd_values(ops):
    """Elements on and one fp32 step beside every code border, constants, a tiny range, values past fp16, NaN."""
    hd = 64
    rows = []
    for scale in (1.0, 0.37109375, 2.0 ** -14):
        lo = -7.0 * scale
        mid = np.float32(np.float16(lo + 8 * np.float16(scale)))
        b = (mid + np.float32(np.float16(scale)) * (np.arange(-7, 8) - np.float32(0.5))).astype(np.float32)
        r = np.concatenate([b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf)), np.zeros(19)])
        r[-1], r[-2] = lo, lo + 15 * scale
        rows.append(r.astype(np.float32))
    rows += [np.full(hd, 3.3, np.float32), np.full(hd, -0.0, np.float32), np.linspace(1, 1 + 1e-6, hd).astype(np.float32),
             np.linspace(-1e30, 1e30, hd).astype(np.float32), np.linspace(0, 1e-9, hd).astype(np.float32),
             np.where(np.arange(hd) == 5, np.inf, 1).astype(np.float32), np.linspace(1000, 1001, hd).astype(np.float32)]
    k = np.stack(rows)
    n = len(rows)
    pool = torch.zeros(1, 72 * hd, dtype=torch.uint8, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    c = ops.Kv4Cache(pool, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), lens, 1, hd)
    ops.kv4_append(c, torch.from_numpy(k[None]).cuda(), torch.from_numpy(-k[None]).cuda())
    want = np.zeros((1, 72 * hd), np.uint8)
    R.store(want, [0], 1, hd, k, -k, 0)
    np.testing.assert_array_equal(pool.cpu().numpy(), want)
    bad = k.copy()
    bad[2, 9] = np.nan
    ops.kv4_append(c, torch.from_numpy(bad[None]).cuda(), torch.from_numpy(k[None]).cuda())
    gk, gv = torch.zeros(1, n, hd, device="cuda"), torch.zeros(1, n, hd, device="cuda")
    ops.kv4_read(c, gk, gv)
    gk = gk.cpu().numpy()[0]
    assert np.isnan(gk[2]).all() and np.isfinite(np.delete(gk, 2, 0)).all() and torch.isfinite(gv).all()


def check_attention(ops, m, q, n_heads, n_q, out, wi=None, wo=None):
    got = out.cpu().numpy()
    for i, t in enumerate(m.lens):
        K, V = m.loaded(i)
        want, w, top = R.attend(q[i].cpu().numpy(), K, V, n_q)
        tol = 16 * 2.0 ** -24 * max(1.0, top)
        empty = max(0, n_q - t)
        assert (got[i][:empty] == 0).all()
        if t:
            err = np.linalg.norm(got[i] - want) / np.linalg.norm(want)
            assert err <= tol, (i, t, err, tol)
        if wi is not None:
            a, b = wi[i].cpu().numpy(), wo[i].cpu().numpy()
            assert (b[:, t:] == 0).all()
            rows = n_q * (n_heads // m.n_kv)
            assert (np.abs(b[:, :t] - (a[:, :t] + w)) <= tol * w + 2.0 ** -22 * (np.abs(a[:, :t]) + w) + rows * 2.0 ** -126).all(), i


ATTN = [  # heads, kv heads, head_dim, queries, lengths
    (32, 4, 64, 1, [1]), (32, 4, 64, 1, [64, 0, 65, 1, 640]), (32, 8, 128, 1, [300, 1023]), (8, 8, 128, 1, [130]),
    (12, 4, 64, 1, [77, 1000]), (16, 1, 128, 1, [333]), (2, 1, 256, 1, [500, 3]), (6, 2, 192, 1, [129, 0]),
    (14, 2, 64, 3, [2, 300, 1]), (40, 8, 128, 2, [100, 4]), (4, 4, 64, 9, [513, 8, 70]), (8, 2, 128, 65, [65, 200, 3]),
    (2, 2, 256, 33, [90]), (6, 2, 192, 17, [150]), (36, 1, 64, 5, [129]), (8, 2, 64, 130, [1000]),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n_heads,n_kv,hd,n_q,lens", ATTN)
def test_attention(ops, n_heads, n_kv, hd, n_q, lens, weights):
    print(f"case attn {n_heads}/{n_kv} hd={hd} n_q={n_q} {lens} weights={weights}", flush=True)
    rng = np.random.default_rng(n_heads * 7 + hd + n_q + sum(lens))
    m = Made(ops, rng, lens, n_kv, hd, max_pages=max((t + 63) // 64 for t in lens) + 2)
    n = len(lens)
    q = torch.from_numpy(rng.standard_normal((n, n_q, n_heads * hd)).astype(np.float32) * 1.5).cuda()
    out = torch.full_like(q, float("nan"))
    if not weights:
        ops.kv4_attn(out, q, m.cache, n_heads)
        return check_attention(ops, m, q, n_heads, n_q, out)
    wi = torch.from_numpy(rng.random((n, n_kv, m.table.shape[1] * 64)).astype(np.float32)).cuda()
    wo = torch.full_like(wi, float("nan"))
    ops.kv4_attn(out, q, m.cache, n_heads, weights_in=wi, weights_out=wo)
    check_attention(ops, m, q, n_heads, n_q, out, wi, wo)
    # in place, and the same bits
    w2, out2 = wi.clone(), torch.empty_like(out)
    ops.kv4_attn(out2, q, m.cache, n_heads, weights_in=w2, weights_out=w2)
    assert torch.equal(w2, wo) and torch.equal(out, out2)
    assert device_errors() == 0


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n_seq,n_heads,n_kv,hd,n_q,cap", [
    (5, 8, 2, 64, 1, 40), (5, 8, 2, 128, 3, 333), (5, 8, 2, 64, 20, 41), (5, 4, 4, 256, 40, 40), (33, 8, 4, 64, 1, 100),
    (33, 16, 4, 64, 2, 128)])
def test_attention_in_tables_with_room(ops, n_seq, n_heads, n_kv, hd, n_q, cap, weights):
    """Tables of many more pages than the sequences have: their pages are shared out over the blocks all the same."""
    print(f"case room {n_seq} {n_heads}/{n_kv} hd={hd} n_q={n_q} cap={cap} weights={weights}", flush=True)
    rng = np.random.default_rng(cap + n_q + hd)
    lens = [int(t) for t in rng.permutation([0, 1, 64, 65, 700, *rng.integers(1, 500, n_seq)])[:n_seq]]
    m = Made(ops, rng, lens, n_kv, hd, max_pages=cap)
    q = torch.from_numpy(rng.standard_normal((n_seq, n_q, n_heads * hd)).astype(np.float32)).cuda()
    out = torch.full_like(q, float("nan"))
    wi = torch.from_numpy(rng.random((n_seq, n_kv, cap * 64)).astype(np.float32)).cuda() if weights else None
    wo = torch.full_like(wi, float("nan")) if weights else None
    ops.kv4_attn(out, q, m.cache, n_heads, **(dict(weights_in=wi, weights_out=wo) if weights else {}))
    check_attention(ops, m, q, n_heads, n_q, out, wi, wo)
    assert device_errors() == 0


@pytest.mark.parametrize("n_q", [2, 12])
def test_attention_long_and_strided(ops, n_q):
    """Many pages for one head, q inside wider rows and off 16 bytes."""
    rng = np.random.default_rng(11)
    n_heads, n_kv, hd = 4, 1, 128
    m = Made(ops, rng, [9001, 4097], n_kv, hd)
    wide = torch.from_numpy(rng.standard_normal((2, n_q, n_heads * hd + 5)).astype(np.float32)).cuda()
    q = wide[:, :, 3:3 + n_heads * hd]
    out = torch.empty(2, n_q, n_heads * hd, device="cuda")
    wi = torch.zeros(2, n_kv, m.table.shape[1] * 64, device="cuda")
    wo = torch.empty_like(wi)
    ops.kv4_attn(out, q, m.cache, n_heads, weights_in=wi, weights_out=wo)
    check_attention(ops, m, q, n_heads, n_q, out, wi, wo)


@pytest.mark.parametrize("n_q", [1, 6, 45])
def test_attention_sharp_and_flat_scores(ops, n_q):
    """Queries that pick one position (scores of hundreds), and zero queries (every probability the same)."""
    rng = np.random.default_rng(3)
    n_heads, n_kv, hd = 8, 2, 128
    m = Made(ops, rng, [700, 90], n_kv, hd, scale=4.0)
    q = torch.from_numpy((rng.standard_normal((2, n_q, n_heads * hd)) * 30).astype(np.float32)).cuda()
    q[:, :, :2 * hd] = 0
    q[1, :, 3 * hd:4 * hd] *= 1e-20
    out, wi = torch.empty_like(q), torch.zeros(2, n_kv, m.table.shape[1] * 64, device="cuda")
    wo = torch.empty_like(wi)
    ops.kv4_attn(out, q, m.cache, n_heads, weights_in=wi, weights_out=wo)
    check_attention(ops, m, q, n_heads, n_q, out, wi, wo)


@pytest.mark.parametrize("n_q", [1, 11])
def test_attention_small_values_beside_large_scales(ops, n_q):
    """The heaviest position has values a thousandth of the others', as a sink position has."""
    rng = np.random.default_rng(4)
    n_heads, n_kv, hd, t = 4, 1, 64, 190
    m = Made(ops, rng, [t], n_kv, hd)
    q = torch.from_numpy(rng.standard_normal((1, n_q, n_heads * hd)).astype(np.float32)).cuda()
    # a first position along the last query's heads
    m.k[0][0] = q.cpu().numpy()[0, -1].reshape(n_heads, hd).sum(0) * 3
    m.v[0][0] *= 1e-3
    m.v[0][5] *= 1e3
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    out = torch.empty_like(q)
    ops.kv4_attn(out, q, m.cache, n_heads)
    check_attention(ops, m, q, n_heads, n_q, out)


@pytest.mark.parametrize("hd", [64, 192])
@pytest.mark.parametrize("n_q", [1, 3, 12])
def test_attention_tiny_values_after_large_ones(ops, n_q, hd):
    """Values of 2^10 that no query looks at, beside and before those of 2^-14 that all look at: the large ones get
    probabilities below 2^-60, so the small ones alone decide the output."""
    rng = np.random.default_rng(41 + hd)
    n_heads, n_kv, t = 8, 2, 330
    m = Made(ops, rng, [t], n_kv, hd)
    u = rng.choice([-1.0, 1.0], hd)
    seen = np.arange(t) % 64 > 40                             # the end of every page
    seen[:70] = False                                         # and nothing of the first one
    k = rng.standard_normal((t, n_kv, hd)) * 0.1 + np.where(seen, 3.0, -3.0)[:, None, None] * u
    v = rng.standard_normal((t, n_kv, hd)) * np.where(seen, 2.0 ** -14, 2.0 ** 10)[:, None, None]
    m.k[0], m.v[0] = (x.reshape(t, -1).astype(np.float32) for x in (k, v))
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = rng.standard_normal((1, n_q, n_heads, hd)) * 0.1 + 10 / np.sqrt(hd) * u
    q = torch.from_numpy(q.reshape(1, n_q, n_heads * hd).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    ops.kv4_attn(out, q, m.cache, n_heads)
    assert out.abs().max() < 2.0 ** -10
    check_attention(ops, m, q, n_heads, n_q, out)


@pytest.mark.parametrize("n_q,t", [(1, 150), (1, 1100), (3, 150), (9, 150), (9, 1100)])
@pytest.mark.parametrize("size", [1e20, 1e33])
def test_attention_huge_scores(ops, n_q, t, size):
    """Queries so long that every score of a row is below -1e20, or -1e32: the largest position takes it all.  The
    scores of two positions differ by far more than their roundings, so the output is that position's value."""
    rng = np.random.default_rng(6)
    n_heads, n_kv, hd = 8, 2, 64
    m = Made(ops, rng, [t], n_kv, hd)
    m.k[0] = (np.arange(t)[:, None] * 0.01 + 1 + np.zeros(n_kv * hd)).astype(np.float32)   # constant groups: scale 0
    ops.kv4_append(m.cache, torch.from_numpy(m.k[0][None]).cuda(), torch.from_numpy(m.v[0][None]).cuda())
    q = torch.full((1, n_q, n_heads * hd), -size, device="cuda")
    out, w = torch.empty_like(q), torch.zeros(1, n_kv, m.table.shape[1] * 64, device="cuda")
    ops.kv4_attn(out, q, m.cache, n_heads, weights_in=w, weights_out=w)
    V = m.loaded(0)[1][:, 0]                                      # position 0 has the smallest key
    assert (w[0, :, 1:] == 0).all() and (w[0, :, 0] == n_q * n_heads // n_kv).all()
    got = out.cpu().numpy().reshape(n_q, n_heads, hd)
    for h in range(n_heads):
        want = V[h // (n_heads // n_kv)]
        assert (np.abs(got[:, h] - want) <= 2.0 ** -21 * np.abs(want).max()).all()


@pytest.mark.parametrize("n_q", [4, 40])
def test_attention_not_finite(ops, n_q):
    """A NaN key makes the rows that see it NaN, a NaN value its 64 dims; rows that do not see it, and what lies
    behind a length (NaN and infinite pairs there, see Made), stay clean."""
    rng = np.random.default_rng(8)
    n_heads, n_kv, hd, t = 4, 2, 128, 100
    for side in ("k", "v", "q"):
        m = Made(ops, rng, [t, 30], n_kv, hd)
        q = torch.from_numpy(rng.standard_normal((2, n_q, n_heads * hd)).astype(np.float32)).cuda()
        if side == "q":
            q[0, 1, 5] = float("nan")
        else:
            getattr(m, side)[0][t - 2, hd + 70] = np.nan          # head 1, dims 64.., seen by the last two queries
            lens = m.dlens.clone()
            m.dlens.copy_(torch.tensor([t, 0], dtype=torch.int32))
            pad = lambda x: torch.from_numpy(np.stack([x, x])).cuda()
            ops.kv4_append(m.cache, pad(m.k[0]), pad(m.v[0]))
            m.dlens.copy_(lens)
        out = torch.empty_like(q)
        wi = torch.zeros(2, n_kv, m.table.shape[1] * 64, device="cuda")
        wo = torch.empty_like(wi)
        ops.kv4_attn(out, q, m.cache, n_heads, weights_in=wi, weights_out=wo)
        nan = torch.isnan(out).view(2, n_q, n_heads, hd).cpu().numpy()
        want = np.zeros_like(nan)
        if side == "q":
            want[0, 1, 0] = True
        elif side == "k":
            want[0, n_q - 2:, 2:] = True
        else:
            want[0, n_q - 2:, 2:, 64:] = True
        np.testing.assert_array_equal(nan, want)
        assert torch.isfinite(wo[1]).all()


def test_attention_bad_pages_are_reported(ops):
    rng = np.random.default_rng(9)
    n_heads, n_kv, hd = 4, 2, 64
    m = Made(ops, rng, [100, 200, 90], n_kv, hd)
    q = torch.from_numpy(rng.standard_normal((3, 1, n_heads * hd)).astype(np.float32)).cuda()
    out, good = torch.empty_like(q), torch.empty_like(q)
    ops.kv4_attn(good, q, m.cache, n_heads)
    assert device_errors() == 0
    for page in (-1, m.n_pages, 2 ** 31 - 1):
        t = m.dtable.clone()
        t[1, 3] = page
        c = ops.Kv4Cache(m.dpool, t, m.dlens, n_kv, hd)
        before = m.dpool.clone()
        wi = torch.zeros(3, n_kv, t.shape[1] * 64, device="cuda")
        wo = torch.empty_like(wi)
        ops.kv4_attn(out, q, c, n_heads, weights_in=wi, weights_out=wo)
        assert device_errors() == 4
        assert torch.isnan(out[1]).all() and torch.equal(out[0::2], good[0::2]) and torch.isfinite(wo[0::2]).all()
        k = torch.zeros(3, 70, n_kv * hd, device="cuda")
        v = torch.zeros_like(k)
        ops.kv4_read(c, k, v)
        assert device_errors() == 4 and torch.isnan(k[1, -3]).all() and torch.isfinite(k[0]).all()
        row = torch.randn(3, 1, n_kv * hd, device="cuda")
        ops.kv4_append(c, row, row)
        assert device_errors() == 4
        changed = (m.dpool != before).any(1).nonzero().flatten().tolist()
        assert set(changed) <= {int(m.table[0, 1]), int(m.table[2, 1])}
        m.dpool.copy_(before)
    for length in (-1, t.shape[1] * 64 + 1):
        lens = m.dlens.clone()
        lens[1] = length
        c = ops.Kv4Cache(m.dpool, m.dtable, lens, n_kv, hd)
        ops.kv4_attn(out, q, c, n_heads)
        assert device_errors() == 4
        assert torch.isnan(out[1]).all() and torch.equal(out[0::2], good[0::2])


EVICT = [  # kv heads, head_dim, lengths, budget, sink, recent
    (1, 64, [1], 1, 0, 0), (2, 64, [65, 64, 0, 200], 64, 4, 20), (1, 128, [1000], 130, 0, 0), (2, 128, [700, 63], 65, 65, 0),
    (1, 192, [300], 100, 0, 100), (1, 256, [129, 500], 128, 7, 121), (3, 64, [3000, 100], 1025, 4, 300), (1, 64, [70], 1, 0, 0),
    (2, 64, [2500], 2200, 1, 64), (1, 64, [16385, 90], 64, 1, 7), (2, 64, [20000, 16384, 0], 4500, 4, 300),
    (1, 64, [40000], 40000, 0, 0), (1, 64, [33000], 100, 60, 40),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_kv,hd,lens,budget,sink,recent", EVICT)
def test_evict(ops, n_kv, hd, lens, budget, sink, recent, in_place):
    print(f"case evict {n_kv} {hd} {lens} {budget} {sink} {recent} in_place={in_place}", flush=True)
    rng = np.random.default_rng(hd + budget)
    n = len(lens)
    m = Made(ops, rng, lens, n_kv, hd, max_pages=max(max(lens), budget) // 64 + 2)
    slots = m.table.shape[1] * 64
    w = np.round(np.exp(rng.standard_normal((n, n_kv, slots)) * 2) * 8).astype(np.float32) / 8   # many ties
    w[rng.random(w.shape) < 0.02] = np.nan
    w[rng.random(w.shape) < 0.05] *= -0.0
    w[rng.random(w.shape) < 0.01] = np.inf
    dw = torch.from_numpy(w).cuda()
    kept = torch.full((n, n_kv, budget), -7, dtype=torch.int32, device="cuda")
    if in_place:
        to, tw, pool, table = m.cache, dw, m.dpool, m.table
    else:
        dp = (budget + 63) // 64 + 1
        table = rng.permutation(n * dp).astype(np.int32).reshape(n, dp)
        pool = torch.from_numpy(rng.integers(0, 256, (n * dp, n_kv * 72 * hd), dtype=np.uint8)).cuda()
        tw = torch.full((n, n_kv, dp * 64), 7.0, device="cuda")
        to = ops.Kv4Cache(pool, torch.from_numpy(table).cuda(), torch.full((n,), -3, dtype=torch.int32, device="cuda"), n_kv, hd)
    before, src_before = pool.cpu().numpy(), m.dpool.clone()
    ops.kv4_evict(m.cache, to, dw, tw, budget, sink, recent, kept)
    got, want, host = pool.cpu().numpy(), before.copy(), m.pool.copy()
    fill(host, m)
    for i, t in enumerate(lens):
        new = min(t, budget)
        assert int(to.lens[i]) == new
        for p in range((new + 63) // 64):
            want[table[i, p]] = 0
        for h in range(n_kv):
            f = R.keep(w[i, h], t, budget, sink, recent)
            g = kept[i, h].cpu().numpy()
            np.testing.assert_array_equal(g[:new], f)
            assert (g[new:] == -1).all()
            gw = tw[i, h].cpu().numpy()
            np.testing.assert_array_equal(gw[:new].view(np.uint32), w[i, h, f].view(np.uint32))
            assert (gw[new:] == 0).all()
            # the kept rows' codes and pairs, page by page of the destination
            src = host[m.table[i]].reshape(-1, n_kv, 72 * hd)[:, h]
            for p in range((new + 63) // 64):
                g = f[64 * p:64 * p + 64]
                b = want[table[i, p]].reshape(n_kv, -1)[h]
                for at, shift, pair in R.places(hd):
                    code = (src[(g // 64)[:, None], at[g % 64]] >> shift[g % 64].astype(np.uint8)) & 15
                    np.bitwise_or.at(b, at[:len(g)], code << shift[:len(g)].astype(np.uint8))
                    for o in (0, 1):
                        b.view(np.uint16)[pair[:len(g)] + o] = src.view(np.uint16)[(g // 64)[:, None], pair[g % 64] + o]
    np.testing.assert_array_equal(got, want)
    if not in_place:
        assert torch.equal(m.dpool, src_before) and m.dlens.tolist() == list(lens)
    assert device_errors() == 0


def test_evict_reports_bad_pages(ops):
    rng = np.random.default_rng(12)
    n_kv, hd = 1, 64
    m = Made(ops, rng, [200, 200], n_kv, hd)
    t = m.dtable.clone()
    t[0, 1] = 10 ** 6
    c = ops.Kv4Cache(m.dpool, t, m.dlens, n_kv, hd)
    w = torch.rand(2, n_kv, t.shape[1] * 64, device="cuda")
    to = ops.Kv4Cache(torch.zeros(4, 72 * hd, dtype=torch.uint8, device="cuda"), torch.tensor([[0, 1], [2, -5]], dtype=torch.int32, device="cuda"),
                      torch.zeros(2, dtype=torch.int32, device="cuda"), n_kv, hd)
    wd = torch.zeros(2, n_kv, 128, device="cuda")
    kept = torch.empty(2, n_kv, 100, dtype=torch.int32, device="cuda")
    ops.kv4_evict(c, to, w, wd, 100, 0, 10, kept)
    assert device_errors() == 4
    k, v = torch.zeros(2, 100, hd, device="cuda"), torch.zeros(2, 100, hd, device="cuda")
    ops.kv4_read(to, k, v)
    assert device_errors() == 4
    lost = ((kept[0, 0] >= 64) & (kept[0, 0] < 128)).cpu()
    assert lost.any() and torch.equal(torch.isnan(k[0]).all(1).cpu(), lost) and torch.equal(torch.isnan(v[0]).all(1).cpu(), lost)
    assert torch.isfinite(k[1, :64]).all() and torch.isnan(k[1, 64:]).all()


def test_serving_run(ops):
    """A batch as it is served: prompts appended in chunks with their weights, decode steps, evictions in place between
    them, every output against 64 bits on a cache that the oracle carries along."""
    rng = np.random.default_rng(21)
    n, n_heads, n_kv, hd, budget, sink, recent = 3, 8, 2, 64, 100, 2, 30
    mp = 4
    table = rng.permutation(n * mp).astype(np.int32).reshape(n, mp)
    pool = torch.zeros(n * mp, n_kv * 72 * hd, dtype=torch.uint8, device="cuda")
    lens = torch.zeros(n, dtype=torch.int32, device="cuda")
    c = ops.Kv4Cache(pool, torch.from_numpy(table).cuda(), lens, n_kv, hd)
    w = torch.zeros(n, n_kv, mp * 64, device="cuda")
    held = [[np.zeros((0, hd)) for _ in range(2 * n_kv)] for _ in range(n)]   # per head: K, V
    hw = [[np.zeros(0) for _ in range(n_kv)] for _ in range(n)]
    for step, new in enumerate([70, 64, 1, 1, 5, 1, 60, 1]):
        k, v = rng.standard_normal((2, n, new, n_kv * hd)).astype(np.float32)
        q = rng.standard_normal((n, new, n_heads * hd)).astype(np.float32)
        lens += new
        ops.kv4_append(c, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        out = torch.empty(n, new, n_heads * hd, device="cuda")
        ops.kv4_attn(out, torch.from_numpy(q).cuda(), c, n_heads, weights_in=w, weights_out=w)
        got, gw = out.cpu().numpy(), w.cpu().numpy()
        for i in range(n):
            for h in range(n_kv):
                for j, x in enumerate((k, v)):
                    held[i][2 * h + j] = np.concatenate([held[i][2 * h + j], R.held(x[i][:, h * hd:(h + 1) * hd])])
            K, V = np.stack(held[i][0::2]), np.stack(held[i][1::2])
            want, p, top = R.attend(q[i], K, V, new)
            tol = 16 * 2.0 ** -24 * max(1.0, top)
            assert np.linalg.norm(got[i] - want) <= tol * np.linalg.norm(want), (step, i)
            for h in range(n_kv):
                hw[i][h] = np.concatenate([hw[i][h], np.zeros(new)]) + p[h]
                t = len(hw[i][h])
                assert (np.abs(gw[i, h, :t] - hw[i][h]) <= (tol + (step + 1) * 2.0 ** -22) * hw[i][h] + 2.0 ** -100).all() and (gw[i, h, t:] == 0).all()
        if step in (1, 5, 6):
            kept = torch.empty(n, n_kv, budget, dtype=torch.int32, device="cuda")
            ops.kv4_evict(c, c, w, w, budget, sink, recent, kept)
            assert lens.tolist() == [budget] * n
            for i in range(n):
                for h in range(n_kv):
                    f = R.keep(gw[i, h], len(hw[i][h]), budget, sink, recent)
                    np.testing.assert_array_equal(kept[i, h].cpu().numpy(), f)
                    hw[i][h] = hw[i][h][f]
                    for j in range(2):
                        held[i][2 * h + j] = held[i][2 * h + j][f]
    assert device_errors() == 0


def test_graph_replay_follows_lens_and_table(ops):
    """A captured decode step replayed while the lengths, the table and the inputs change, eager work between."""
    rng = np.random.default_rng(30)
    n_heads, n_kv, hd = 8, 2, 128
    m = Made(ops, rng, [60, 200], n_kv, hd, max_pages=5)
    n = 2
    q = torch.randn(n, 1, n_heads * hd, device="cuda")
    k, v = (torch.randn(n, 1, n_kv * hd, device="cuda") for _ in range(2))
    out, w = torch.empty_like(q), torch.zeros(n, n_kv, 320, device="cuda")
    import libinferbit_amd as L
    ws = torch.empty(L.lib().ibh_kv4_attn_workspace_bytes(m.cache.ref, n_heads, 1, 1), dtype=torch.uint8, device="cuda")

    def step():
        m.dlens.add_(1)
        ops.kv4_append(m.cache, k, v)
        ops.kv4_attn(out, q, m.cache, n_heads, weights_in=w, weights_out=w, ws=ws)

    start = (m.dpool.clone(), m.dlens.clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    inputs = [[torch.randn_like(x) for x in (q, k, v)] for _ in range(6)]
    results = []
    for mode in ("graph", "eager"):
        m.dpool.copy_(start[0]); m.dlens.copy_(start[1]); w.zero_()
        got = []
        for i, xs in enumerate(inputs):
            for a, b in zip((q, k, v), xs):
                a.copy_(b)
            if i == 3:
                m.dlens[0] = 0                                   # a sequence ends, another begins in its row
                w[0] = 0
            g.replay() if mode == "graph" else step()
            torch.cuda.synchronize()
            got.append((out.clone(), w.clone(), m.dpool.clone()))
        results.append(got)
    for a, b in zip(*results):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_another_stream(ops):
    rng = np.random.default_rng(31)
    m = Made(ops, rng, [300], 2, 64)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q = torch.randn(1, 1, 8 * 64, device="cuda")
        out = torch.empty_like(q)
        ops.kv4_attn(out, q, m.cache, 8)
    s.synchronize()
    check_attention(ops, m, q, 8, 1, out)


def test_python_refusals(ops):
    rng = np.random.default_rng(32)
    m = Made(ops, rng, [10, 20], 2, 64)
    c = m.cache
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    with pytest.raises(ValueError):
        ops.kv4_append(c, z(2, 1, 127), z(2, 1, 127))
    with pytest.raises(ValueError):
        ops.kv4_append(c, z(2, 2, 128), z(2, 1, 128))
    with pytest.raises(ValueError):
        ops.kv4_append(c, z(3, 1, 128), z(3, 1, 128))
    with pytest.raises(ValueError):
        ops.kv4_append(c, z(2, 128, 3).transpose(1, 2), z(2, 128, 3).transpose(1, 2))
    with pytest.raises(TypeError):
        ops.kv4_read(c, z(2, 1, 128, dtype=torch.float16), z(2, 1, 128, dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.kv4_attn(torch.zeros(2, 1, 256), z(2, 1, 256), c, 4)
    with pytest.raises(ValueError):
        ops.kv4_attn(z(2, 1, 256), z(2, 1, 256), c, 4, weights_in=z(2, 2, 64))
    with pytest.raises(ValueError):
        ops.kv4_attn(z(2, 1, 256), z(2, 1, 256), c, 4, weights_in=z(2, 2, 63), weights_out=z(2, 2, 63))
    import libinferbit_amd as L
    with pytest.raises(L.IbhError):
        ops.kv4_attn(z(2, 1, 192), z(2, 1, 192), c, 3)
    with pytest.raises(TypeError):
        ops.kv4_evict(c, c, z(2, 2, 64), z(2, 2, 64), 5, 0, 0, z(2, 2, 5))
    with pytest.raises(L.IbhError):                               # half in place
        ops.kv4_evict(c, c, z(2, 2, 64), z(2, 2, 64), 5, 0, 0, z(2, 2, 5, dtype=torch.int32))
    with pytest.raises(L.IbhError):
        ops.kv4_attn(z(2, 1, 2048), z(2, 1, 2048), Made(ops, rng, [4100, 1], 2, 64).cache, 32, ws=z(8, dtype=torch.uint8))
