"""The paged 4-bit cache at the limits of its calls: large batches and tables with
room, the library's workspace, pages that sequences share, long evictions."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import kv4 as R
from test_kv4_gpu import Made, check_attention, device_errors, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def batch(ops, n_seq, n_kv, hd, max_pages, held):
    """n_seq sequences in rows of max_pages pages; those of `held` {sequence: (K, V) rows} hold something, each one page."""
    table = torch.zeros(n_seq, max_pages, dtype=torch.int32, device="cuda")
    lens = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    pool = torch.zeros(max(1, len(held)), n_kv * 72 * hd, dtype=torch.uint8)
    for j, (i, (k, v)) in enumerate(held.items()):
        R.store(pool.numpy(), [j], n_kv, hd, k, v, 0)
        table[i, 0], lens[i] = j, len(k)
    return ops.Kv4Cache(pool.cuda(), table, lens, n_kv, hd)


def some(rng, where, n_kv, hd):
    return {i: tuple(rng.standard_normal((2, n, n_kv * hd)).astype(np.float32)) for i, n in where.items()}


@pytest.mark.parametrize("n_seq,n_kv,max_pages,weights", [(256, 8, 2048, False), (64, 8, 8192, False), (256, 8, 2048, True)])
def test_attention_of_a_batch_in_long_tables(ops, n_seq, n_kv, max_pages, weights):
    """2^22 pages of table: what a call launches goes by its blocks, not by its tables' room."""
    print(f"case long tables {n_seq} {n_kv} {max_pages} {weights}", flush=True)
    rng = np.random.default_rng(81)
    hd, n_heads = 64, n_kv
    held = some(rng, {0: 3, 17: 64, n_seq - 1: 1}, n_kv, hd)
    c = batch(ops, n_seq, n_kv, hd, max_pages, held)
    q = torch.from_numpy(rng.standard_normal((n_seq, 1, n_heads * hd)).astype(np.float32)).cuda()
    out = torch.full_like(q, float("nan"))
    w = torch.full((n_seq, n_kv, 64 * max_pages), 1.0, device="cuda") if weights else None
    ops.kv4_attn(out, q, c, n_heads, **(dict(weights_in=w, weights_out=w) if weights else {}))
    got = out.cpu().numpy()
    for i in range(n_seq):
        if i not in held:
            assert (got[i] == 0).all()
            continue
        K, V = (R.held(x).reshape(-1, n_kv, hd).transpose(1, 0, 2) for x in held[i])
        want, p, top = R.attend(q[i].cpu().numpy(), K, V, 1)
        tol = 16 * 2.0 ** -24 * max(1.0, top)
        assert np.linalg.norm(got[i] - want) <= tol * np.linalg.norm(want)
        if weights:
            n = K.shape[1]
            assert (np.abs(w[i, :, :n].cpu().numpy() - 1 - p) <= tol * p + 2.0 ** -22 * (1 + p)).all()
    if weights:
        assert float(w.sum(dtype=torch.float64)) == pytest.approx(sum(n_kv * (len(k) + 1) for k, _ in held.values()), rel=1e-5)
    assert device_errors() == 0


def test_append_and_read_of_a_large_batch(ops):
    """More than 2^22 blocks: 70000 sequences of 32 KV heads, all but two left out."""
    rng = np.random.default_rng(82)
    n_seq, n_kv, hd = 70000, 32, 64
    table = torch.zeros(n_seq, 1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    lens[3], lens[n_seq - 1], table[n_seq - 1, 0] = 1, 1, 1
    pool = torch.zeros(2, n_kv * 72 * hd, dtype=torch.uint8, device="cuda")
    c = ops.Kv4Cache(pool, table, lens, n_kv, hd)
    k, v = (torch.zeros(n_seq, 1, n_kv * hd, device="cuda") for _ in range(2))
    rows = rng.standard_normal((2, 2, 1, n_kv * hd)).astype(np.float32)
    for x, r in zip((k, v), rows):
        x[3], x[n_seq - 1] = torch.from_numpy(r[0]).cuda(), torch.from_numpy(r[1]).cuda()
    ops.kv4_append(c, k, v)
    want = np.zeros((2, n_kv * 72 * hd), np.uint8)
    for j in range(2):
        R.store(want, [j], n_kv, hd, rows[0][j], rows[1][j], 0)
    np.testing.assert_array_equal(pool.cpu().numpy(), want)
    ops.kv4_read(c, k, v)
    for x, r in zip((k, v), rows):
        for i, y in ((3, r[0]), (n_seq - 1, r[1])):
            np.testing.assert_array_equal(x[i].cpu().numpy(), R.held(y).astype(np.float32))
        assert int((x != 0).any(-1).sum()) == 2
    assert device_errors() == 0


def test_evict_into_a_large_batch(ops):
    """2^22 destination pages, nearly all of them without a kept position."""
    rng = np.random.default_rng(83)
    n_seq, n_kv, hd, budget = 256, 8, 64, 20
    held = some(rng, {0: 3, 17: 64, n_seq - 1: 21}, n_kv, hd)
    c = batch(ops, n_seq, n_kv, hd, 1, held)
    table = torch.zeros(n_seq, 2048, dtype=torch.int32, device="cuda")
    for j, i in enumerate(held):
        table[i, 0] = j
    to = ops.Kv4Cache(torch.zeros(3, n_kv * 72 * hd, dtype=torch.uint8, device="cuda"), table,
                      torch.full((n_seq,), -1, dtype=torch.int32, device="cuda"), n_kv, hd)
    w = torch.from_numpy(rng.random((n_seq, n_kv, 64)).astype(np.float32)).cuda()
    dw = torch.full((n_seq, n_kv, 64 * 2048), 7.0, device="cuda")
    kept = torch.empty(n_seq, n_kv, budget, dtype=torch.int32, device="cuda")
    ops.kv4_evict(c, to, w, dw, budget, 2, 5, kept)
    assert to.lens.tolist() == [min(budget, len(held[i][0])) if i in held else 0 for i in range(n_seq)]
    k, v = (torch.zeros(n_seq, budget, n_kv * hd, device="cuda") for _ in range(2))
    ops.kv4_read(to, k, v)
    for i, kv in held.items():
        n = len(kv[0])
        for h in range(n_kv):
            f = R.keep(w[i, h].cpu().numpy(), n, budget, 2, 5)
            np.testing.assert_array_equal(kept[i, h, :len(f)].cpu().numpy(), f)
            np.testing.assert_array_equal(dw[i, h, :len(f)].cpu().numpy(), w[i, h].cpu().numpy()[f])
            for got, x in zip((k, v), kv):
                want = R.held(x).astype(np.float32)[f][:, h * hd:(h + 1) * hd]
                np.testing.assert_array_equal(got[i, budget - len(f):, h * hd:(h + 1) * hd].cpu().numpy(), want)
    assert int((dw != 0).sum()) == sum(n_kv * min(budget, len(x[0])) for x in held.values())
    assert device_errors() == 0


# ── workspaces ───────────────────────────────────────────────────────────────
def raw(name, *args):
    import libinferbit_amd as L
    rc = getattr(L.lib(), name)(*args)
    msg = L.lib().ibh_last_error() if rc else b""
    return rc, msg.decode()


@pytest.mark.parametrize("n_q,lens,weights", [(1, [900], True), (1, [3000], False), (1, [3000], True), (12, [700], True)])
def test_attention_in_the_library_workspace(ops, n_q, lens, weights):
    """ws NULL: the same bits as in a workspace of the caller's."""
    import libinferbit_amd as L
    rng = np.random.default_rng(84)
    n_heads, n_kv, hd = 8, 2, 64
    m = Made(ops, rng, lens, n_kv, hd)
    assert 0 <= L.lib().ibh_kv4_attn_workspace_bytes(m.cache.ref, n_heads, n_q, weights) <= 4 << 20
    q = torch.randn(len(lens), n_q, n_heads * hd, device="cuda")
    w = torch.rand(len(lens), n_kv, m.table.shape[1] * 64, device="cuda") if weights else None
    out, own = torch.empty_like(q), torch.empty_like(q)
    w2 = None if w is None else torch.empty_like(w)
    w3 = None if w is None else torch.empty_like(w)
    ptr = lambda t: None if t is None else t.data_ptr()
    rc, msg = raw("ibh_kv4_attn", m.cache.ref, out.data_ptr(), q.data_ptr(), n_heads, n_q, n_heads * hd, ptr(w), ptr(w2),
                  None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, msg
    ops.kv4_attn(own, q, m.cache, n_heads, weights_in=w, weights_out=w3)
    assert torch.equal(out, own) and (w is None or torch.equal(w2, w3))


def test_calls_beyond_the_library_workspace_are_refused(ops):
    import libinferbit_amd as L
    rng = np.random.default_rng(85)
    n_heads, n_kv, hd = 8, 2, 64
    m = Made(ops, rng, [17000, 300], n_kv, hd)
    stream = torch.cuda.current_stream().cuda_stream
    q = torch.randn(2, 40, n_heads * hd, device="cuda")
    out = torch.full_like(q, 3.5)
    assert L.lib().ibh_kv4_attn_workspace_bytes(m.cache.ref, n_heads, 40, 0) > 4 << 20
    rc, msg = raw("ibh_kv4_attn", m.cache.ref, out.data_ptr(), q.data_ptr(), n_heads, 40, n_heads * hd, None, None, None, 0, stream)
    assert rc == -3 and "workspace" in msg
    slots = m.table.shape[1] * 64
    # an eviction's need goes by its KV heads: 4 rows fit, 8 do not
    w = torch.rand(2, n_kv, slots, device="cuda")
    assert L.lib().ibh_kv4_evict_workspace_bytes(m.cache.ref) <= 4 << 20
    kept, want = (torch.empty(2, n_kv, 100, dtype=torch.int32, device="cuda") for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    to = lambda: ops.Kv4Cache(torch.zeros(4, n_kv * 72 * hd, dtype=torch.uint8, device="cuda"), table, torch.zeros(2, dtype=torch.int32, device="cuda"), n_kv, hd)
    a, b, wa, wb = to(), to(), *(torch.zeros(2, n_kv, 128, device="cuda") for _ in range(2))
    rc, msg = raw("ibh_kv4_evict", m.cache.ref, a.ref, w.data_ptr(), wa.data_ptr(), 100, 3, 7, kept.data_ptr(), None, 0, stream)
    assert rc == 0, msg
    ops.kv4_evict(m.cache, b, w, wb, 100, 3, 7, want)
    assert torch.equal(kept, want) and torch.equal(a.pool, b.pool) and torch.equal(wa, wb)
    both = ops.Kv4Cache(m.dpool, torch.cat([m.dtable] * 2), torch.cat([m.dlens] * 2), n_kv, hd)
    big = ops.Kv4Cache(torch.zeros(8, n_kv * 72 * hd, dtype=torch.uint8, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2),
                       torch.full((4,), 9, dtype=torch.int32, device="cuda"), n_kv, hd)
    w2, wd, k2 = torch.cat([w] * 2), torch.full((4, n_kv, 128), 3.5, device="cuda"), torch.full((4, n_kv, 100), -9, dtype=torch.int32, device="cuda")
    rc, msg = raw("ibh_kv4_evict", both.ref, big.ref, w2.data_ptr(), wd.data_ptr(), 100, 3, 7, k2.data_ptr(), None, 0, stream)
    assert rc == -3 and "workspace" in msg
    torch.cuda.synchronize()
    assert (out == 3.5).all() and (wd == 3.5).all() and (k2 == -9).all() and big.lens.tolist() == [9] * 4


# ── unequal counts ───────────────────────────────────────────────────────────
def test_a_batch_of_unequal_counts(ops):
    """Decode steps, a verify step that is cut back, and a prompt chunk in one batch: a call for each count, over caches of
    those sequences' rows and one pool, weights included."""
    rng = np.random.default_rng(86)
    n_heads, n_kv, hd, mp = 4, 2, 64, 4
    start, new = [100, 63, 0, 70], [1, 5, 90, 1]
    m = Made(ops, rng, start, n_kv, hd, max_pages=mp)
    w = torch.from_numpy(rng.random((4, n_kv, mp * 64)).astype(np.float32)).cuda()
    for i, t in enumerate(start):
        w[i, :, t:] = 0
    w0 = w.cpu().numpy()
    lens = list(start)
    probs, most = [np.zeros((n_kv, mp * 64)) for _ in start], 1.0
    for step, counts in enumerate((new, [1, 1, 1, 1])):
        for i, n in enumerate(counts):
            lens[i] += n
        m.dlens.copy_(torch.tensor(lens, dtype=torch.int32))
        for n in sorted(set(counts)):
            idx = torch.tensor([i for i, x in enumerate(counts) if x == n], device="cuda")
            c = ops.Kv4Cache(m.dpool, m.dtable[idx], m.dlens[idx], n_kv, hd)
            k, v = rng.standard_normal((2, len(idx), n, n_kv * hd)).astype(np.float32)
            q = rng.standard_normal((len(idx), n, n_heads * hd)).astype(np.float32)
            out, wi = torch.empty(len(idx), n, n_heads * hd, device="cuda"), w[idx]
            ops.kv4_append(c, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
            ops.kv4_attn(out, torch.from_numpy(q).cuda(), c, n_heads, weights_in=wi, weights_out=wi)
            w[idx] = wi
            for j, i in enumerate(idx.tolist()):
                m.k[i], m.v[i] = np.concatenate([m.k[i], k[j]]), np.concatenate([m.v[i], v[j]])
                want, p, top = R.attend(q[j], *m.loaded(i), n)
                probs[i][:, :lens[i]] += p
                most = max(most, top)
                assert np.linalg.norm(out[j].cpu().numpy() - want) <= 16 * 2.0 ** -24 * max(1.0, top) * np.linalg.norm(want)
        if step == 0:                                             # three of the five drafts are rejected
            lens[1] -= 3
            m.k[1], m.v[1] = m.k[1][:lens[1]], m.v[1][:lens[1]]
            w[1, :, lens[1]:] = 0
            probs[1][:, lens[1]:] = 0
    for i in range(4):
        want = w0[i] + probs[i]
        assert (np.abs(w[i].cpu().numpy() - want) <= (16 * 2.0 ** -24 * most + 2 * 2.0 ** -22) * want + 2.0 ** -100).all()   # as above, and each call's sums
    assert device_errors() == 0


# ── shared pages ─────────────────────────────────────────────────────────────
@pytest.mark.parametrize("n_q,weights", [(1, False), (1, True), (5, True), (20, True)])
def test_sequences_that_share_full_pages(ops, n_q, weights):
    """Three sequences on one prompt's 5 full pages, one of them with nothing else: each as if the pages were its own, an
    eviction into other pages too, and the shared pages unchanged."""
    print(f"case shared n_q={n_q} weights={weights}", flush=True)
    rng = np.random.default_rng(87)
    n_heads, n_kv, hd, lens = 8, 2, 64, [400, 320, 377]
    m = Made(ops, rng, lens, n_kv, hd)
    for i in (1, 2):
        m.k[i][:320], m.v[i][:320] = m.k[0][:320], m.v[0][:320]
        m.table[i, :5] = m.table[0, :5]
    m.dtable.copy_(torch.from_numpy(m.table))
    for i in (0, 2):                                              # what lies behind the shared pages
        one = ops.Kv4Cache(m.dpool, m.dtable[i:i + 1].contiguous(), m.dlens[i:i + 1].contiguous(), n_kv, hd)
        ops.kv4_append(one, *(torch.from_numpy(x[i][None, 320:]).cuda() for x in (m.k, m.v)))
    before = m.dpool.clone()
    q = torch.from_numpy(rng.standard_normal((3, n_q, n_heads * hd)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    wi = torch.from_numpy(rng.random((3, n_kv, m.table.shape[1] * 64)).astype(np.float32)).cuda() if weights else None
    wo = torch.empty_like(wi) if weights else None
    ops.kv4_attn(out, q, m.cache, n_heads, **(dict(weights_in=wi, weights_out=wo) if weights else {}))
    check_attention(ops, m, q, n_heads, n_q, out, wi, wo)
    if weights:
        budget, sink, recent = 200, 4, 50
        to = ops.Kv4Cache(torch.zeros(12, n_kv * 72 * hd, dtype=torch.uint8, device="cuda"), torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4),
                          torch.zeros(3, dtype=torch.int32, device="cuda"), n_kv, hd)
        wd, kept = torch.empty(3, n_kv, 256, device="cuda"), torch.empty(3, n_kv, budget, dtype=torch.int32, device="cuda")
        ops.kv4_evict(m.cache, to, wo, wd, budget, sink, recent, kept)
        k, v = (torch.empty(3, budget, n_kv * hd, device="cuda") for _ in range(2))
        ops.kv4_read(to, k, v)
        for i in range(3):
            for h in range(n_kv):
                f = R.keep(wo[i, h].cpu().numpy(), lens[i], budget, sink, recent)
                np.testing.assert_array_equal(kept[i, h].cpu().numpy(), f)
                for got, x in ((k, m.k), (v, m.v)):
                    want = R.held(x[i]).astype(np.float32)[f][:, h * hd:(h + 1) * hd]
                    np.testing.assert_array_equal(got[i, :, h * hd:(h + 1) * hd].cpu().numpy(), want)
    assert torch.equal(m.dpool, before) and device_errors() == 0


# ── evictions of long rows ───────────────────────────────────────────────────
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sink,recent", [   # 17 to 32 segments of a row; segments of more than 4096 positions
    ([70001, 300], 5000, 3, 1000), ([131071], 64, 1, 7), ([131072, 0, 65537], 66000, 0, 0), ([200000, 90], 150001, 4, 2000),
    ([200000], 199999, 0, 0), ([262143, 131071], 8192, 16, 2048)])
def test_evict_long_rows(ops, lens, budget, sink, recent, in_place):
    print(f"case evict long {lens} {budget} {sink} {recent} in_place={in_place}", flush=True)
    rng = np.random.default_rng(budget + len(lens))
    n, n_kv, hd = len(lens), 1, 64
    mp = (max(lens) + 63) // 64
    pool = rng.integers(0, 256, (n * mp, 72 * hd), dtype=np.uint8)   # the bytes are moved, whatever they are
    table = rng.permutation(n * mp).astype(np.int32).reshape(n, mp)
    w = np.round(np.exp(rng.standard_normal((n, n_kv, mp * 64)) * 2) * 8).astype(np.float32) / 8   # ties in every segment
    w[rng.random(w.shape) < 0.02] = np.nan
    dev = lambda x: torch.from_numpy(x).cuda()
    dpool, dw = dev(pool.copy()), dev(w)
    src = ops.Kv4Cache(dpool, dev(table), torch.tensor(lens, dtype=torch.int32, device="cuda"), n_kv, hd)
    to, tw, ttable, before = src, dw, table, pool
    if not in_place:
        dp = (budget + 63) // 64 + 1
        ttable = rng.permutation(n * dp).astype(np.int32).reshape(n, dp)
        before = rng.integers(0, 256, (n * dp, 72 * hd), dtype=np.uint8)
        tw = torch.full((n, n_kv, dp * 64), 7.0, device="cuda")
        to = ops.Kv4Cache(dev(before.copy()), dev(ttable), torch.full((n,), -3, dtype=torch.int32, device="cuda"), n_kv, hd)
    kept = torch.full((n, n_kv, budget), -7, dtype=torch.int32, device="cuda")
    ops.kv4_evict(src, to, dw, tw, budget, sink, recent, kept)
    want = before.copy()
    for i, t in enumerate(lens):
        new = min(t, budget)
        f = R.keep(w[i, 0], t, budget, sink, recent)
        assert int(to.lens[i]) == new
        g = kept[i, 0].cpu().numpy()
        np.testing.assert_array_equal(g[:new], f)
        gw = tw[i, 0].cpu().numpy()
        np.testing.assert_array_equal(gw[:new].view(np.uint32), w[i, 0, f].view(np.uint32))
        assert (g[new:] == -1).all() and (gw[new:] == 0).all()
        rows = pool[table[i]]                                     # [page, byte]
        half = rows.view(np.uint16)
        pages = (new + 63) // 64
        for at, shift, pair in R.places(hd):
            code = np.zeros((pages * 64, hd), np.uint8)
            code[:new] = (rows[(f // 64)[:, None], at[f % 64]] >> shift[f % 64].astype(np.uint8)) & 15
            b = np.zeros((pages, 72 * hd), np.uint8)
            for hi in (0, 4):                                     # each byte holds two codes
                use = shift == hi
                b[:, at[use]] |= code.reshape(pages, 64, hd)[:, use] << hi
            pr = np.zeros((pages * 64, 2), np.uint16)
            pr[:new] = half[(f // 64)[:, None], pair[f % 64][:, :1] + np.arange(2)]
            b.view(np.uint16)[:, pair[:, :1] + np.arange(2)] = pr.reshape(pages, 64, 2)
            lo = int(at.min())
            want[ttable[i, :pages], lo:lo + 36 * hd] = b[:, lo:lo + 36 * hd]
    np.testing.assert_array_equal(to.pool.cpu().numpy(), want)
    assert device_errors() == 0


# ── far pages, graphs, streams ───────────────────────────────────────────────
def test_pages_beyond_four_gigabytes(ops):
    """Pages at both ends of a pool of 5 GB: stored, read, attended to by few and by many rows, moved in place and away."""
    rng = np.random.default_rng(90)
    n_heads, n_kv, hd, lens = 8, 8, 128, [300, 130]
    size = n_kv * 72 * hd
    n_pages = (5 << 30) // size
    pool = torch.empty(n_pages, size, dtype=torch.uint8, device="cuda")
    table = np.array([[n_pages - 1, 0, n_pages - 2, n_pages // 2, n_pages - 7], [n_pages - 3, n_pages - 4, 1, 2, 3]], np.int32)
    c = ops.Kv4Cache(pool, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), n_kv, hd)
    k, v = rng.standard_normal((2, 2, 300, n_kv * hd)).astype(np.float32)
    ops.kv4_append(c, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    rk, rv = (torch.empty(2, 300, n_kv * hd, device="cuda") for _ in range(2))
    ops.kv4_read(c, rk, rv)
    rows = [(k[i, 300 - t:], v[i, 300 - t:]) for i, t in enumerate(lens)]
    for i, t in enumerate(lens):
        for got, x in zip((rk, rv), rows[i]):
            np.testing.assert_array_equal(got[i, 300 - t:].cpu().numpy(), R.held(x).astype(np.float32))
    heads = lambda x: R.held(x).reshape(-1, n_kv, hd).transpose(1, 0, 2)
    w = torch.zeros(2, n_kv, 5 * 64, device="cuda")
    for n_q in (1, 40):
        q = torch.from_numpy(rng.standard_normal((2, n_q, n_heads * hd)).astype(np.float32)).cuda()
        out = torch.empty_like(q)
        ops.kv4_attn(out, q, c, n_heads, weights_in=w, weights_out=w)
        for i in range(2):
            want, _, top = R.attend(q[i].cpu().numpy(), heads(rows[i][0]), heads(rows[i][1]), n_q)
            assert np.linalg.norm(out[i].cpu().numpy() - want) <= 16 * 2.0 ** -24 * max(1.0, top) * np.linalg.norm(want)
    before = w.cpu().numpy()
    far = ops.Kv4Cache(pool, torch.tensor([[n_pages - 20, 20], [n_pages - 21, 21]], dtype=torch.int32, device="cuda"),
                       torch.zeros(2, dtype=torch.int32, device="cuda"), n_kv, hd)
    wd, kept = torch.empty(2, n_kv, 128, device="cuda"), torch.empty(2, n_kv, 100, dtype=torch.int32, device="cuda")
    for dst, wt in ((far, wd), (c, w)):
        ops.kv4_evict(c, dst, w, wt, 100, 2, 30, kept)
        gk, gv = (torch.empty(2, 100, n_kv * hd, device="cuda") for _ in range(2))
        ops.kv4_read(dst, gk, gv)
        for i, t in enumerate(lens):
            for h in range(n_kv):
                f = R.keep(before[i, h], t, 100, 2, 30)
                for got, x in zip((gk, gv), rows[i]):
                    np.testing.assert_array_equal(got[i, :, h * hd:(h + 1) * hd].cpu().numpy(), R.held(x).astype(np.float32)[f][:, h * hd:(h + 1) * hd])
    assert device_errors() == 0


def captured(f):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f()
    return g


@pytest.mark.parametrize("mp,in_place", [(6, False), (6, True), (300, False), (300, True)])
def test_captured_evictions_follow_lens_and_weights(ops, mp, in_place):
    """An eviction captured once (rows of one block, and long ones), replayed while lengths, weights and pages change."""
    rng = np.random.default_rng(91)
    n_kv, hd, budget = 2, 64, 150
    m = Made(ops, rng, [mp * 64, 200], n_kv, hd, max_pages=mp)
    w = torch.zeros(2, n_kv, mp * 64, device="cuda")
    kept = torch.empty(2, n_kv, budget, dtype=torch.int32, device="cuda")
    dpool, dlens, dw = torch.zeros(8, n_kv * 72 * hd, dtype=torch.uint8, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, n_kv, 256, device="cuda")
    to = m.cache if in_place else ops.Kv4Cache(dpool, torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), dlens, n_kv, hd)
    tw = w if in_place else dw
    pool0 = m.dpool.clone()
    g = captured(lambda: ops.kv4_evict(m.cache, to, w, tw, budget, 3, 40, kept))
    inputs = [([mp * 64, 200], 1), ([151, 0], 2), ([mp * 64 - 65, 150], 3), ([1, 383], 4)]
    seen = {}
    for mode in ("graph", "eager"):
        for lens, seed in inputs:
            m.dpool.copy_(pool0)
            dpool.zero_(); dw.zero_(); dlens.zero_()
            m.dlens.copy_(torch.tensor(lens, dtype=torch.int32))
            w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)))
            g.replay() if mode == "graph" else ops.kv4_evict(m.cache, to, w, tw, budget, 3, 40, kept)
            torch.cuda.synchronize()
            got = [x.clone() for x in (kept, to.lens, tw, to.pool)]
            if mode == "graph":
                seen[seed] = got
            else:
                assert all(torch.equal(a, b) for a, b in zip(seen[seed], got)), lens
                assert got[1].tolist() == [min(t, budget) for t in lens]
    assert device_errors() == 0


@pytest.mark.parametrize("n_heads,n_q", [(8, 1), (8, 6), (8, 30)])
def test_two_streams_and_two_graphs_at_once(ops, n_heads, n_q):
    """Calls with weights on two caches on two streams, and two captured ones replayed side by side, give what they give
    one after the other."""
    rng = np.random.default_rng(92)
    n_kv, hd = 2, 128
    made = [Made(ops, rng, lens, n_kv, hd) for lens in ([3000, 70], [500, 2900])]
    qs = [torch.randn(2, n_q, n_heads * hd, device="cuda") for _ in made]
    ws = [torch.rand(2, n_kv, m.table.shape[1] * 64, device="cuda") for m in made]
    outs, wos = [torch.empty_like(q) for q in qs], [torch.empty_like(w) for w in ws]
    call = lambda i: ops.kv4_attn(outs[i], qs[i], made[i].cache, n_heads, weights_in=ws[i], weights_out=wos[i])
    want = []
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        want.append((outs[i].clone(), wos[i].clone()))
    streams = [torch.cuda.Stream() for _ in made]
    graphs = [captured(lambda i=i: call(i)) for i in range(2)]
    for how in ("calls", "graphs"):
        for x in outs + wos:
            x.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    call(i) if how == "calls" else graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i][0]) and torch.equal(wos[i], want[i][1]), how
    assert device_errors() == 0
