"""The paged 4-bit KV cache without a GPU: the page layout, and the calls that
are refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from libinferbit_amd import _lib, ops
from oracle import kv4 as R


@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_layout_covers_every_byte_once(hd):
    (k, ks, kp), (v, vs, vp) = R.places(hd)
    seen = np.zeros((72 * hd, 2), int)
    for at, shift in ((k, ks), (v, vs)):
        np.add.at(seen, (at, shift // 4), 1)
    for pair in (kp, vp):
        for half in (0, 1):
            b = 2 * np.unique(pair + half)
            for o in (0, 1):
                seen[b + o] += 1
    assert (seen == 1).all()


def test_oracle_store_and_load_agree():
    rng = np.random.default_rng(0)
    n_kv, hd, n = 2, 128, 100
    pool = rng.integers(0, 256, (4, n_kv * 72 * hd), dtype=np.uint8)
    k, v = rng.standard_normal((2, n, n_kv * hd)).astype(np.float32)
    R.store(pool, [3, 1], n_kv, hd, k, v, 0)
    K, V = R.load(pool, [3, 1], n_kv, hd, n)
    np.testing.assert_array_equal(K.transpose(1, 0, 2).reshape(n, -1), R.held(k))
    np.testing.assert_array_equal(V.transpose(1, 0, 2).reshape(n, -1), R.held(v))
    # a code is at most half a step off, the ends at most what fp16 takes from scale and mid
    c, s, m = R.quantise(k)
    step = np.repeat(s.astype(np.float64), 64, -1).reshape(k.shape)
    assert (np.abs(R.held(k) - k) <= step * (0.5 + 16 * 2 ** -11) + np.repeat(np.abs(m.astype(np.float64)), 64, -1).reshape(k.shape) * 2 ** -11).all()


GOOD = dict(pool=4096, table=4096, lens=4096, n_pages=4, n_seq=2, max_pages=2, n_kv=2, head_dim=64)


def desc(**change):
    d = {**GOOD, **change}
    return _lib.Kv4Desc(*(d[f] for f, _ in _lib.Kv4Desc._fields_))


def refused(name, *args, code=-5):
    rc = getattr(_lib.lib(), name)(*args)
    msg = _lib.lib().ibh_last_error()
    assert rc == code and msg, (rc, msg)
    return msg.decode()


BAD_CACHES = [dict(pool=0), dict(pool=4104), dict(table=0), dict(lens=0), dict(n_pages=0), dict(n_seq=0), dict(n_seq=-1),
              dict(max_pages=0), dict(max_pages=1 << 25), dict(n_kv=0), dict(head_dim=0), dict(head_dim=96),
              dict(head_dim=32), dict(head_dim=320), dict(head_dim=-64)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(bad):
    c = C.byref(desc(**bad))
    refused("ibh_kv4_append", c, 4096, 4096, 1, 128, None)
    refused("ibh_kv4_read", c, 4096, 4096, 1, 128, None)
    refused("ibh_kv4_attn", c, 4096, 4096, 4, 1, 256, None, None, 4096, 1 << 30, None)
    refused("ibh_kv4_evict", c, C.byref(desc(table=8192, lens=8192)), 4096, 8192, 64, 0, 0, 4096, None, 0, None)
    refused("ibh_kv4_evict", C.byref(desc(table=8192, lens=8192)), c, 4096, 8192, 64, 0, 0, 4096, None, 0, None)


def test_bad_arguments_are_refused():
    c = C.byref(desc())
    for k, v, n, stride in ((0, 4096, 1, 128), (4096, 0, 1, 128), (4096, 4096, 0, 128), (4096, 4096, 1, 127)):
        refused("ibh_kv4_append", c, k, v, n, stride, None)
        refused("ibh_kv4_read", c, k, v, n, stride, None)
    attn = lambda out=4096, q=4096, heads=4, n_q=1, stride=256, wi=None, wo=None, ws=4096, size=1 << 30: (
        c, out, q, heads, n_q, stride, wi, wo, ws, size, None)
    for bad in (dict(out=0), dict(q=0), dict(heads=0), dict(heads=3), dict(heads=-2), dict(n_q=0), dict(stride=255),
                dict(wi=4096), dict(wo=4096)):
        refused("ibh_kv4_attn", *attn(**bad))
    c = C.byref(desc(max_pages=64))                              # long enough for splits, so for a workspace
    refused("ibh_kv4_attn", *attn(size=1), code=-3)
    refused("ibh_kv4_attn", *attn(ws=4100), code=-3)
    c = C.byref(desc())
    to = C.byref(desc(table=8192, lens=8192))
    evict = lambda src=c, dst=to, ws=4096, wd=8192, budget=64, sink=0, recent=0, kept=4096: (
        src, dst, ws, wd, budget, sink, recent, kept, None, 0, None)
    for bad in (dict(ws=0), dict(wd=0), dict(kept=0), dict(budget=0), dict(budget=129), dict(sink=-1), dict(recent=-1),
                dict(sink=65), dict(sink=33, recent=32), dict(dst=C.byref(desc(table=8192, lens=8192, n_kv=4))),
                dict(dst=C.byref(desc(table=8192, lens=8192, head_dim=128))),
                dict(dst=C.byref(desc(table=8192, lens=8192, n_seq=3))), dict(wd=4096), dict(dst=C.byref(desc(table=8192))),
                dict(dst=c), dict(dst=C.byref(desc(pool=8192)), wd=4096),
                dict(dst=C.byref(desc(max_pages=1)), wd=4096), dict(dst=C.byref(desc(lens=8192)), wd=4096)):
        refused("ibh_kv4_evict", *evict(**bad))


def test_more_work_than_a_launch_takes_is_refused():
    c = C.byref(desc(n_seq=1 << 20, n_kv=64, max_pages=1 << 10))
    assert "launch" in refused("ibh_kv4_append", c, 4096, 4096, 1, 64 * 64, None)
    assert "launch" in refused("ibh_kv4_read", c, 4096, 4096, 1, 64 * 64, None)
    assert "launch" in refused("ibh_kv4_attn", c, 4096, 4096, 64, 1, 4096, None, None, 4096, (1 << 63) - 1, None)
    to = C.byref(desc(n_seq=1 << 20, n_kv=64, max_pages=1 << 10, table=8192, lens=8192))
    assert "launch" in refused("ibh_kv4_evict", c, to, 4096, 8192, 64, 0, 0, 4096, 4096, (1 << 63) - 1, None)
    refused("ibh_kv4_attn", C.byref(desc()), 4096, 4096, 1 << 20, 1 << 20, (1 << 31) - 1, None, None, 4096, 1 << 62, None)


def test_sizes():
    L = _lib.lib()
    assert L.ibh_kv4_page_bytes(8, 128) == 8 * 9216
    for kv, hd in ((0, 128), (8, 96), (8, 0), (-1, 64), (8, 320)):
        assert L.ibh_kv4_page_bytes(kv, hd) == 0
    assert L.ibh_kv4_attn_workspace_bytes(C.byref(desc(max_pages=64)), 4, 1, 0) > 0
    assert L.ibh_kv4_evict_workspace_bytes(C.byref(desc())) == 0
    assert L.ibh_kv4_evict_workspace_bytes(C.byref(desc(max_pages=257))) > 0
    long = desc(max_pages=257), desc(max_pages=257, table=8192, lens=8192)
    refused("ibh_kv4_evict", C.byref(long[0]), C.byref(long[1]), 4096, 8192, 64, 0, 0, 4096, 4096, 1, None, code=-3)
    refused("ibh_kv4_evict", C.byref(long[0]), C.byref(long[1]), 4096, 8192, 64, 0, 0, 4096, 4100, 1 << 30, None, code=-3)
    assert L.ibh_kv4_attn_workspace_bytes(C.byref(desc()), 0, 1, 1) == 0


def test_python_wrappers_refuse():
    pool = torch.zeros(4, 2 * 72 * 64, dtype=torch.uint8)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.Kv4Cache(pool, table, lens, 2, 64)                   # not on a GPU
    with pytest.raises(ValueError):
        ops.Kv4Cache(pool, table[0], lens, 2, 64)
    with pytest.raises(TypeError):
        ops.Kv4Cache(pool, table.long(), lens, 2, 64)
    with pytest.raises(TypeError):
        ops.Kv4Cache(pool.float(), table, lens, 2, 64)
    with pytest.raises(ValueError):
        ops.Kv4Cache(pool[:, :-1], table, lens, 2, 64)           # not whole pages
