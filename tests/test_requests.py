"""The operators around a batch's projections without a GPU: the oracle against closed forms, and the calls that are
refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from libinferbit_amd import _lib, ops
from oracle import requests as R


def refused(name, *args, code=-5):
    rc = getattr(_lib.lib(), name)(*args)
    msg = _lib.lib().ibh_last_error()
    assert rc == code and msg, (rc, msg)
    return msg.decode()


def test_oracle_codes_are_the_nearest():
    rng = np.random.default_rng(0)
    p = (rng.standard_normal(300) * np.exp(rng.standard_normal(300))).astype(np.float32)
    q, s = R.codes(p, 0.7)
    steps = p / (np.repeat(s, R.GROUP)[:300] / 0.7)
    assert (np.abs(steps - q) <= 0.5 + 1e-12).all() and np.abs(q).max() == 127
    # halves go away from zero: with 127 as the largest the steps are the numbers themselves
    q, s = R.codes(np.array([127, 0.5, -0.5, 1.5, 2.5, -2.5, 0.49999997, 126.5], np.float32), 1.0)
    assert q.tolist() == [127, 1, -1, 2, 3, -3, 0, 127] and s[0] == 1
    q, s = R.codes(np.zeros(130, np.float32), 1.0)
    assert not q.any() and (s == 1e-10).all()


def test_oracle_norm_of_equal_elements():
    h, p, r = R.norm(np.full((2, 64), 3.0), np.full((2, 64), 1.0), np.full(64, 0.5), 0.0)
    assert (h == 4).all() and (p == 2).all() and (r == 0.25).all()


def test_oracle_logprobs_of_equal_logits():
    lp, ent, ids, top, lse = R.logprobs(np.zeros((1, 8)), [[3, 8, -1]], 3)
    assert lp[0, 0] == -np.log(8) and np.isnan(lp[0, 1:]).all() and ids.tolist() == [[0, 1, 2]]
    np.testing.assert_allclose(ent, np.log(8))


N, B = 256, 3
GAP = 1 << 20                      # addresses this far apart hold none of the test's operands twice


def norm_args(**c):
    d = dict(y=GAP, q=2 * GAP, s=3 * GAP, h=4 * GAP, x=5 * GAP, delta=6 * GAP, weight=7 * GAP, eps=1e-5, N=N, B=B, xs=N,
             ds=N, stream=None)
    assert not set(c) - set(d)
    return tuple({**d, **c}.values())


@pytest.mark.parametrize("bad", [dict(x=0), dict(weight=0), dict(y=0, q=0, s=0), dict(q=0), dict(s=0), dict(N=0),
                                 dict(N=-1), dict(N=(1 << 30) + 1), dict(B=-1), dict(xs=N - 1), dict(ds=N - 1),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(B=1 << 22, N=1, xs=1, ds=1, x=1 << 40, delta=1 << 41, y=1 << 42, q=1 << 43, s=1 << 44, h=1 << 45)])
def test_norm_refuses(bad):
    refused("ibh_add_rmsnorm", *norm_args(**bad))


@pytest.mark.parametrize("bad", [dict(h=GAP), dict(y=5 * GAP + 4), dict(y=5 * GAP, xs=N + 1), dict(h=6 * GAP, ds=N + 4),
                                 dict(y=7 * GAP), dict(h=7 * GAP), dict(q=5 * GAP), dict(s=5 * GAP), dict(q=3 * GAP + 4),
                                 dict(q=6 * GAP), dict(s=7 * GAP), dict(q=GAP + 4 * N * B - 1), dict(h=6 * GAP - 4)])
def test_norm_refuses_overlaps(bad):
    assert "overlaps" in refused("ibh_add_rmsnorm", *norm_args(**bad))


def lora_desc(**c):
    d = dict(a=GAP, b=2 * GAP, scales=3 * GAP, ranks=4 * GAP, n=4, rank=16, N=N, M=128, kind=0)
    assert not set(c) - set(d)
    return _lib.LoraDesc(*{**d, **c}.values())


def lora_args(desc=None, **c):
    d = dict(out=5 * GAP, base=6 * GAP, x=7 * GAP, ids=8 * GAP, B=B, os=128, bs=128, xs=N, ws=9 * GAP, size=GAP, stream=None)
    assert not set(c) - set(d)
    return (C.byref(desc or lora_desc()), *{**d, **c}.values())


@pytest.mark.parametrize("bad", [dict(a=0), dict(b=0), dict(n=0), dict(n=-1), dict(rank=0), dict(rank=257), dict(N=0),
                                 dict(M=0), dict(N=(1 << 20) + 1), dict(M=(1 << 20) + 1), dict(kind=2), dict(kind=-1)])
def test_lora_refuses_adapters(bad):
    refused("ibh_lora", *lora_args(lora_desc(**bad)))
    assert _lib.lib().ibh_lora_workspace_bytes(C.byref(lora_desc(**bad)), 1) == 0


@pytest.mark.parametrize("bad", [dict(out=0), dict(x=0), dict(ids=0), dict(B=-1), dict(os=127), dict(bs=127), dict(xs=N - 1)])
def test_lora_refuses(bad):
    refused("ibh_lora", *lora_args(**bad))


@pytest.mark.parametrize("bad", [dict(out=7 * GAP), dict(out=6 * GAP + 4), dict(out=6 * GAP, os=129), dict(out=8 * GAP),
                                 dict(out=GAP), dict(out=2 * GAP), dict(out=3 * GAP), dict(out=4 * GAP)])
def test_lora_refuses_overlaps(bad):
    assert "overlaps" in refused("ibh_lora", *lora_args(**bad))


def test_lora_refuses_workspaces():
    big = lora_desc(rank=64, N=4096)
    need = _lib.lib().ibh_lora_workspace_bytes(C.byref(big), B)
    assert need > 0
    refused("ibh_lora", *lora_args(big, xs=4096, size=need - 1), code=-3)
    refused("ibh_lora", *lora_args(big, xs=4096, ws=9 * GAP + 4), code=-3)
    assert _lib.lib().ibh_lora_workspace_bytes(C.byref(big), 0) == 0
    refused("ibh_lora", None, *lora_args()[1:])


def test_more_rows_than_a_launch_takes_are_refused():
    far = [k << 40 for k in range(1, 9)]
    d = _lib.LoraDesc(far[0], far[1], far[2], far[3], 4, 16, 64, 64, 0)
    assert "launch" in refused("ibh_lora", C.byref(d), far[4], None, far[5], far[6], 1 << 22, 64, 0, 64, far[7], 1 << 40, None)
    assert "launch" in refused("ibh_logprobs", far[0], far[1], None, None, far[2], far[3], 100, 1 << 24, 100, 1, 0, None, 0, None)


def log_args(**c):
    d = dict(out=GAP, entropy=2 * GAP, ids=3 * GAP, top=4 * GAP, z=5 * GAP, tokens=6 * GAP, V=1000, B=B, stride=1000, n=2, k=5,
             ws=7 * GAP, size=GAP, stream=None)
    assert not set(c) - set(d)
    return tuple({**d, **c}.values())


@pytest.mark.parametrize("bad", [dict(z=0), dict(out=0), dict(tokens=0), dict(ids=0), dict(top=0), dict(V=0), dict(V=-1),
                                 dict(V=(1 << 30) + 1), dict(B=-1), dict(stride=999), dict(n=-1), dict(k=-1), dict(k=65),
                                 dict(n=0, k=0, entropy=0)])
def test_logprobs_refuses(bad):
    refused("ibh_logprobs", *log_args(**bad))


@pytest.mark.parametrize("bad", [dict(out=5 * GAP), dict(entropy=GAP + 4), dict(ids=4 * GAP + 8), dict(top=6 * GAP),
                                 dict(entropy=5 * GAP + 4 * 2999), dict(out=6 * GAP)])
def test_logprobs_refuses_overlaps(bad):
    assert "overlaps" in refused("ibh_logprobs", *log_args(**bad))


def test_no_rows_are_nothing_to_do():
    L = _lib.lib()
    assert L.ibh_add_rmsnorm(*norm_args(B=0, x=0, y=0)) == 0
    assert L.ibh_lora(*lora_args(B=0, out=0, x=0, ids=0)) == 0
    assert L.ibh_logprobs(*log_args(B=0, z=0)) == 0


def test_python_wrappers_refuse():
    x = torch.zeros(2, 128)
    for call in (lambda: ops.add_rmsnorm(x, x, x[0], 1e-5), lambda: ops.add_rmsnorm(x, x[0], x[0], 1e-5),
                 lambda: ops.logprobs(x[:, 0], x, x[:, 0].int()), lambda: ops.logprobs(None, x[0], None),
                 lambda: ops.lora(x, x, x, x, x[:, 0].int()),
                 lambda: ops.lora(x, x, x.half().view(2, 1, 128), x.half().view(2, 128, 1), x[:, 0].int())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.lora(x, x, x.view(2, 1, 128), x.view(2, 128, 1), x[:, 0].int())
