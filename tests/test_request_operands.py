"""Operands at the edge of what the operators around a batch's projections take, without a GPU: no call gets as far as a
launch."""
import ctypes as C

from libinferbit_amd import _lib


def lora(B, n=4, rank=64, N=4096, M=4096, a=1 << 40, b=2 << 40, out=3 << 40, base=None, x=5 << 40, ids=6 << 40, os=4096, bs=4096, xs=4096):
    """The return code of a call with a workspace of 8 bytes, which is looked at last and found too small (-3) in every call
    that gets there."""
    d = _lib.LoraDesc(a, b, None, None, n, rank, N, M, 0)
    return _lib.lib().ibh_lora(C.byref(d), out, base, x, ids, B, os, bs, xs, 7 << 40, 8, None)


def test_no_rows_need_no_adapters():
    """A server without adapters yet, or a batch that has run out: nothing to do."""
    assert lora(1) == -3
    assert lora(0) == 0
    assert lora(0, n=0, a=None, b=None, out=None, x=None, ids=None) == 0
    assert lora(1, n=0) == -5
