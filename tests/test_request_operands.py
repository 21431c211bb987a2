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


def test_rows_that_take_turns():
    """Columns of one wide array: rows of out between those of x and base, but not on them."""
    S, at = 16384, lambda f: (3 << 40) + 4 * f
    for x, base in ((4096, 8192), (8192, 4096), (-4096, -8192), (12288, -4096), (4096 + 3 * S, None), (4096 - 2 * S, 8192 - S)):
        assert lora(5, x=at(x), base=None if base is None else at(base), os=S, xs=S, bs=S) == -3, (x, base)
    for x in (0, 1, -1, 4095, -4095, 12289, -12289, S - 4095, 2 * S - 4095, -S + 4095, -2 * S + 1):
        assert lora(5, x=at(x), os=S, xs=S) == -5, x
        assert lora(5, base=at(x), os=S, bs=S) == (-3 if x == 0 else -5), x
    # single rows, and rows that lie unequally far apart, by all that lies between their first and last number
    assert lora(1, x=at(4096), os=S, xs=S) == lora(1, x=at(-4096)) == -3
    assert lora(1, x=at(4095), os=S, xs=S) == -5
    assert lora(2, x=at(4096), os=S, xs=S + 4096) == -5
    assert lora(2, x=at(S + 4096), os=S, xs=S + 4096) == -3


def test_overlap_of_rows_by_trying_all():
    """Whether a call is refused, against the rows' numbers themselves."""
    for s in (8, 11):
        mine = {i * s + j for i in range(66) for j in range(5)}
        for off in range(-3 * s, 3 * s + 1):
            others = {off + i * s + j for i in range(66) for j in range(3)}
            assert lora(66, N=3, M=5, x=(3 << 40) + 4 * off, os=s, xs=s) == (-5 if mine & others else -3), (s, off)


def test_large_ranks_take_two_launches():
    """Both products of few rows in one launch (which needs no workspace) work ranks out eight after eight: up to 32."""
    need = lambda rank, N: _lib.lib().ibh_lora_workspace_bytes(C.byref(_lib.LoraDesc(1 << 40, 2 << 40, None, None, 4, rank, N, 1024, 0)), 32)
    assert need(8, 8192) == need(16, 4096) == need(32, 2048) == need(32, 64) == 0
    assert need(33, 64) == 32 * 40 * 4 and need(64, 1024) == 32 * 64 * 4 and need(256, 256) == 32 * 256 * 4
    assert need(32, 2049) == 32 * 32 * 4
