"""Operands on a GPU that is not the current one, without a GPU: stand-ins for tensors, and no call that gets as far as the
library."""
import contextlib

import pytest
import torch

from libinferbit_amd import _lib, ops, session


class Tensor:
    """As much of a tensor of GPU `index` as the checks look at."""
    is_cuda, dtype, shape = True, torch.float32, torch.Size([4, 128])

    def __init__(self, index):
        self.index, self.device = index, f"cuda:{index}"

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 40

    def numel(self):
        return 512


class Library:
    """Takes down what is called."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def on_gpu_0(monkeypatch):
    library = Library()
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(ops, "_stream", lambda: 100)
    monkeypatch.setattr(ops, "lib", lambda: library)
    monkeypatch.setattr(session, "lib", lambda: library)
    return library


def bare(cls, **fields):
    o = cls.__new__(cls)
    for k, v in fields.items():
        setattr(o, k, v)
    return o


# each call with the operands that it takes
CALLS = {
    "parallel_matmul": (4, lambda t: ops.parallel_matmul(*t, 4, 128, 4)),
    "quantize_input_int8_g128": (3, lambda t: ops.quantize_input_int8_g128(*t, 128)),
    "parallel_matmul_w4a8": (5, lambda t: ops.parallel_matmul_w4a8(*t, 4, 128)),
    "matmul_w4a8_x": (6, lambda t: ops.matmul_w4a8_x(*t[:4], 4, 128, *t[4:])),
    "matmul_w4a8_batch": (5, lambda t: ops.matmul_w4a8_batch(*t, 4, 128, 1, 4)),
    "matmul_int8_batch": (4, lambda t: ops.matmul_int8_batch(*t, 4, 128, 1, 4)),
    "gemm_int8": (5, lambda t: ops.gemm_int8(*t[:4], 4, 128, 1, 4, ws=t[4])),
    "kv_cache_write": (6, lambda t: ops.kv_cache_write(*t[:4], 0, *t[4:], 1, 64, 8)),
    "attn_decode": (6, lambda t: ops.attn_decode(*t, 0, 1, 1, 64, 8)),
    "PqDeviceTensor.matmul": (3, lambda t: bare(ops.PqDeviceTensor, s=ops.PqTensor(), ws=t[2]).matmul(*t[:2])),
    "PqDeviceTensor.matmul_policy": (3, lambda t: bare(ops.PqDeviceTensor, s=ops.PqTensor(), ws=t[2]).matmul_policy(*t[:2], 1)),
    "PqDeviceTensor.matmul_q8lut": (3, lambda t: bare(ops.PqDeviceTensor, s=ops.PqTensor(), ws=t[2]).matmul_q8lut(*t[:2])),
    "PqDeviceTensor.matmul_streaming": (3, lambda t: bare(ops.PqDeviceTensor, s=ops.PqTensor(), ws=t[2]).matmul_streaming(*t[:2])),
    "Int4gDeviceTensor.matmul": (3, lambda t: bare(ops.Int4gDeviceTensor, s=ops.Int4gTensor(), keep=t[2:]).matmul(*t[:2])),
    "Int4gDeviceTensor.matmul_batched": (3, lambda t: bare(ops.Int4gDeviceTensor, s=ops.Int4gTensor(), keep=t[2:]).matmul_batched(*t[:2])),
    "session.matmul": (2, lambda t: bare(session.PqSession, _h=None).matmul("w", *t)),
}


@pytest.mark.parametrize("name", CALLS)
def test_operands_of_another_gpu_are_refused(name, on_gpu_0):
    """A launch on the current GPU with another's addresses would fault there."""
    n, call = CALLS[name]
    call([Tensor(0)] * n)
    assert len(on_gpu_0.calls) == 1
    for i in range(n):
        with pytest.raises(ValueError, match="cuda:1"):
            call([Tensor(int(k == i)) for k in range(n)])
    assert len(on_gpu_0.calls) == 1


def test_calls_that_follow_their_operands(on_gpu_0, monkeypatch):
    """The norm on GPU 1 while GPU 0 is the current one, and on the current one; operands of both are refused."""
    went = []

    @contextlib.contextmanager
    def device(i):
        went.append(i)
        yield

    monkeypatch.setattr(torch.cuda, "device", device)
    weight = {i: Tensor(i) for i in range(2)}
    for w in weight.values():
        w.shape = torch.Size([128])
    for i in range(2):
        ops.add_rmsnorm(Tensor(i), Tensor(i), weight[i], 1e-5)
    assert went == [1] and [(name, a[-1]) for name, a in on_gpu_0.calls] == [("ibh_add_rmsnorm", 100), ("ibh_add_rmsnorm", 101)]
    for y, x, w in ((0, 1, 1), (1, 0, 0), (0, 0, 1)):
        with pytest.raises(ValueError, match="cuda:"):
            ops.add_rmsnorm(Tensor(y), Tensor(x), weight[w], 1e-5)
