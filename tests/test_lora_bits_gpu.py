"""Low-rank adapters to the last bit: sums of a single product, which fp32 holds, and numbers at the lower end of fp32's
range."""
import numpy as np
import pytest
import torch

from libinferbit_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def one_hot(B, N, M, R, kind, seed, bits):
    """Adapters with a single rank that is not zero, rows with a single number: of `bits` bits, a's numbers of
    24 - bits, b's and the scales powers of two.  (out, the result, which fp32 holds)."""
    rng = np.random.default_rng(seed)
    n = min(R, 16)
    rank = np.array([k * R // n + k % max(1, R // n) for k in range(n)])
    sign = lambda *s: rng.integers(0, 2, s) * 2.0 - 1

    def odd(width, *s):                                  # numbers of [1, 2) that take all of their bits
        return 1.0 + (rng.integers(0, 1 << (width - 1), s) | 1) * 2.0 ** (1 - width) if width > 1 else np.ones(s)

    a = np.zeros((n, R, N))
    a[np.arange(n), rank] = odd(24 - bits, n, N) * 2.0 ** rng.integers(-3, 4, (n, N)) * sign(n, N)
    b = 2.0 ** rng.integers(-3, 4, (n, M, R)) * sign(n, M, R)
    scales = 2.0 ** rng.integers(-2, 3, n)
    ids = rng.integers(0, n, B)
    row = np.arange(B)
    col = (row * 64 + row * 37 % 64) % N                 # every step of 64 columns, every place in one
    x = np.zeros((B, N))
    x[row, col] = odd(bits, B) * 2.0 ** rng.integers(-10, 10, B) * sign(B)
    t = a[ids, rank[ids], col] * x[row, col] * scales[ids]
    want = t[:, None] * b[ids, :, rank[ids]]
    gpu = lambda v, dt: torch.from_numpy(v).to(dt).cuda()
    out = torch.full((B, M), 7.0, device="cuda")
    ops.lora(out, gpu(x, torch.float32), gpu(a, TYPES[kind]), gpu(b, TYPES[kind]), gpu(ids, torch.int32), scales=gpu(scales, torch.float32))
    return out.cpu().numpy().astype(np.float64), want


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("R", [16, 32, 64, 100, 256])
@pytest.mark.parametrize("B,N,M", [(64, 2048, 260), (64, 300, 261), (200, 48, 260), (200, 45, 261), (200, 2048, 261), (150, 2051, 260),
                                   (200, 4160, 260), (200, 4163, 261), (600, 4160, 64)])
def test_all_bits_of_a_single_product(B, N, M, R, kind):
    """x of 24 bits by powers of two, of 13 by fp16's 11, of 16 by bf16's 8: a product has 24 bits at most, and so has any
    sum of its parts, which lie in the same 24 places."""
    for seed, bits in enumerate((24, 13, 16) if kind == "fp16" else (24, 16)):
        out, want = one_hot(B, N, M, R, kind, 10 * R + seed, bits)
        np.testing.assert_array_equal(out, want, err_msg=f"bits {bits}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B", [64, 65, 200])
def test_small_numbers(B, kind):
    """One number a row, 2^-149 to 2^-100, and A x as small: exact up to 64 rows; from 65 on what lies below 2^-133 is cut
    off, once from x and once from A x (whose last places here are 2^-145 at most, so that fp32 holds it)."""
    rng = np.random.default_rng(B)
    N, M = 128, 8
    for low, ea, eb in ((-149, 0, 0), (-130, 0, 3), (-116, -6, 10)):
        x = np.zeros((B, N), np.float32)
        x[np.arange(B), np.arange(B) * 29 % N] = np.ldexp(1 + (rng.integers(0, 1 << 23, B) | 1) * 2.0 ** -23, rng.integers(low, -99, B)) * rng.choice([-1, 1], B)
        a, b = np.full((1, 16, N), 0.0), np.full((1, M, 16), 2.0 ** eb)
        a[0, 5] = 2.0 ** ea
        out = torch.empty(B, M, device="cuda")
        ops.lora(out, torch.from_numpy(x).cuda(), torch.from_numpy(a).cuda().to(TYPES[kind]), torch.from_numpy(b).cuda().to(TYPES[kind]),
                 torch.zeros(B, dtype=torch.int32, device="cuda"))
        out = out.cpu().numpy().astype(np.float64)
        t = x.astype(np.float64).sum(1) * 2.0 ** ea
        want = (t * 2.0 ** eb)[:, None]
        far = 0 if B <= 64 else 2.0 ** -133 * (2.0 ** ea + 1) * 2.0 ** eb
        assert (np.abs(out - want) <= far).all(), (low, np.abs(out - want).max() / 2.0 ** eb)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B", [64, 65])
def test_sums_beyond_the_range(B, kind):
    """An infinite sum stays one up to 64 rows and is no number from 65 on, where it may be; a finite one beside it stays."""
    x = torch.ones(B, 32)
    x[1, 3], x[1, 4], x[2, 7], x[3, 3] = 3e38, 3e38, float("-inf"), 3e38
    out = torch.empty(B, 4, device="cuda")
    ops.lora(out, x.cuda(), torch.ones(1, 8, 32, device="cuda", dtype=TYPES[kind]) / 8, torch.ones(1, 4, 8, device="cuda", dtype=TYPES[kind]) * 4,
             torch.zeros(B, dtype=torch.int32, device="cuda"))
    out = out.cpu()
    assert not torch.isfinite(out[1:3]).any()
    if B <= 64:
        assert (out[1] == float("inf")).all() and (out[2] == float("-inf")).all()
    assert not torch.isfinite(out[3]).any()              # eight times 3e38 / 8 + 31 / 8, by 4: beyond the range as well
    assert (out[4:] == 128).all() and (out[0] == 128).all()
