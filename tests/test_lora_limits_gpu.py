"""Low-rank adapters at the limits of their sizes: as many outputs as a call takes."""
import pytest
import torch

from libinferbit_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B", [1, 3])
def test_the_most_outputs_at_the_largest_rank(B, kind):
    """2^20 outputs of rank 256, which takes the smallest blocks of outputs: 65536 of them."""
    N, M, R = 32, 1 << 20, 256
    g = torch.Generator("cuda").manual_seed(B)
    a = (torch.randn(1, R, N, generator=g, device="cuda") / 6).to(TYPES[kind])
    b = (torch.randn(1, M, R, generator=g, device="cuda") / 16).to(TYPES[kind])
    x, ids = torch.randn(B, N, generator=g, device="cuda"), torch.tensor([0, -1, 0][:B], dtype=torch.int32, device="cuda")
    out = torch.full((B, M), 7.0, device="cuda")
    ops.lora(out, x, a, b, ids)
    for i in range(B):
        if ids[i] < 0:
            assert (out[i] == 0).all()
            continue
        t = (a[0].double() * x[i].double()).sum(1)
        for m in range(0, M, M // 16):
            part = b[0, m:m + M // 16].double()
            want, size = (part * t).sum(1), (part.abs() * (a[0].double() * x[i].double()).abs().sum(1)).sum(1)
            # 32 products and 256: chains of fewer than 300 additions, half a step each
            assert ((out[i, m:m + M // 16] - want).abs() <= 300 * 2.0 ** -24 * size).all(), m
