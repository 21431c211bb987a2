"""Low-rank adapters at the limits of their sizes and places: as many outputs as a call takes, rows that take turns."""
import numpy as np
import pytest
import torch

from libinferbit_amd import ops
from oracle import requests as R

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


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B", [1, 9, 64, 90, 300])
@pytest.mark.parametrize("N,M,rank", [(64, 96, 8), (61, 77, 5), (2048, 256, 64), (8, 4, 16)])
@pytest.mark.parametrize("order", ["out x base", "base out x", "x base out"])
def test_columns_of_one_array(B, N, M, rank, order, kind):
    """out, x and base beside each other in each row; what is not out's stays as it is."""
    g = torch.Generator().manual_seed(B + N)
    a, b = (torch.randn(3, rank, N, generator=g) / N ** 0.5).to(TYPES[kind]), (torch.randn(3, M, rank, generator=g) / rank ** 0.5).to(TYPES[kind])
    ids = torch.randint(-1, 3, (B,), generator=g, dtype=torch.int32)
    wide, at, place = torch.randn(B, N + 2 * M + 5, generator=g), 0, {}
    for name in order.split():
        place[name] = slice(at, at + (N if name == "x" else M))
        at = place[name].stop + 1
    on = wide.cuda()
    ops.lora(on[:, place["out"]], on[:, place["x"]], a.cuda(), b.cuda(), ids.cuda(), base=on[:, place["base"]])
    want, size = R.lora(wide[:, place["base"]].numpy(), wide[:, place["x"]].numpy(), a.float().numpy(), b.float().numpy(), ids.tolist())
    out = on[:, place["out"]].cpu().numpy()
    # chains of at most (N + rank) / 32 + 128 additions, half a step each, and the base's
    assert (np.abs(out - want) <= 2.0 ** -24 * (((N + rank) / 32 + 132) * size + 2 * np.abs(want))).all()
    rest = torch.ones(wide.shape[1], dtype=torch.bool)
    rest[place["out"]] = False
    assert torch.equal(on.cpu()[:, rest], wide[:, rest])
