"""Rows whose blocks hold entries far smaller than their largest, which meets a weight of zero.

What a product takes of a row: entries from 2^-13 of their block's largest on as they are; smaller ones in steps of 2^-20 (bfloat16) or 2^-36 (float32) of
it at most, off by half a step.  The float32 sums: at most K additions, each off by 2^-23 of what has been summed; the float32 result: 2^-24."""

import pytest
import torch

from thing_htn_2026_b200 import ops

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -20, torch.float32: 2.0 ** -36}
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def weight_without_first(n, k, seed):
    """Any codes, the first of every block of 32 zero; scales of 2^-3 to 2^3."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    codes[:, ::32] = 0
    scales = torch.randint(124, 131, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    held = codes[:, 0::2] | codes[:, 1::2] << 4
    w = torch.tensor(MAGNITUDES, dtype=torch.float64, device="cuda")[codes.long() & 7] * torch.where(codes >= 8, -1.0, 1.0)
    return ops.mx4_from_parts(held, scales, k), w * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


@pytest.mark.parametrize("down", [5, 12, 13, 16, 19, 24, 33, 41])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 4, 8, 20, 60, 150])
def test_small_entries(m, dtype, down):
    """Entries of 2^-down to 2^(1-down) of their block's largest."""
    n, k = 130, 640
    g = torch.Generator(device="cuda").manual_seed(down)
    x = (1 + torch.rand((m, k), generator=g, device="cuda")) * torch.where(torch.rand((m, k), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x *= 2.0 ** -down
    x[:, ::32] = 1.0
    x = (x * 2.0 ** torch.randint(-20, 20, (m, 1), generator=g, device="cuda")).to(dtype)
    weight, w = weight_without_first(n, k, 3)
    got = ops.linear_mx4(x, weight, out_dtype=torch.float32).double()
    x64 = x.double()
    y = x64 @ w.t()
    limit = k * 2.0 ** -23 * (x64.abs() @ w.abs().t())
    if down > 13:
        limit += STEP[dtype] / 2 * (x64[:, ::32].abs().repeat_interleave(32, dim=1) @ w.abs().t())
    limit += 2.0 ** -24 * (y.abs() + limit)
    assert ((got - y).abs() <= limit).all(), float(((got - y).abs() / limit).max())
