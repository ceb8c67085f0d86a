"""Sums so long that a tile's products take more than the 20 ms after which a wait for a single stage gives up."""

import pytest
import torch

from thing_htn_2026_b200 import ops

pytestmark = pytest.mark.gpu


def test_a_sum_of_four_million_columns():
    """192 float32 rows are six terms: 2,304 clocks of products for 128 columns, 39 ms at 1.965 GHz.  All but the first and the last 64 entries of a row
    are zero, and adding zeros is exact: at most 128 additions are off by 2^-23 of what has been summed, the rows by 2^-22 of a block's
    largest entry, the result's rounding by 2^-24."""
    m, n, k, ends = 192, 24, 1 << 22, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.zeros((m, k), device="cuda")
    x[:, :ends] = torch.randn((m, ends), generator=g, device="cuda")
    x[:, -ends:] = torch.randn((m, ends), generator=g, device="cuda")
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    weight = ops.mx4_from_parts(codes, torch.full((n, k // 32), 127, device="cuda", dtype=torch.uint8), k)
    err = ops.new_error_word("cuda")
    got = ops.linear_mx4(x, weight, err=err)
    ops.raise_on_device_error(err, "test")
    at = torch.cat([torch.arange(ends), torch.arange(k - ends, k)]).cuda()
    pairs = codes[:, torch.cat([torch.arange(ends // 2), torch.arange((k - ends) // 2, k // 2)]).cuda()]
    c = torch.stack((pairs & 15, pairs >> 4), dim=-1).flatten(1).long()
    w = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    x64 = x[:, at].double()
    y = x64 @ w.t()
    tops = x64.abs().unflatten(1, (-1, 32)).amax(dim=2).repeat_interleave(32, dim=1)
    limit = 128 * 2.0 ** -23 * (x64.abs() @ w.abs().t()) + 2.0 ** -22 * (tops @ w.abs().t())
    limit += 2.0 ** -24 * (y.abs() + limit)
    assert ((got.double() - y).abs() <= limit).all()
