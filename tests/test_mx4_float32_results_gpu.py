"""Float32 results of bfloat16 rows and rows in 4 bits are summed as in float32 (see test_float32_rows_are_summed_as_in_float32 for the bound)."""

import pytest
import torch

from test_mx4_gpu import weight_of
from thing_htn_2026_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [1000, 4096, 12288])
@pytest.mark.parametrize("m", [3, 8, 32, 64, 65, 100, 300, 1000])
@pytest.mark.parametrize("quantized", [False, True])
def test_float32_results_are_summed_as_in_float32(m, k, quantized):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16()
    weight, w = weight_of(1024, k, k)
    given = ops.quantize_mx4(x) if quantized else x
    y = (ops.dequantize_mx4(given) if quantized else x).double() @ w.t()
    error = ops.linear_mx4(given, weight, out_dtype=torch.float32).double() - y
    assert error.norm() <= (k / 6) ** 0.5 * 2.0 ** -24 * y.norm()
