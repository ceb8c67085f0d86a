"""A matrix that was quantised to be multiplied is no weight: a product reads its weight while the kernels before it are still at work, and that
one's kernel lets the next be scheduled ahead of its end."""

import pytest
import torch

from thing_htn_2026_b200 import ops


def test_such_a_matrix_is_refused_as_a_weight():
    rows, columns = 4, 64
    q = ops.Mx4.__new__(ops.Mx4)._set(torch.zeros(ops._mx4_bytes(rows, columns), dtype=torch.uint8), rows, columns, only_rows=True)
    x = torch.zeros(2, columns)
    for product in (ops.linear_mx4, ops.linear, ops.linear_swiglu):
        with pytest.raises(ops.KernelError, match="to_multiply"):
            product(x, q)


@pytest.mark.gpu
def test_which_matrices_are_such():
    x = torch.randn(3, 96, device="cuda")
    q, w = ops.quantize_mx4(x, to_multiply=True), ops.quantize_mx4(x)
    parts = ops.mx4_from_parts(torch.zeros((3, 48), dtype=torch.uint8, device="cuda"), torch.zeros((3, 3), dtype=torch.uint8, device="cuda"), 96)
    assert q.only_rows and not w.only_rows and not parts.only_rows and not ops.Mx4(w.data.clone(), 3, 96).only_rows
    with pytest.raises(ops.KernelError, match="to_multiply"):
        ops.linear_mx4(w, q)
    with pytest.raises(ops.KernelError, match="to_multiply"):
        ops.linear(x, q)
    assert torch.equal(ops.linear_mx4(q, w), ops.linear_mx4(w, w)) and torch.equal(ops.dequantize_mx4(q), ops.dequantize_mx4(w))
