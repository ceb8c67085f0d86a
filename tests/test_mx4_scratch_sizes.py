"""Remembered sizes of the 4-bit products' scratch: for each device, and no more of them than a fixed number."""

import torch

from thing_htn_2026_b200 import ops


class Library:
    """One that needs m bytes on device 0 and 2 m on device 1."""

    def __init__(self, device):
        self.device, self.calls = device, 0

    def thn_mx4_pair_scratch(self, kind, m, n, k, size):
        self.calls += 1
        size._obj.value = m * (1 + self.device[0])


def test_sizes_are_remembered(monkeypatch):
    device = [0]
    library = Library(device)
    monkeypatch.setattr(ops, "lib", lambda: library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: device[0], raising=False)
    monkeypatch.setattr(ops, "_mx4_terms_needs", {})
    monkeypatch.setattr(ops, "_MX4_KEPT", 50)
    need = lambda m: ops._mx4_terms_need("thn_mx4_pair_scratch", 1, m, 256, 512)
    assert need(7) == 7 and need(7) == 7 and library.calls == 1
    device[0] = 1
    assert need(7) == 14 and library.calls == 2
    device[0] = 0
    assert need(7) == 7 and library.calls == 2
    for m in range(1, 500):
        assert need(m) == m
        assert len(ops._mx4_terms_needs) <= 50


def test_the_rows_of_the_product_of_few_rows_stand_once():
    """Scratch is asked of the product that takes the rows; the library says which that is."""
    for kind in range(3):
        most = ops._mx4_few_rows(kind)
        assert most == ops.lib().thn_mx4_stream_rows(kind) and most >= 8
