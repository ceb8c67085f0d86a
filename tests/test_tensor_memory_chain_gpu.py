"""Kernels that hold tensor memory, one behind the other: grouped experts on pairs, 4-bit products on pairs and of few rows, in a recorded graph and
on two streams, give what each gives alone."""

import math

import pytest
import torch

from thing_htn_2026_b200 import ops

pytestmark = pytest.mark.gpu


def operands():
    g = torch.Generator(device="cuda").manual_seed(7)

    def rand(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0, std, generator=g)

    hidden, experts, ff, shared_ff, top, rows = 512, 8, 256, 256, 2, 700
    width = experts * ff + shared_ff
    x = rand(rows, hidden).bfloat16()
    w_up, w_down = rand(2 * width, hidden, std=hidden ** -0.5).bfloat16(), rand(hidden, width, std=ff ** -0.5).bfloat16()
    z = rand(rows, experts + 1)
    routing = ops.moe_route(z, experts, 1, 1, top, 1.0, scoring="softmax_chosen")
    weight = ops.quantize_mx4(rand(19000, hidden, std=0.05).bfloat16())
    narrow = ops.quantize_mx4(rand(640, 2560, std=0.05).bfloat16())
    few, long_rows = x[:3].contiguous(), rand(5, 2560).bfloat16()
    err = ops.new_error_word(torch.device("cuda"))
    experts_of = lambda: ops.grouped_experts(x, routing, w_up, w_down, ff, shared_ff, (math.inf, math.inf, 1.0, 0.0, "output"), z, experts, err)
    return err, [experts_of,
                 lambda: ops.linear_mx4(few, weight, err=err),
                 lambda: ops.linear_mx4(x, weight, err=err),
                 lambda: ops.linear_mx4(long_rows, narrow, err=err),
                 experts_of,
                 lambda: ops.linear_mx4(ops.quantize_mx4(few, to_multiply=True), weight, err=err),
                 lambda: ops.linear_mx4(ops.quantize_mx4(x, to_multiply=True), weight, err=err),
                 lambda: ops.linear(few, w_up, err=err)]


def test_one_behind_the_other():
    err, calls = operands()
    want = []
    for call in calls:
        torch.cuda.synchronize()
        want.append(call())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [call() for _ in range(3) for call in calls]
    for _ in range(5):
        graph.replay()
    again = [call() for _ in range(3) for call in calls]
    ops.raise_on_device_error(err, "test")
    for results in (got, again):
        assert all(torch.equal(results[i], want[i % len(calls)]) for i in range(len(results)))


def test_side_by_side():
    err, calls = operands()
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(4):
        for stream, order in zip(streams, (calls, calls[::-1])):
            with torch.cuda.stream(stream):
                got.append([call() for call in order][::1 if order is calls else -1])
    torch.cuda.synchronize()
    ops.raise_on_device_error(err, "test")
    for results in got:
        assert all(torch.equal(a, b) for a, b in zip(results, want))
