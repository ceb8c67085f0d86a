"""Matrices in microscaled 4-bit floating point against their definition in 64 bits.

Quantising and going back are exact but for the one rounding that the definition names, so codes, scales and values are
compared for equality.  A product's error is bounded by arithmetic:

* its float32 sums: at most K additions, each off by a unit in the last place at most, 2^-23 of what has been summed so far:
  K 2^-23 sum |x w|;
* rows in bfloat16 or float32 are multiplied as they are; a kernel may hold them as whole multiples of a block's step, off by half a
  step, at most 2^-16 (bfloat16) or 2^-22 (float32) of the block's largest entry: that times sum over the row of top |w|;
* the one rounding to the output: half a step, 2^-8 (bfloat16) or 2^-24 (float32) of the value.
"""

import numpy as np
import pytest
import torch

from plain import mx4_plain as plain
from thing_htn_2026_b200 import ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ROW_STEP = {torch.bfloat16: 2.0 ** -16, torch.float32: 2.0 ** -22}
DTYPES = [torch.bfloat16, torch.float32]


def as64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def rows_of(rows, columns, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, columns), generator=g) * spread
    x *= 2.0 ** torch.randint(-3, 4, (rows, columns), generator=g)
    return x.to(dtype).cuda()


def weight_of(n, k, seed):
    """(the library's matrix, its values in float64 on the device): any codes, scales of 2^-9 to 2^-1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = -(-k // 32)
    stored = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(118, 127, (n, blocks), generator=g, device="cuda", dtype=torch.uint8)
    codes = torch.stack((stored & 15, stored >> 4), dim=-1).flatten(1)[:, :k].long()
    values = torch.tensor(plain.MAGNITUDES, device="cuda")[codes & 7] * torch.where(codes >= 8, -1.0, 1.0).double()
    values *= torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)[:, :k]
    return ops.mx4_from_parts(stored, scales, k), values


def scale_bytes(q):
    """[rows, blocks] of a matrix's scales."""
    tiles = q.scales.cpu().numpy().reshape(q.scales.shape[0], q.scales.shape[1], 32, 4, 4)
    flat = tiles.transpose(0, 3, 2, 1, 4).reshape(q.scales.shape[0] * 128, -1)      # row = 32 * (middle axis) + lane
    return flat[:q.rows, :-(-q.columns // 32)]


def check_quantized(x):
    q = ops.quantize_mx4(x)
    codes, scales = plain.quantize(as64(x))
    assert np.array_equal(scale_bytes(q), scales)
    got = q.codes.cpu().numpy()
    want = np.zeros((q.rows, q.codes.shape[1]), dtype=np.uint8)
    stored = plain.stored(codes, q.columns)
    want[:, :stored.shape[1]] = stored
    assert np.array_equal(got, want)
    for dtype in DTYPES:
        np.testing.assert_array_equal(as64(ops.dequantize_mx4(q, dtype)), plain.values(codes, scales, q.columns))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 32), (1, 2560), (3, 31), (5, 33), (37, 1000), (127, 128), (128, 136), (129, 264),
                                          (300, 520), (2, 4099)])
def test_quantized_matrix_is_the_definition(rows, columns, dtype):
    check_quantized(rows_of(rows, columns, dtype, rows * 10007 + columns))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_midpoint_sign_and_scale(dtype):
    """Blocks whose largest entry is 4 or 7.5 of their scale, with every midpoint between two magnitudes and its neighbours, over all
    scales that the type reaches, zeros of both signs, subnormal numbers and blocks of zeros."""
    eps = torch.finfo(dtype).eps
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    rows = []
    for top in (4.0, 7.5):
        for e in list(range(-133, -120)) + list(range(-5, 6)) + list(range(120, 126)):
            row = torch.cat([torch.tensor([top, -0.0, 0.0, -6.0 if top > 6 else -3.0], dtype=torch.float64), middle, -middle,
                             middle * (1 + eps), middle * (1 - eps)])
            rows.append(row * 2.0 ** e)
    x = torch.stack(rows + [torch.zeros(32, dtype=torch.float64), -torch.zeros(32, dtype=torch.float64)]).to(dtype).cuda()
    assert torch.isfinite(x).all()
    check_quantized(x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_number_that_is_not_finite(dtype, bad):
    x = rows_of(4, 200, dtype, 5)
    x[1, 40] = bad
    x[3, 199] = bad
    check_quantized(x)
    values = as64(ops.dequantize_mx4(ops.quantize_mx4(x)))
    gone = np.isnan(values)
    assert gone[1, 32:64].all() and gone[3, 192:].all() and gone.sum() == 32 + 8


@pytest.mark.parametrize("columns", [1, 31, 32, 95, 128, 1000])
def test_stored_parts_keep_every_code_and_scale(columns):
    g = np.random.default_rng(columns)
    codes = g.integers(0, 16, (130, -(-columns // 32), 32), dtype=np.uint8)
    scales = g.integers(0, 255, (130, -(-columns // 32)), dtype=np.uint8)
    scales[7, 0] = 255
    stored = plain.stored(codes, columns)
    if columns % 2:
        stored[:, -1] |= 0x50          # the half byte behind the last entry means nothing
    q = ops.mx4_from_parts(torch.from_numpy(stored).cuda(), torch.from_numpy(scales).cuda(), columns)
    assert q.shape == (130, columns)
    with np.errstate(over="ignore"):
        want = plain.values(codes, scales, columns).astype(np.float32)      # 6 * 2^127 is beyond float32
    np.testing.assert_array_equal(ops.dequantize_mx4(q).cpu().numpy(), want)


def tops(x):
    """For every entry of float64 [rows, columns], the largest magnitude of its block."""
    blocks = torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    return blocks.amax(dim=2).repeat_interleave(32, dim=1)[:, :x.shape[1]]


def bound(x, w, y, x_dtype, out_dtype, bias):
    """How far a product may be off, entry by entry (see the top of this file)."""
    sums = x.abs() @ w.abs().t()
    if bias is not None:
        sums += bias.abs()
    e = x.shape[1] * 2.0 ** -23 * sums
    if x_dtype is not None:
        e += ROW_STEP[x_dtype] * (tops(x) @ w.abs().t())
    return e + HALF_STEP[out_dtype] * (y.abs() + e)


def check_product(m, n, k, x_dtype, out_dtype, with_bias=False, quantized=False, seed=0, spread=1.0):
    x = rows_of(m, k, x_dtype, seed + 1, spread)
    weight, w = weight_of(n, k, seed + 2)
    bias = rows_of(1, n, x_dtype, seed + 3)[0] if with_bias else None
    err = ops.new_error_word("cuda")
    given = ops.quantize_mx4(x) if quantized else x
    got = ops.linear_mx4(given, weight, out_dtype=out_dtype, bias=bias, err=err)
    assert got.dtype == out_dtype and tuple(got.shape) == (m, n)
    ops.raise_on_device_error(err, "test")
    x64 = torch.from_numpy(plain.values(*plain.quantize(as64(x)), k)).cuda() if quantized else x.double()
    b64 = None if bias is None else bias.double()
    y = x64 @ w.t() + (0 if bias is None else b64)
    error = (got.double() - y).abs()
    limit = bound(x64, w, y, None if quantized else x_dtype, out_dtype, b64)
    assert (error <= limit).all(), (error / limit.clamp(min=1e-300)).max()


SIZES = [(1, 1, 1), (1, 128, 256), (1, 2560, 2560), (2, 100, 32), (3, 515, 1096), (5, 1333, 1000), (8, 640, 2432), (9, 129, 4100), (16, 256, 640),
         (17, 384, 128), (31, 130, 384), (33, 257, 999), (42, 512, 256), (43, 512, 256), (64, 1000, 512), (77, 515, 1096), (100, 24, 8192),
         (128, 128, 128), (129, 300, 1500), (200, 2000, 320), (257, 513, 130), (300, 256, 3000), (511, 260, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_of_rows_as_they_are(m, n, k, dtype):
    check_product(m, n, k, dtype, dtype, with_bias=(m + n) % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_of_quantized_rows(m, n, k, dtype):
    check_product(m, n, k, dtype, dtype, with_bias=(m + n) % 2 == 0, quantized=True)


@pytest.mark.parametrize("m", [4, 60, 300])
@pytest.mark.parametrize("quantized", [False, True])
def test_product_with_the_other_output_type(m, quantized):
    check_product(m, 260, 500, torch.bfloat16, torch.float32, quantized=quantized)
    check_product(m, 260, 500, torch.float32, torch.bfloat16, quantized=quantized)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 19100, 2050), (8, 19100, 1300), (3, 9700, 2600), (5, 200, 20000), (20, 19100, 700), (60, 9700, 1000)])
def test_product_of_many_pieces_of_k_a_block(m, n, k, dtype):
    """Blocks that go round their ring of stages several times."""
    check_product(m, n, k, dtype, dtype)
    check_product(m, n, k, dtype, dtype, quantized=True)


@pytest.mark.parametrize("quantized", [False, True])
def test_rows_of_several_bands(quantized):
    """More bytes of rows than are multiplied by all of the weight at once, with a last band and a last tile of another size."""
    m, n, k = (4100, 520, 8200) if not quantized else (13000, 520, 8200)
    x = rows_of(m, k, torch.bfloat16, 1)
    weight, w = weight_of(n, k, 2)
    given = ops.quantize_mx4(x) if quantized else x
    got = ops.linear_mx4(given, weight, out_dtype=torch.float32)
    few = torch.cat([torch.arange(0, m, 97), torch.arange(m - 70, m)]).cuda()
    x64 = (ops.dequantize_mx4(given) if quantized else x)[few].double()
    y = x64 @ w.t()
    error = (got[few].double() - y).abs()
    assert (error <= bound(x64, w, y, None if quantized else torch.bfloat16, torch.float32, None)).all()
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("k", [1000, 4096, 12288])
@pytest.mark.parametrize("m", [3, 8, 32, 33, 100, 300])
def test_float32_rows_are_summed_as_in_float32(m, k):
    """The error's root mean square is at most that of products added one after the other in float32: with both signs the partial sum
    after i of K grows as sqrt(i / K) of the result, and each addition is off by 2^-24 / sqrt(3) of it in the mean, so sqrt(K / 6) 2^-24 of the
    result's."""
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x = torch.randn((m, k), generator=g, device="cuda")
    weight, w = weight_of(1024, k, k)
    y = x.double() @ w.t()
    error = ops.linear_mx4(x, weight).double() - y
    assert error.norm() <= (k / 6) ** 0.5 * 2.0 ** -24 * y.norm()


@pytest.mark.parametrize("spread", [2.0 ** -60, 2.0 ** 60])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 150])
def test_product_of_far_rows(m, dtype, spread):
    check_product(m, 200, 700, dtype, dtype, spread=spread)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("m", [2, 40, 140, 300])
def test_what_is_not_a_number_stays_in_its_row_and_column(m, quantized):
    """A NaN or an infinity in a row of x makes that row NaN, one in a row of the weight that column; the rest is as without them."""
    x = rows_of(m, 600, torch.bfloat16, 3)
    g = torch.Generator().manual_seed(4)
    w = torch.randn((200, 600), generator=g).cuda()
    clean = ops.linear_mx4(ops.quantize_mx4(x) if quantized else x, ops.quantize_mx4(w))
    x[1, 555] = float("nan")
    w[130, 17] = float("inf")
    got = ops.linear_mx4(ops.quantize_mx4(x) if quantized else x, ops.quantize_mx4(w))
    assert torch.isnan(got[1]).all() and torch.isnan(got[:, 130]).all()
    keep_rows = torch.arange(m, device="cuda") != 1
    keep = torch.arange(200, device="cuda") != 130
    assert torch.equal(got[keep_rows][:, keep], clean[keep_rows][:, keep])


def test_no_rows():
    weight, _ = weight_of(10, 64, 0)
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.quantize_mx4(x).shape == (0, 64)
    assert tuple(ops.dequantize_mx4(ops.quantize_mx4(x)).shape) == (0, 64)
    assert tuple(ops.linear_mx4(x, weight).shape) == (0, 10)
    assert tuple(ops.linear_mx4(ops.quantize_mx4(x), weight).shape) == (0, 10)


def test_refusals():
    weight, _ = weight_of(10, 64, 0)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.KernelError, match="dtype"):
        ops.quantize_mx4(x.half())
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.quantize_mx4(x.t())
    with pytest.raises(ops.KernelError, match="matrix"):
        ops.quantize_mx4(x[0])
    with pytest.raises(ops.KernelError, match="matrix"):
        ops.quantize_mx4(x[:, :0].contiguous())
    with pytest.raises(ops.KernelError, match="dtype"):
        ops.dequantize_mx4(weight, torch.float16)
    with pytest.raises(ops.KernelError, match="shapes"):
        ops.linear_mx4(x[:, :32].contiguous(), weight)
    with pytest.raises(ops.KernelError, match="shapes"):
        ops.linear_mx4(ops.quantize_mx4(x[:, :32].contiguous()), weight)
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.linear_mx4(torch.zeros((64, 2), dtype=torch.bfloat16, device="cuda").t(), weight)
    with pytest.raises(ops.KernelError, match="out_dtype"):
        ops.linear_mx4(x, weight, out_dtype=torch.float16)
    with pytest.raises(ops.KernelError, match="bias"):
        ops.linear_mx4(x, weight, bias=torch.zeros(9, device="cuda"))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.linear_mx4(x.cpu(), weight)
    narrow, _ = weight_of(3, 1, 0)
    with pytest.raises(ops.KernelError, match="at most"):
        ops.linear_mx4(torch.zeros(((1 << 24) + 1, 1), dtype=torch.bfloat16, device="cuda"), narrow)
    with pytest.raises(ops.KernelError, match="Mx4"):
        ops.linear_mx4(x, torch.zeros((10, 64), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ops.KernelError, match="err"):
        ops.linear_mx4(x, weight, err=torch.zeros(1, device="cuda"))
    with pytest.raises(ops.KernelError, match="Mx4"):
        ops.dequantize_mx4(x)
    parts = torch.zeros((4, 32), dtype=torch.uint8, device="cuda")
    with pytest.raises(ops.KernelError, match="codes"):
        ops.mx4_from_parts(parts, torch.zeros((4, 3), dtype=torch.uint8, device="cuda"), 64)
    with pytest.raises(ops.KernelError, match="codes"):
        ops.mx4_from_parts(parts, torch.zeros((4, 2), dtype=torch.uint8, device="cuda"), 70)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 20, 90])
def test_rows_that_begin_anywhere(m, dtype):
    """Rows and a bias whose first entry is not at a multiple of 16 bytes."""
    n, k = 300, 512
    weight, _ = weight_of(n, k, 7)
    x, bias = rows_of(m, k, dtype, 8), rows_of(1, n, dtype, 9)[0]
    shifted = torch.empty(m * k + 1, dtype=dtype, device="cuda")[1:].view(m, k).copy_(x)
    moved = torch.empty(n + 1, dtype=dtype, device="cuda")[1:].copy_(bias)
    assert shifted.data_ptr() % 16 and shifted.is_contiguous()
    assert torch.equal(ops.linear_mx4(shifted, weight, bias=moved), ops.linear_mx4(x, weight, bias=bias))
    a, b = ops.quantize_mx4(shifted), ops.quantize_mx4(x)
    assert torch.equal(a.codes, b.codes) and np.array_equal(scale_bytes(a), scale_bytes(b))


@pytest.mark.parametrize("m,n,k", [(1, 2560, 9728), (8, 6144, 2560), (40, 2560, 4096), (300, 1000, 1000)])
@pytest.mark.parametrize("quantized", [False, True])
def test_the_same_call_gives_the_same_bits(m, n, k, quantized):
    weight, _ = weight_of(n, k, 1)
    x = rows_of(m, k, torch.bfloat16, 2)
    given = ops.quantize_mx4(x) if quantized else x
    first = ops.linear_mx4(given, weight, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(ops.linear_mx4(given, weight, out_dtype=torch.float32), first)


@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 32), (130, 96), (129, 4128), (5, 4100), (7, 2056), (300, 77)])
def test_stored_parts_that_begin_anywhere(rows, columns):
    """Stored codes and scales at odd addresses, beside the same at whole pieces; the unused half of a row's last byte is not taken."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    codes = torch.randint(0, 256, (rows, (columns + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(0, 256, (rows, -(-columns // 32)), generator=g, device="cuda", dtype=torch.uint8)
    moved = [torch.empty(t.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(t.shape).copy_(t) for t in (codes, scales)]
    want = torch.zeros((rows, -(-columns // 128) * 64), dtype=torch.uint8, device="cuda")
    want[:, :codes.shape[1]] = codes
    if columns % 2:
        want[:, codes.shape[1] - 1] &= 15
    for parts in ((codes, scales), moved):
        q = ops.mx4_from_parts(*parts, columns)
        assert torch.equal(q.codes, want) and np.array_equal(scale_bytes(q), scales.cpu().numpy())


def test_a_matrix_from_its_bytes():
    weight, _ = weight_of(130, 200, 3)
    again = ops.Mx4(weight.data.clone(), 130, 200)
    assert torch.equal(ops.dequantize_mx4(again), ops.dequantize_mx4(weight)) and again.nbytes == weight.nbytes
    for data, rows in ((weight.data[:-1], 130), (weight.data, 257), (weight.data.view(2, -1), 130), (weight.data.view(torch.int8), 130),
                       (weight.data.cpu(), 130)):
        with pytest.raises(ops.KernelError, match="Mx4"):
            ops.Mx4(data, rows, 200)
    with pytest.raises(ops.KernelError, match="Mx4"):
        ops.Mx4(torch.zeros(weight.nbytes + 1, dtype=torch.uint8, device="cuda")[1:], 130, 200)


def test_another_stream_and_a_recorded_graph():
    """Calls on a side stream, two recorded graphs that are replayed in turn with inputs of their own, and eager calls between."""
    weight, w = weight_of(384, 512, 9)
    inputs = [rows_of(m, 512, torch.bfloat16, 20 + m) for m in (2, 70)]
    want = [ops.linear_mx4(x, weight) for x in inputs] + [ops.linear_mx4(ops.quantize_mx4(x), weight) for x in inputs]
    static = [x.clone() for x in inputs]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.linear_mx4(x, weight) for x in static]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([ops.linear_mx4(x, weight), ops.linear_mx4(ops.quantize_mx4(x, to_multiply=True), weight)])
        graphs.append(graph)
    for _ in range(3):
        for x in static:
            x.zero_()
        for graph in graphs:
            graph.replay()
        assert all((o == 0).all() for pair in outs for o in pair)
        for x, source in zip(static, inputs):
            x.copy_(source)
        for graph in reversed(graphs):
            graph.replay()
        eager = ops.linear_mx4(inputs[0], weight)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for i in range(2):
            assert torch.equal(again[i], want[i])
            assert torch.equal(outs[i][0], want[i]) and torch.equal(outs[i][1], want[2 + i])


@pytest.mark.parametrize("m", [1, 8, 40, 100])
def test_a_weight_that_was_written_just_before(m):
    """Quantised, brought back, or taken from its parts by the kernel ahead of the product that reads it, again and again in the same memory."""
    n, k, count = 19000, 2560, 12
    g = torch.Generator(device="cuda").manual_seed(1)
    source = [torch.randn((n, k), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    parts = [(torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8),
              torch.randint(118, 127, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8)) for _ in range(2)]
    x = rows_of(m, k, torch.bfloat16, 2)
    makes = [lambda i: ops.quantize_mx4(source[i]), lambda i: ops.mx4_from_parts(*parts[i], k)]
    for make in makes:
        held = [make(i) for i in range(2)]
        torch.cuda.synchronize()
        want = [ops.linear_mx4(x, w) for w in held]
        torch.cuda.synchronize()
        got = [ops.linear_mx4(x, make(i % 2)) for i in range(count)]
        got += [ops.linear_mx4(ops.quantize_mx4(x), make(i % 2)) for i in range(count)]
        rows = ops.linear_mx4(ops.quantize_mx4(x), held[0]), ops.linear_mx4(ops.quantize_mx4(x), held[1])
        for i in range(count):
            assert torch.equal(got[i], want[i % 2]) and torch.equal(got[count + i], rows[i % 2])
    held = [ops.quantize_mx4(s) for s in source]
    back = [ops.dequantize_mx4(w, torch.bfloat16) for w in held]
    torch.cuda.synchronize()
    want = [ops.linear(x, w) for w in back]
    torch.cuda.synchronize()
    del back
    got = [ops.linear(x, ops.dequantize_mx4(held[i % 2], torch.bfloat16)) for i in range(count)]
    assert all(torch.equal(got[i], want[i % 2]) for i in range(count))


def test_two_streams_at_once():
    """The same weight multiplied on two streams whose calls overlap: few rows, many rows and quantised rows."""
    weight, _ = weight_of(4000, 2048, 5)
    inputs = [rows_of(m, 2048, dtype, m) for m, dtype in ((1, torch.bfloat16), (6, torch.float32), (30, torch.bfloat16), (260, torch.bfloat16),
                                                         (100, torch.float32))]

    def all_products():
        return [ops.linear_mx4(x, weight) for x in inputs] + [ops.linear_mx4(ops.quantize_mx4(x), weight) for x in inputs]

    want = all_products()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(all_products())
    torch.cuda.synchronize()
    for products in got:
        assert all(torch.equal(a, b) for a, b in zip(products, want))


@pytest.mark.parametrize("m,entry", [(5, "thn_mx4_stream"), (60, "thn_mx4_stream"), (200, "thn_mx4_pair")])
@pytest.mark.parametrize("quantized", [False, True])
def test_a_wait_that_runs_out_is_reported(m, entry, quantized):
    """Nothing is loaded: the waits for it end, the error word says so, the result is no number."""
    weight, _ = weight_of(300, 640, 1)
    x = rows_of(m, 640, torch.bfloat16, 2)
    q = ops.quantize_mx4(x)
    out = torch.zeros((m, 300), dtype=torch.float32, device="cuda")
    err = ops.new_error_word("cuda")
    data, scales, kind = (q.codes, q.scales, 2) if quantized else (x, None, 1)
    room = torch.empty(ops._mx4_terms_need(entry + "_scratch", kind, m, 300, 640) or 16, dtype=torch.uint8, device="cuda")
    ops._call(entry, out.data_ptr(), 0, data.data_ptr(), ops._ptr(scales), kind, weight.codes.data_ptr(), weight.scales.data_ptr(), None, 0,
              room.data_ptr(), room.numel(), m, 300, 640, 1, err.data_ptr(), ops._stream())
    with pytest.raises(ops.KernelError, match="gave up"):
        ops.raise_on_device_error(err, "test")
    assert torch.isnan(out).all()
    again = ops.linear_mx4(q if quantized else x, weight, out_dtype=torch.float32, err=err)
    ops.raise_on_device_error(err, "test")
    assert torch.isfinite(again).all()
