"""The block-scaled FP8 linear on the GPU against float64: quantizers bit for bit, products within
the rounding bound of their fp32 sums."""

from __future__ import annotations

import threading
import time

import numpy as np
import pytest
import torch

import fp8_reference as ref
from qpu_xla.fp8 import (
    PreparedFP8Experts,
    PreparedFP8Linear,
    QuantizedBlocksFP8,
    QuantizedRowsFP8,
    quantize_blocks_fp8,
    quantize_rows_fp8,
)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def draw(shape, dtype=torch.float32, seed=0, std=1.0) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def blocks(device, n: int, k: int, seed: int = 1, experts: int = 0) -> QuantizedBlocksFP8:
    return quantize_blocks_fp8(device, draw((experts, n, k) if experts else (n, k), seed=seed, std=0.05))


def check_rows(rows: QuantizedRowsFP8, x: torch.Tensor) -> None:
    values, scales = ref.quantize_rows(x)
    torch.testing.assert_close(rows.scales.double(), scales, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(rows.values.double(), values, rtol=0, atol=0, equal_nan=True)


def check_product(y: torch.Tensor, exact: torch.Tensor, magnitude: torch.Tensor, k: int) -> None:
    assert y.shape == exact.shape
    excess = ((y.double() - exact).abs() - ref.product_tolerance(exact, magnitude, k, y.dtype)).max().item() if y.numel() else 0.0
    assert excess <= 0.0, f"beyond the bound by {excess}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 127), (5, 128), (2, 129), (9, 255), (33, 1000), (70, 5001), (64, 8192), (1, 28672)])
def test_row_quantizer_is_bit_exact(cuda_device, dtype, rows, cols) -> None:
    x = draw((rows, cols), dtype, seed=rows * 7 + cols)
    check_rows(quantize_rows_fp8(cuda_device, x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_row_quantizer_ties_and_magnitudes(cuda_device, dtype) -> None:
    """Values on and beside every e4m3 border (the scale is 1: each group's largest is 448), and
    groups from the smallest to the largest magnitudes of the type."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    borders = torch.cat([codes, (codes[1:] + codes[:-1]) / 2]).to(dtype)
    beside = torch.cat([torch.nextafter(borders, torch.full_like(borders, 1e4)), torch.nextafter(borders, torch.full_like(borders, -1e4))])
    values = torch.cat([borders, beside, -borders, -beside]).double().clamp(-448, 448).to(dtype)
    values = torch.cat([values, torch.zeros(-values.numel() % 127, dtype=dtype)]).view(-1, 127)
    x = torch.cat([torch.full((values.shape[0], 1), 448.0, dtype=dtype), values], dim=1).cuda()
    check_rows(quantize_rows_fp8(cuda_device, x), x)
    exponents = torch.linspace(*((-14.0, 15.9) if dtype == torch.float16 else (-120.0, 127.0)), 300, dtype=torch.float64)
    x = (draw((300, 128), seed=5).cpu().double().clamp(-1, 1) * torch.exp2(exponents)[:, None]).to(dtype).cuda()
    check_rows(quantize_rows_fp8(cuda_device, x), x)


def test_row_quantizer_zero_nan_and_infinite_groups(cuda_device) -> None:
    x = draw((6, 300), seed=3)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 140] = float("inf")
    x[3, 299] = -float("inf")
    x[4, 128:256] = -0.0
    rows = quantize_rows_fp8(cuda_device, x)
    dequantized = rows.dequantize()
    assert torch.equal(dequantized[0], torch.zeros_like(dequantized[0]))
    for row, group in ((1, 0), (2, 1), (3, 2)):
        damaged = torch.arange(300, device="cuda") // 128 == group
        assert dequantized[row][damaged].isnan().all()
        assert dequantized[row][~damaged].isfinite().all()
    keep = [0, 4, 5]
    check_rows(QuantizedRowsFP8(rows.values[keep], rows.scales[keep]), x[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_row_quantizer_takes_strided_and_unaligned_rows(cuda_device, dtype) -> None:
    base = draw((20, 700), dtype, seed=4)
    for x in (base[:, :512], base[:, 3:516], base[1::3, 8:520], base[5:6, 1:2]):
        check_rows(quantize_rows_fp8(cuda_device, x), x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(9, 300), (900, 4097)])
def test_row_quantizer_at_every_alignment(cuda_device, dtype, rows, cols) -> None:
    for stride in (cols + 7, cols + 8 + cols % 2, 2 * cols + 2):
        base = draw((rows + 1, stride), dtype, seed=stride)
        for start in range(8):
            x = base.view(-1)[start : start + rows * stride].view(rows, stride)[:, :cols]
            check_rows(quantize_rows_fp8(cuda_device, x), x)
        x = base[1:, : 2 * (cols // 2)]
        gated = quantize_rows_fp8(cuda_device, x, gated=True)
        again = quantize_rows_fp8(cuda_device, x.clone(), gated=True)
        assert torch.equal(gated.values.view(torch.uint8), again.values.view(torch.uint8)) and torch.equal(gated.scales, again.scales)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols, std", [(1, 1, 1.0), (4, 128, 1.0), (7, 333, 3.0), (40, 5632, 1.0), (50, 500, 40.0)])
def test_gated_rows(cuda_device, dtype, rows, cols, std) -> None:
    """exp is within 2 steps of 2^-23 (CUDA's bound), the sum and the product round once, the quotient is
    the rounded one: below 5 steps (2^-20.6) together, so the scale is that close. The value is then
    within half an e4m3 step (2^-4 of it, or 2^-10 of the scale below the normal range). Gates down to
    -160 go through the overflow of exp."""
    x = draw((rows, 2 * cols), dtype, seed=cols, std=std)
    rows_fp8 = quantize_rows_fp8(cuda_device, x, gated=True)
    exact = ref.silu_gate(x)
    _, scales = ref.quantize_rows(exact)
    torch.testing.assert_close(rows_fp8.scales.double(), scales, rtol=2.0**-20, atol=0)
    wide = ref.spread(rows_fp8.scales.double(), rows, cols, 1)
    bound = exact.abs() * (2.0**-4 + 2.0**-19) + wide * (2.0**-10 + 2.0**-19)
    assert ((rows_fp8.dequantize().double() - exact).abs() <= bound).all()


def test_gates_of_every_size(cuda_device) -> None:
    """One gate per group, across the range of fp32's exp and past both of its ends."""
    gates = torch.cat([torch.linspace(-110.0, 110.0, 400), torch.tensor([-1e30, -1e-30, 0.0, 1e-30, 1e30])])
    x = torch.zeros((gates.numel(), 256), device="cuda")
    x[:, 0], x[:, 128] = gates.cuda(), 3.0
    exact = ref.silu_gate(x)[:, 0]
    have = quantize_rows_fp8(cuda_device, x, gated=True).scales[:, 0].double() * 448.0
    wanted = exact.abs().clamp_min(448.0 * 2.0**-60)
    assert ((have - wanted).abs() <= 2.0**-20 * wanted).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, k", [(1, 1), (128, 128), (130, 300), (257, 1000)])
def test_block_quantizer_is_bit_exact(cuda_device, dtype, n, k) -> None:
    w = draw((n, k), dtype, seed=n + k)
    quantized = quantize_blocks_fp8(cuda_device, w)
    values, scales = ref.quantize_blocks(w)
    assert torch.equal(quantized.scales.double(), scales)
    assert torch.equal(quantized.values.double(), values)
    stacked = quantize_blocks_fp8(cuda_device, torch.stack([w, w * 3]))
    assert torch.equal(stacked.values[0].view(torch.uint8), quantized.values.view(torch.uint8))
    assert torch.equal(stacked.values[1].double(), ref.quantize_blocks(w * 3)[0])


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 300, 700])
@pytest.mark.parametrize("n, k", [(256, 256), (130, 1410), (1000, 2048)])
def test_linear_row_counts(cuda_device, rows, n, k) -> None:
    weight = blocks(cuda_device, n, k)
    x = draw((rows, k), torch.bfloat16, seed=rows)
    values, scales = ref.quantize_rows(x)
    exact, magnitude = ref.product(values, scales, weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        check_product(plan.forward(x), exact, magnitude, k)
        check_product(plan.forward(x, dtype=torch.float32), exact, magnitude, k)


@pytest.mark.parametrize("n, k", [(1, 1), (7, 16), (128, 100), (129, 128), (5, 129), (300, 17), (64, 5000), (4100, 640), (1, 28672)])
@pytest.mark.parametrize("rows", [1, 20, 260])
def test_linear_shapes(cuda_device, rows, n, k) -> None:
    weight = blocks(cuda_device, n, k)
    x = draw((rows, k), seed=n)
    values, scales = ref.quantize_rows(x)
    exact, magnitude = ref.product(values, scales, weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        check_product(plan.forward(x), exact, magnitude, k)


# One tile shape of the product each: a few rows, with and without a split K, and several such tiles; few
# wide tiles whose K is split in 4 and in 2; wide tiles alone and in pairs, more of them than SMs; a
# ragged last tile everywhere.
KERNELS = [(5, 300, 4096), (30, 40000, 300), (200, 1000, 4096), (300, 1000, 8192), (333, 5000, 2049), (640, 9000, 300), (1023, 5001, 384), (1023, 10000, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, n, k", KERNELS)
def test_every_kernel_and_output_layout(cuda_device, dtype, rows, n, k) -> None:
    """Contiguous, aligned and unaligned outputs inside a wider tensor, whose rest stays as it was."""
    weight = blocks(cuda_device, n, k)
    bias = draw((n,), seed=8)
    x = draw((rows, k), seed=rows)
    values, scales = ref.quantize_rows(x)
    exact, magnitude = ref.product(values, scales, weight.values, weight.scales)
    exact, magnitude = exact + bias.double(), magnitude + bias.double().abs()
    with PreparedFP8Linear(cuda_device, weight, bias=bias) as plan:
        y = plan.forward(x, dtype=dtype)
        check_product(y, exact, magnitude, k)
        assert torch.equal(plan.forward(x, dtype=dtype), y)
        for start, extra in ((8, 16 - n % 8), (3, 7)):
            wide = torch.full((rows + 2, n + start + extra), 7.0, dtype=dtype, device="cuda")
            plan.forward(x, out=wide[1:-1, start : start + n])
            assert torch.equal(wide[1:-1, start : start + n], y)
            wide[1:-1, start : start + n] = 7.0
            assert (wide == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "counts, trailing, n, k",
    [([130, 0, 1, 255, 40], 9, 300, 4096), ([130, 0, 1, 255, 40], 9, 1000, 4096), ([130, 0, 1, 255, 40], 9, 1500, 4096), ([70, 90], 3, 1000, 2048), ([500, 0, 700, 129, 640], 40, 3000, 300), ([1100, 1500, 900, 1025], 17, 3001, 256), ([1100, 1500, 900, 1025], 17, 3200, 256)],
)
def test_every_kernel_with_experts(cuda_device, dtype, counts, trailing, n, k) -> None:
    weight, x, offsets, exact, magnitude = expert_case(cuda_device, counts, n, k, trailing)
    with PreparedFP8Experts(cuda_device, weight) as plan:
        y = plan.forward(x, offsets, dtype=dtype)
        check_product(y, exact, magnitude, k)
        assert (y[sum(counts) :] == 0).all()
        wide = torch.full((x.shape[0] + 2, n + 16 - n % 8), 7.0, dtype=dtype, device="cuda")
        plan.forward(x, offsets, out=wide[1:-1, 8 : 8 + n])
        assert torch.equal(wide[1:-1, 8 : 8 + n], y)
        wide[1:-1, 8 : 8 + n] = 7.0
        assert (wide == 7.0).all()


@pytest.mark.parametrize("source", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 150, 520])
def test_linear_types_bias_and_strides(cuda_device, source, dtype, rows) -> None:
    n, k = 384, 513
    weight = blocks(cuda_device, n, k)
    bias = draw((n,), seed=8)
    x = draw((rows, k + 7), source, seed=9)[:, 3 : 3 + k]
    values, scales = ref.quantize_rows(x)
    exact, magnitude = ref.product(values, scales, weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight, bias=bias) as plan:
        wide = torch.full((rows + 2, n + 5), 7.0, dtype=dtype, device="cuda")
        out = wide[1:-1, 2 : 2 + n]
        assert plan.forward(x, out=out) is out
        check_product(out, exact + bias.double(), magnitude + bias.double().abs(), k)
        untouched = wide.clone()
        untouched[1:-1, 2 : 2 + n] = 7.0
        assert (untouched == 7.0).all()


@pytest.mark.parametrize("rows", [1, 40, 400])
def test_gated_linear_is_the_product_of_the_gated_rows(cuda_device, rows) -> None:
    n, k = 200, 700
    weight = blocks(cuda_device, n, k)
    x = draw((rows, 2 * k), torch.bfloat16, seed=rows)
    quantized = quantize_rows_fp8(cuda_device, x, gated=True)
    exact, magnitude = ref.product(quantized.values, quantized.scales, weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight, gated=True) as plan:
        check_product(plan.forward(x), exact, magnitude, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows, n, k", [(1, 1, 1), (1, 500, 900), (3, 130, 77), (4, 2048, 1000), (12, 300, 128), (16, 100, 100), (1, 2000, 2047), (5, 130, 1024), (1, 200, 9000)])
def test_rows_quantized_inside_the_product(cuda_device, dtype, gated, rows, n, k) -> None:
    """A few rows of a small matrix take one launch: bit for bit what the two steps give."""
    weight = blocks(cuda_device, n, k)
    wide = draw((rows + 1, 2 * k + 3), dtype, seed=k)
    for source in (wide[1:, : 2 * k if gated else k], wide[1:, 3 : 3 + (2 * k if gated else k)].contiguous()):
        with PreparedFP8Linear(cuda_device, weight, gated=gated) as plan:
            expected = plan.forward_quantized(quantize_rows_fp8(cuda_device, source, gated=gated), dtype=dtype)
            assert torch.equal(plan.forward(source), expected)


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_quantized_rows_give_the_same_product(cuda_device, rows) -> None:
    weight = blocks(cuda_device, 500, 900)
    x = draw((rows, 900), seed=rows)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        assert torch.equal(plan.forward_quantized(quantize_rows_fp8(cuda_device, x)), plan.forward(x))
        moved = quantize_rows_fp8(cuda_device, x)
        transposed = QuantizedRowsFP8(moved.values, moved.scales.t().contiguous().t())
        assert torch.equal(plan.forward_quantized(transposed), plan.forward(x))


@pytest.mark.parametrize("rows", [4, 30, 300])
@pytest.mark.parametrize("k", [1, 17, 100, 250])
def test_bytes_behind_a_row_do_not_count(cuda_device, rows, k) -> None:
    """Quantized rows end inside their last 16 bytes; whatever lies behind (NaN here) is not read as theirs."""
    values = torch.full((rows, (k + 15) // 16 * 16), 0x7F, dtype=torch.uint8, device="cuda")
    values[:, :k] = 0x38  # 1.0
    ones = QuantizedBlocksFP8(torch.ones((300, k), device="cuda").to(torch.float8_e4m3fn), torch.ones((3, -(-k // 128)), device="cuda"))
    with PreparedFP8Linear(cuda_device, ones) as plan:
        y = plan.forward_quantized(QuantizedRowsFP8(values.view(torch.float8_e4m3fn)[:, :k], torch.ones((rows, -(-k // 128)), device="cuda")))
        assert (y == k).all()


@pytest.mark.parametrize("rows", [20, 300])
def test_a_nan_row_stays_alone(cuda_device, rows) -> None:
    weight = blocks(cuda_device, 300, 600)
    x = draw((rows, 600), seed=2)
    damaged = x.clone()
    damaged[7, 130] = float("nan")
    damaged[11, 0] = float("inf")
    with PreparedFP8Linear(cuda_device, weight) as plan:
        clean, y = plan.forward(x), plan.forward(damaged)
    assert y[[7, 11]].isnan().all()
    others = [r for r in range(rows) if r not in (7, 11)]
    assert torch.equal(y[others], clean[others])


def test_extreme_scales(cuda_device) -> None:
    """Row and weight groups of very different magnitudes, and zero blocks."""
    x = draw((50, 512), seed=1) * torch.exp2(torch.linspace(-30, 30, 50, device="cuda"))[:, None]
    x[:, 128:256] = 0.0
    w = draw((256, 512), seed=2)
    w[:128, 256:384] *= 2.0**40
    w[128:, 384:] = 0.0
    weight = quantize_blocks_fp8(cuda_device, w)
    values, scales = ref.quantize_rows(x)
    exact, magnitude = ref.product(values, scales, weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        check_product(plan.forward(x), exact, magnitude, 512)


def test_empty_batch(cuda_device) -> None:
    with PreparedFP8Linear(cuda_device, blocks(cuda_device, 64, 128)) as plan:
        assert plan.forward(draw((0, 128))).shape == (0, 64)
    assert quantize_rows_fp8(cuda_device, draw((0, 128))).values.shape == (0, 128)


def expert_case(device, counts, n, k, trailing=0, seed=0, dtype=torch.bfloat16):
    weight = blocks(device, n, k, experts=len(counts), seed=seed + 1)
    rows = sum(counts) + trailing
    x = draw((rows, k), dtype, seed=seed)
    offsets = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device="cuda")
    values, scales = ref.quantize_rows(x)
    exact, magnitude = (torch.zeros((rows, n), dtype=torch.float64, device="cuda") for _ in range(2))
    begin = 0
    for e, count in enumerate(counts):
        part = slice(begin, begin + count)
        exact[part], magnitude[part] = ref.product(values[part], scales[part], weight.values[e], weight.scales[e])
        begin += count
    return weight, x, offsets, exact, magnitude


@pytest.mark.parametrize(
    "counts, trailing",
    [
        ([1], 0), ([0, 0, 5, 0], 0), ([3, 0, 1, 17, 16, 0, 2], 0), ([1] * 70, 0), ([0] * 40 + [2] + [0] * 60, 3), ([130, 0, 1, 255, 40], 9),
        ([0, 0], 20), ([600, 1, 0, 3], 0), ([300, 513, 128, 256], 1), ([31] * 33, 5), ([1000, 0, 1200], 2),
    ],
)
@pytest.mark.parametrize("n, k", [(256, 256), (200, 333)])
def test_experts(cuda_device, counts, trailing, n, k) -> None:
    weight, x, offsets, exact, magnitude = expert_case(cuda_device, counts, n, k, trailing)
    with PreparedFP8Experts(cuda_device, weight) as plan:
        check_product(plan.forward(x, offsets), exact, magnitude, k)
        out = torch.full((x.shape[0] + 2, n), 9.0, device="cuda")
        plan.forward(x, offsets, out=out[1:-1])
        check_product(out[1:-1], exact, magnitude, k)
        assert (out[[0, -1]] == 9.0).all()


@pytest.mark.parametrize("rows", [10, 700])
def test_offsets_beyond_the_rows_are_clamped(cuda_device, rows) -> None:
    weight = blocks(cuda_device, 128, 128, experts=4)
    x = draw((rows, 128), seed=1)
    with PreparedFP8Experts(cuda_device, weight) as plan:
        inside = torch.tensor([0, 4, rows, rows, rows], dtype=torch.int32, device="cuda")
        beyond = torch.tensor([-3, 4, rows + 100, 2**31 - 1, 2**31 - 1], dtype=torch.int32, device="cuda")
        assert torch.equal(plan.forward(x, inside), plan.forward(x, beyond))


@pytest.mark.parametrize("rows", [40, 900])
def test_offsets_out_of_order_stay_inside_the_output(cuda_device, rows) -> None:
    """Overlapping ranges leave rows unspecified; nothing outside the output is written and the call ends."""
    weight = blocks(cuda_device, 200, 2048, experts=4)
    x = draw((rows, 2048), seed=1)
    wide = torch.full((rows + 2, 208), 7.0, device="cuda")
    offsets = torch.tensor([0, rows, rows // 4, 2 * rows, 0], dtype=torch.int32, device="cuda")
    with PreparedFP8Experts(cuda_device, weight) as plan:
        plan.forward(x, offsets, out=wide[1:-1, 8:])
        torch.cuda.synchronize()
    assert (wide[[0, -1]] == 7.0).all() and (wide[:, :8] == 7.0).all()


def test_experts_nan_rows_do_not_reach_a_neighbouring_expert(cuda_device) -> None:
    weight, x, offsets, exact, magnitude = expert_case(cuda_device, [5, 4, 6], 256, 256)
    x[5:9] = float("nan")
    with PreparedFP8Experts(cuda_device, weight) as plan:
        y = plan.forward(x, offsets)
    assert y[5:9].isnan().all()
    check_product(y[:5], exact[:5], magnitude[:5], 256)
    check_product(y[9:], exact[9:], magnitude[9:], 256)


@pytest.mark.parametrize("rows", [4, 200, 2100])
def test_one_plan_on_two_streams_and_in_two_graphs(cuda_device, rows) -> None:
    weight = blocks(cuda_device, 1024, 1024)
    inputs = [draw((rows, 1024), torch.bfloat16, seed=s) for s in range(2)]
    with PreparedFP8Linear(cuda_device, weight) as plan:
        expected = [plan.forward(x) for x in inputs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        results: list[list[torch.Tensor]] = [[], []]
        for _ in range(20):
            for s, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    results[s].append(plan.forward(inputs[s]))
        torch.cuda.synchronize()
        for s in range(2):
            assert all(torch.equal(y, expected[s]) for y in results[s])
        graphs, outputs = [], []
        for x in inputs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs.append(plan.forward(x))
            graphs.append(graph)
        for x in inputs:
            x.mul_(-2.0)
        expected = [plan.forward(x) for x in inputs]
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, e) for y, e in zip(outputs, expected))


def test_execute_on_a_queue(cuda_device) -> None:
    weight = blocks(cuda_device, 96, 160)
    x = np.random.default_rng(0).standard_normal((5, 160), dtype=np.float32)
    with PreparedFP8Linear(cuda_device, weight) as plan, cuda_device.queue() as queue:
        source, destination = cuda_device.tensor((5, 160), np.float32), cuda_device.tensor((5, 96), np.float32)
        source.write(x)
        plan.execute(destination, source, queue=queue).wait()
        np.testing.assert_array_equal(destination.numpy(), plan.forward(torch.from_numpy(x).cuda()).cpu().numpy())


def test_close_waits_for_queued_executions(cuda_device) -> None:
    weight = blocks(cuda_device, 96, 160)
    x = np.random.default_rng(1).standard_normal((5, 160), dtype=np.float32)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        expected = plan.forward(torch.from_numpy(x).cuda()).cpu().numpy()
    with cuda_device.queue() as queue:
        source, destination = cuda_device.tensor((5, 160), np.float32), cuda_device.tensor((5, 96), np.float32)
        source.write(x)
        plan = PreparedFP8Linear(cuda_device, weight)
        events = [queue.host_task(lambda: time.sleep(0.05)), *(plan.execute(destination, source, queue=queue) for _ in range(3))]
        plan.close()
        assert all(event.done for event in events)
        np.testing.assert_array_equal(destination.numpy(), expected)


@pytest.mark.parametrize("rows", [1, 4, 40, 600])
def test_source_and_output_in_one_buffer(cuda_device, rows) -> None:
    """Column ranges that do not meet give what separate tensors give; an output over its source is refused."""
    n = k = 256
    weight = blocks(cuda_device, n, k)
    both = draw((rows, k + n), torch.bfloat16)
    source = both[:, :k].clone()
    with PreparedFP8Linear(cuda_device, weight) as plan:
        expected = plan.forward(source)
        with pytest.raises(ValueError, match="overlap"):
            plan.forward(source, out=source)
        plan.forward(both[:, :k], out=both[:, k:])
        torch.testing.assert_close(both, torch.cat((source, expected), 1), rtol=0, atol=0)
    with PreparedFP8Experts(cuda_device, blocks(cuda_device, n, k, experts=2)) as plan:
        with pytest.raises(ValueError, match="overlap"):
            plan.forward(source, torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda"), out=source)


def test_execute_refuses_an_output_over_its_source(cuda_device) -> None:
    with cuda_device.queue() as queue, PreparedFP8Linear(cuda_device, blocks(cuda_device, 64, 64)) as plan:
        source = cuda_device.tensor((5, 64), np.float32)
        with pytest.raises(ValueError, match="overlap"):
            plan.execute(source, source, queue=queue)


@pytest.mark.parametrize("n", [8192, 8191])
def test_rows_beyond_32_bit_offsets(cuda_device, n) -> None:
    """2.2e9 outputs, of the copy engine and of the warps: the last rows lie past 2^31 elements."""
    rows, k = 270_000, 256
    weight = blocks(cuda_device, n, k)
    x = draw((rows, k), torch.bfloat16)
    picked = torch.cat([torch.arange(150), torch.arange(131_000, 131_300), torch.arange(rows - 301, rows)]).cuda()
    exact, magnitude = ref.product(*ref.quantize_rows(x[picked]), weight.values, weight.scales)
    with PreparedFP8Linear(cuda_device, weight) as plan:
        y = plan.forward(x)
        check_product(y[picked], exact, magnitude, k)
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("gated", [False, True])
def test_row_quantizer_beyond_32_bit_offsets(cuda_device, gated) -> None:
    rows, cols = 270_000, 8192
    tile = draw((250, cols), torch.bfloat16, seed=4)
    quantized = quantize_rows_fp8(cuda_device, tile.repeat(rows // 250, 1), gated=gated)
    expected = quantize_rows_fp8(cuda_device, tile, gated=gated)
    if not gated:
        check_rows(expected, tile)
    width = expected.shape[1]
    assert torch.equal(quantized.values.view(torch.uint8).view(-1, 250, width), expected.values.view(torch.uint8).expand(rows // 250, -1, -1))
    assert torch.equal(quantized.scales.view(-1, 250, width // 128), expected.scales.expand(rows // 250, -1, -1))
    del quantized
    torch.cuda.empty_cache()


def test_weight_beyond_32_bit_offsets(cuda_device) -> None:
    """4.6e9 bytes of weight, one matrix and one of three: both kernels, the last columns."""
    for shape in ((70_000, 65_536), (3, 24_000, 65_536)):
        tile = draw((250, 65_536), torch.bfloat16, seed=5, std=0.05)
        full = tile.repeat(shape[-2] * (shape[0] if len(shape) == 3 else 1) // 250, 1).view(shape)
        weight = quantize_blocks_fp8(cuda_device, full)
        del full
        last = slice(shape[-2] - 300 - shape[-2] % 128, shape[-2])
        last = slice(last.start // 128 * 128, last.stop)
        matrix, scales = (weight.values, weight.scales) if len(shape) == 2 else (weight.values[-1], weight.scales[-1])
        for rows in (3, 100):
            x = draw((rows, shape[-1]), torch.bfloat16, seed=rows)
            exact, magnitude = ref.product(*ref.quantize_rows(x), matrix[last], scales[last.start // 128 :])
            if len(shape) == 2:
                with PreparedFP8Linear(cuda_device, weight) as plan:
                    y = plan.forward(x)
            else:
                offsets = torch.tensor([0, 0, 0, rows], dtype=torch.int32, device="cuda")
                with PreparedFP8Experts(cuda_device, weight) as plan:
                    y = plan.forward(x, offsets)
            check_product(y[:, last], exact, magnitude, shape[-1])
        check_tile = ref.quantize_blocks(torch.cat([tile, tile, tile])[last.start % 250 :][:128])
        assert torch.equal(matrix[last][:128].double(), check_tile[0])
        del weight, matrix, scales, plan, y
        torch.cuda.empty_cache()


def test_one_plan_in_two_threads(cuda_device) -> None:
    """Calls at once from threads with a stream each, beside executions on a queue."""
    weight = blocks(cuda_device, 640, 1024)
    inputs = [draw((rows, 1024), seed=rows) for rows in (3, 200)]
    results: list[list[torch.Tensor]] = [[], []]
    with PreparedFP8Linear(cuda_device, weight) as plan, cuda_device.queue() as queue:
        expected = [plan.forward(x) for x in inputs]
        torch.cuda.synchronize()

        def call(i: int) -> None:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    results[i].append(plan.forward(inputs[i]))

        threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
        source, destination = cuda_device.tensor((3, 1024), np.float32), cuda_device.tensor((3, 640), np.float32)
        source.write(inputs[0].cpu().numpy())
        for thread in threads:
            thread.start()
        for _ in range(20):
            plan.execute(destination, source, queue=queue)
        for thread in threads:
            thread.join()
        torch.cuda.synchronize()
        queue.finish()
        np.testing.assert_array_equal(destination.numpy(), expected[0].cpu().numpy())
    for got, want in zip(results, expected):
        assert len(got) == 50 and all(torch.equal(y, want) for y in got)


def test_results_repeat_bit_for_bit(cuda_device) -> None:
    for rows, n, k in ((1, 2048, 2048), (50, 640, 4096), (400, 1000, 1500), (1024, 6000, 512)):
        weight = blocks(cuda_device, n, k)
        x = draw((rows, k), seed=rows)
        with PreparedFP8Linear(cuda_device, weight) as plan:
            first = plan.forward(x)
            assert all(torch.equal(plan.forward(x), first) for _ in range(5))


def test_refusals_on_the_gpu(cuda_device) -> None:
    weight = blocks(cuda_device, 64, 128)
    x = draw((4, 128))
    with PreparedFP8Linear(cuda_device, weight) as plan:
        for bad in (x.double(), x[:, :127], x[0], x.cpu(), x.t().contiguous().t(), x[:1].expand(4, 128)):
            with pytest.raises(ValueError):
                plan.forward(bad)
        for out in (torch.empty((4, 63), device="cuda"), torch.empty((4, 64)), torch.empty((64, 4), device="cuda").t(), torch.empty((4, 64), dtype=torch.float64, device="cuda")):
            with pytest.raises(ValueError):
                plan.forward(x, out=out)
        with pytest.raises(ValueError, match="16-byte"):
            plan.forward_quantized(QuantizedRowsFP8(torch.empty((4, 132), dtype=torch.float8_e4m3fn, device="cuda")[:, :128], torch.ones((4, 1), device="cuda")))
        with pytest.raises(ValueError, match="requires grad"):
            plan.forward(x.clone().requires_grad_())
        with torch.no_grad():
            assert torch.equal(plan.forward(x.clone().requires_grad_()), plan.forward(x))
    with pytest.raises(RuntimeError, match="closed"):
        plan.forward(x)
    with PreparedFP8Experts(cuda_device, blocks(cuda_device, 64, 128, experts=2)) as plan:
        for offsets in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32)):
            with pytest.raises(ValueError, match="offsets"):
                plan.forward(x, offsets)
