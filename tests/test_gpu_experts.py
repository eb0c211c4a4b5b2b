"""Expert routing on the GPU: the sort exactly, the rows' copies exactly, the weighted sums and the
gradients against float64."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
from qpu_xla.experts import (
    ExpertOrder,
    FP8ExpertsFFN,
    combine_tokens,
    combine_tokens_backward,
    gather_tokens,
    gather_tokens_backward,
    sort_tokens,
)
from qpu_xla.fp8 import PreparedFP8Experts, quantize_blocks_fp8, quantize_rows_fp8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# tokens, choices, experts: one of each, more experts than a warp, several chunks of the sort in one cluster
# (the largest: 4096 x 8) and in a grid, one expert
ROUTINGS = [(1, 1, 1), (5, 2, 3), (8, 8, 64), (100, 3, 7), (33, 1, 1024), (1000, 8, 256), (3000, 4, 40), (40000, 2, 1), (2048, 2, 8), (4096, 8, 1024), (4097, 8, 1024), (70000, 8, 100)]


def draw(shape, dtype=torch.float32, seed=0) -> torch.Tensor:
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def draw_ids(tokens: int, choices: int, experts: int, seed: int = 0, dropped: bool = True, dtype=torch.int32) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    low, high = (-1, experts + 2) if dropped else (0, experts)
    return torch.randint(low, high, (tokens, choices), generator=g, device="cuda", dtype=dtype)


def check_order(order: ExpertOrder, ids: torch.Tensor, experts: int) -> None:
    for have, want in zip((order.offsets, order.source, order.position), ref.sort(ids, experts)):
        assert torch.equal(have.cpu(), want)


def picked(rows: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
    """float64 [tokens, choices, width], zero where dropped."""
    kept = position >= 0
    out = torch.zeros((*position.shape, rows.shape[1]), dtype=torch.float64, device=rows.device)
    out[kept] = rows.double()[position[kept].long()]
    return out


@pytest.mark.parametrize("tokens, choices, experts", ROUTINGS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(cuda_device, tokens, choices, experts, dtype) -> None:
    for dropped in (False, True):
        ids = draw_ids(tokens, choices, experts, seed=tokens, dropped=dropped, dtype=dtype)
        check_order(sort_tokens(cuda_device, ids, experts), ids, experts)


def test_sort_of_lopsided_and_extreme_ids(cuda_device) -> None:
    for ids, experts in (
        (torch.full((9000, 2), 3), 5),
        (torch.full((300, 2), -1), 5),
        (torch.full((300, 2), 2**31 - 1), 1024),
        (torch.tensor([[-(2**31)], [0], [2**31 - 1]]), 2),
        (torch.arange(20000).view(-1, 4) % 7, 7),
        (torch.arange(20000).flip(0).view(-1, 4) // 3000, 7),
    ):
        ids = ids.to(torch.int32).cuda()
        check_order(sort_tokens(cuda_device, ids, experts), ids, experts)
    wide = torch.tensor([[2**32], [1], [-(2**40)]], device="cuda")
    check_order(sort_tokens(cuda_device, wide, 2), wide, 2)


def test_sort_of_no_tokens(cuda_device) -> None:
    order = sort_tokens(cuda_device, torch.empty((0, 4), dtype=torch.int32, device="cuda"), 6)
    assert order.offsets.tolist() == [0] * 7 and order.source.numel() == 0
    assert gather_tokens(cuda_device, torch.empty((0, 8), device="cuda"), order).shape == (0, 8)
    assert combine_tokens(cuda_device, torch.empty((0, 8), device="cuda"), torch.empty((0, 4), device="cuda"), order).shape == (0, 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, choices, experts", [(1, 1, 1), (7, 2, 3), (8, 8, 64), (300, 5, 16), (2500, 4, 8)])
@pytest.mark.parametrize("width", [1, 8, 200, 1027])
def test_gather_combine_and_their_gradients(cuda_device, dtype, tokens, choices, experts, width) -> None:
    """Copies and products with a power of two are exact. A sum of j fp32 terms rounds at most once
    per term (an fma each), 2^-24 of the magnitudes; the result once more to its type. A dot product
    of `width` terms, summed per thread and then over the CTA, rounds at most width times."""
    ids = draw_ids(tokens, choices, experts, seed=width)
    order = sort_tokens(cuda_device, ids, experts)
    position, kept = order.position.long(), order.position >= 0
    count = int(order.offsets[-1])
    x = draw((tokens, width), dtype, seed=1)
    rows = gather_tokens(cuda_device, x, order)
    assert torch.equal(rows[position[kept]], x[:, None].expand(-1, choices, -1)[kept])
    assert (rows[count:] == 0).all()
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * 2.0**-8

    grad_rows = draw((tokens * choices, width), dtype, seed=2)
    grad_rows[count:] = float("nan")
    each = picked(grad_rows, order.position)
    exact, magnitude = each.sum(1), each.abs().sum(1)
    grad_x = gather_tokens_backward(cuda_device, grad_rows, order)
    fp32 = choices * 2.0**-24 * magnitude
    assert ((grad_x.double() - exact).abs() <= fp32 + half * (exact.abs() + fp32) + tiny).all()

    weights = torch.rand((tokens, choices), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    weights[~kept] = float("nan")
    rows = draw((tokens * choices, width), dtype, seed=4)
    rows[count:] = float("nan")
    each = picked(rows, order.position) * torch.where(kept, weights, 0.0).double()[:, :, None]
    exact, magnitude = each.sum(1), each.abs().sum(1)
    out = combine_tokens(cuda_device, rows, weights, order)
    fp32 = choices * 2.0**-24 * magnitude
    assert ((out.double() - exact).abs() <= fp32 + half * (exact.abs() + fp32) + tiny).all()

    grad = draw((tokens, width), dtype, seed=5)
    grad_rows, grad_weights = combine_tokens_backward(cuda_device, rows, weights, grad, order)
    assert (grad_rows[count:] == 0).all()
    # weight * grad is rounded to fp32, then to the type
    exact = (weights.double()[:, :, None] * grad.double()[:, None])[kept]
    have = grad_rows.double()[position[kept]]
    assert ((have - exact).abs() <= (half + 2.0**-24 * (1 + half)) * exact.abs() + tiny).all()
    each = picked(rows, order.position) * grad.double()[:, None]
    assert (grad_weights[~kept] == 0).all()
    assert ((grad_weights.double() - each.sum(2)).abs() <= (width + 8) * 2.0**-24 * each.abs().sum(2) + 1e-38).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_rows(cuda_device, dtype) -> None:
    tokens, choices, experts, width = 50, 3, 6, 64
    order = sort_tokens(cuda_device, draw_ids(tokens, choices, experts), experts)
    weights = torch.rand((tokens, choices), device="cuda")
    for start in (0, 1, 2, 8):
        x = draw((tokens, width + 24), dtype, seed=start)[:, start : start + width]
        wide = torch.full((tokens * choices + 2, width + 24), 5.0, dtype=dtype, device="cuda")
        out = wide[1:-1, start : start + width]
        gather_tokens(cuda_device, x, order, out=out)
        assert torch.equal(out, gather_tokens(cuda_device, x.contiguous(), order))
        back = torch.full((tokens, width + 24), 5.0, dtype=dtype, device="cuda")
        combine_tokens(cuda_device, out, weights, order, out=back[:, start : start + width])
        assert torch.equal(back[:, start : start + width], combine_tokens(cuda_device, out.contiguous(), weights, order))
        grad_rows, grad_weights = combine_tokens_backward(cuda_device, out, weights, x, order)
        assert torch.equal(grad_rows, combine_tokens_backward(cuda_device, out.contiguous(), weights, x.contiguous(), order)[0])
        each = picked(out, order.position) * x.double()[:, None]
        assert ((grad_weights.double() - each.sum(2)).abs() <= (width + 8) * 2.0**-24 * each.abs().sum(2)).all()
        out.fill_(5.0)
        back.fill_(5.0)
        assert (wide == 5.0).all()


def test_gradients_against_differences(cuda_device) -> None:
    """combine is linear in the rows and in the weights, so a central difference along a direction is
    its derivative up to the fp32 sums: 300 x 64 products, each within (5 + 3) roundings."""
    tokens, choices, experts, width = 300, 4, 9, 64
    order = sort_tokens(cuda_device, draw_ids(tokens, choices, experts), experts)
    rows, grad = draw((tokens * choices, width), seed=1), draw((tokens, width), seed=2)
    weights = torch.rand((tokens, choices), device="cuda")
    grad_rows, grad_weights = combine_tokens_backward(cuda_device, rows, weights, grad, order)
    step_rows, step_weights = draw(rows.shape, seed=3), draw(weights.shape, seed=4)
    step_rows[int(order.offsets[-1]) :] = 0.0

    def along(d_rows, d_weights) -> tuple[float, float]:
        plus = combine_tokens(cuda_device, rows + d_rows, weights + d_weights, order).double()
        minus = combine_tokens(cuda_device, rows - d_rows, weights - d_weights, order).double()
        difference = (plus - minus) / 2 * grad.double()
        return difference.sum().item(), (plus.abs() + minus.abs()).mul(grad.double().abs()).sum().item()

    slope, magnitude = along(step_rows, 0.0)
    assert abs(slope - (grad_rows.double() * step_rows.double()).sum().item()) <= 8 * choices * 2.0**-24 * magnitude
    slope, magnitude = along(0.0, step_weights)
    assert abs(slope - (grad_weights.double() * step_weights.double()).sum().item()) <= (width + 8) * choices * 2.0**-24 * magnitude
    step_x = draw((tokens, width), seed=5)
    g = draw((tokens * choices, width), seed=6)
    forward = (gather_tokens(cuda_device, step_x, order).double() * g.double()).sum().item()
    backward = (gather_tokens_backward(cuda_device, g, order).double() * step_x.double()).sum().item()
    bound = choices * 2.0**-24 * (g.double().abs().sum() * step_x.double().abs().max()).item()
    assert abs(forward - backward) <= bound


def test_rows_beyond_32_bit_offsets(cuda_device) -> None:
    """2.2e9 elements: the last rows lie past 2^31 elements."""
    tokens, choices, width = 540_000, 2, 2048
    ids = (torch.arange(tokens * choices, device="cuda", dtype=torch.int32) % 3).view(tokens, choices)
    order = sort_tokens(cuda_device, ids, 3)
    x = torch.arange(tokens, device="cuda").remainder(251).to(torch.bfloat16)[:, None].expand(-1, width).contiguous()
    rows = gather_tokens(cuda_device, x, order)
    token = order.source.long() // choices
    assert torch.equal(rows[:, 0], x[token, 0]) and torch.equal(rows[:, -1], x[token, -1])
    weights = torch.full((tokens, choices), 0.5, device="cuda")
    out = combine_tokens(cuda_device, rows, weights, order)
    assert torch.equal(out[:, 0], x[:, 0]) and torch.equal(out[:, -1], x[:, -1])
    del rows, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens, choices, experts, width, inner", [(1, 2, 4, 256, 128), (9, 3, 8, 512, 384), (700, 2, 5, 384, 256)])
def test_expert_ffn_end_to_end(cuda_device, tokens, choices, experts, width, inner) -> None:
    """The layer is its steps, bit for bit, and each step is within its bound of float64 of what it was
    given: a second quantizer rounds to three bits what the product before it rounded to 24, so a
    value at a border may fall to either side and only the steps have a bound of their own."""
    ids = torch.stack([torch.randperm(experts)[:choices] for _ in range(tokens)]).to(torch.int32).cuda()
    ids[tokens // 2] = -1
    weights = torch.rand((tokens, choices), device="cuda")
    gate_up = quantize_blocks_fp8(cuda_device, draw((experts, 2 * inner, width), seed=1) * 0.05)
    down = quantize_blocks_fp8(cuda_device, draw((experts, width, inner), seed=2) * 0.05)
    source = draw((tokens, width), seed=3)
    with FP8ExpertsFFN(cuda_device, gate_up, down) as layer:
        out = layer.forward(source, ids, weights)
        order = sort_tokens(cuda_device, ids, experts)
        sorted_rows = gather_tokens(cuda_device, source, order)
        hidden = layer.gate_up.forward(sorted_rows, order.offsets)
        rows = layer.down.forward(hidden, order.offsets)
    assert torch.equal(out, combine_tokens(cuda_device, rows, weights, order))
    check_order(order, ids, experts)
    first = ref.quantize_rows(sorted_rows)
    second = quantize_rows_fp8(cuda_device, hidden, gated=True)
    bounds = order.offsets.tolist()
    assert bounds[-1] == (tokens - 1) * choices
    for e in range(experts):
        part = slice(bounds[e], bounds[e + 1])
        for have, (values, scales), weight in ((hidden, first, gate_up), (rows, (second.values, second.scales), down)):
            exact, magnitude = ref.product(values[part], scales[part], weight.values[e], weight.scales[e])
            error = (have[part].double() - exact).abs()
            assert (error <= ref.product_tolerance(exact, magnitude, weight.shape[2], torch.float32)).all()
    each = picked(rows, order.position) * weights.double()[:, :, None]
    assert ((out.double() - each.sum(1)).abs() <= (choices + 1) * 2.0**-24 * each.abs().sum(1)).all()
    assert (out[tokens // 2] == 0).all()


@pytest.mark.parametrize("tokens", [3, 400])
def test_tokens_straight_into_the_experts(cuda_device, tokens) -> None:
    """forward_tokens quantizes from the tokens what forward quantizes from their sorted copy."""
    order = sort_tokens(cuda_device, draw_ids(tokens, 3, 6), 6)
    x = draw((tokens, 300), torch.bfloat16)
    with PreparedFP8Experts(cuda_device, quantize_blocks_fp8(cuda_device, draw((6, 200, 300), seed=1))) as plan:
        assert torch.equal(plan.forward_tokens(x, order), plan.forward(gather_tokens(cuda_device, x, order), order.offsets))


def test_the_layer_in_a_graph_on_its_own_stream(cuda_device) -> None:
    tokens, choices, experts, width = 64, 2, 8, 256
    gate_up = quantize_blocks_fp8(cuda_device, draw((experts, 256, width), seed=1) * 0.05)
    down = quantize_blocks_fp8(cuda_device, draw((experts, width, 128), seed=2) * 0.05)
    ids, x = draw_ids(tokens, choices, experts), draw((tokens, width), torch.bfloat16)
    weights = torch.rand((tokens, choices), device="cuda")
    with FP8ExpertsFFN(cuda_device, gate_up, down) as layer:
        layer.forward(x, ids, weights)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.forward(x, ids, weights)
        for seed in (7, 8):
            ids.copy_(draw_ids(tokens, choices, experts, seed=seed))
            x.copy_(draw((tokens, width), torch.bfloat16, seed=seed))
            expected = layer.forward(x, ids, weights)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expected)


def test_refusals_on_the_gpu(cuda_device) -> None:
    ids = draw_ids(4, 2, 3)
    order = sort_tokens(cuda_device, ids, 3)
    x, weights = draw((4, 16)), torch.rand((4, 2), device="cuda")
    rows = gather_tokens(cuda_device, x, order)
    for call in (
        lambda: sort_tokens(cuda_device, ids.float(), 3),
        lambda: sort_tokens(cuda_device, ids.cpu(), 3),
        lambda: sort_tokens(cuda_device, ids, 0),
        lambda: sort_tokens(cuda_device, ids, 1025),
        lambda: gather_tokens(cuda_device, x[:3], order),
        lambda: gather_tokens(cuda_device, x.double(), order),
        lambda: gather_tokens(cuda_device, rows[:4], order, out=rows),
        lambda: combine_tokens(cuda_device, rows, weights.half(), order),
        lambda: combine_tokens(cuda_device, rows, weights[:3], order),
        lambda: combine_tokens(cuda_device, rows[:7], weights, order),
        lambda: combine_tokens(cuda_device, rows, weights, order, out=rows[:4]),
        lambda: combine_tokens_backward(cuda_device, rows, weights, x.half(), order),
        lambda: combine_tokens_backward(cuda_device, rows, weights, x[:, :8], order),
        lambda: gather_tokens(cuda_device, x.clone().requires_grad_(), order),
        lambda: combine_tokens(cuda_device, rows, weights.clone().requires_grad_(), order),
    ):
        with pytest.raises(ValueError):
            call()
