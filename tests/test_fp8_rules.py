"""Host-side rules of the FP8 plans and the expert routing: argument checks that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from qpu_xla import Device, _native
from qpu_xla.experts import ExpertOrder, FP8ExpertsFFN, gather_tokens, sort_tokens
from qpu_xla.fp8 import (
    PreparedFP8Experts,
    PreparedFP8Linear,
    QuantizedBlocksFP8,
    QuantizedRowsFP8,
    check_apart,
    check_matrix,
    quantize_blocks_fp8,
    quantize_rows_fp8,
)

E4M3 = torch.float8_e4m3fn


def weight(*shape: int) -> QuantizedBlocksFP8:
    *batch, n, k = shape
    return QuantizedBlocksFP8(torch.zeros(shape, dtype=E4M3), torch.ones((*batch, -(-n // 128), -(-k // 128))))


def test_quantized_containers_check_their_shapes_and_types() -> None:
    assert weight(130, 300).shape == (130, 300)
    assert weight(3, 130, 300).dequantize().shape == (3, 130, 300)
    for values, scales in (
        (torch.zeros((130, 300), dtype=E4M3), torch.ones((1, 3))),
        (torch.zeros((130, 300), dtype=E4M3), torch.ones((2, 3), dtype=torch.float64)),
        (torch.zeros((130, 300), dtype=torch.uint8), torch.ones((2, 3))),
        (torch.zeros((300,), dtype=E4M3), torch.ones((3,))),
        (torch.zeros((2, 130, 300), dtype=E4M3), torch.ones((2, 3))),
        (torch.zeros((0, 300), dtype=E4M3), torch.ones((0, 3))),
    ):
        with pytest.raises(ValueError):
            QuantizedBlocksFP8(values, scales)
    with pytest.raises(ValueError, match="one float32 scale"):
        QuantizedRowsFP8(torch.zeros((2, 300), dtype=E4M3), torch.ones((2, 2)))
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        QuantizedRowsFP8(torch.zeros((2, 300)), torch.ones((2, 3)))


def test_dequantization_spreads_each_scale_over_its_group() -> None:
    rows = QuantizedRowsFP8(torch.ones((2, 130)).to(E4M3), torch.tensor([[2.0, 3.0], [4.0, 5.0]]))
    assert rows.dequantize()[0, 127:130].tolist() == [2.0, 3.0, 3.0]
    blocks = QuantizedBlocksFP8(torch.ones((129, 129)).to(E4M3), torch.tensor([[2.0, 3.0], [4.0, 5.0]]))
    assert blocks.dequantize()[127:129, 127:129].tolist() == [[2.0, 3.0], [4.0, 5.0]]


def test_calls_need_the_cuda_backend() -> None:
    with Device.fake() as device:
        for call in (
            lambda: quantize_rows_fp8(device, torch.zeros((2, 8))),
            lambda: quantize_blocks_fp8(device, torch.zeros((2, 8))),
            lambda: PreparedFP8Linear(device, weight(8, 8)),
            lambda: PreparedFP8Experts(device, weight(2, 8, 8)),
            lambda: sort_tokens(device, torch.zeros((2, 2), dtype=torch.int32), 2),
        ):
            with pytest.raises(ValueError, match="CUDA backend"):
                call()


def test_plans_check_the_weight_rank_before_the_device() -> None:
    with Device.fake() as device:
        with pytest.raises(ValueError, match="rank-2"):
            PreparedFP8Linear(device, weight(2, 8, 8))
        with pytest.raises(ValueError, match="rank-3"):
            PreparedFP8Experts(device, weight(8, 8))
        with pytest.raises(ValueError, match="at most 1024"):
            PreparedFP8Experts(device, weight(1025, 1, 1))
        with pytest.raises(ValueError, match="gate_up"):
            FP8ExpertsFFN(device, weight(2, 24, 8), weight(2, 8, 10))


def test_expert_order_checks_its_tensors() -> None:
    offsets, source, position = (torch.zeros(s, dtype=torch.int32) for s in (3, 8, (4, 2)))
    order = ExpertOrder(offsets, source, position)
    assert (order.experts, order.tokens, order.choices, order.rows) == (2, 4, 2, 8)
    for fields in ((offsets.long(), source, position), (offsets, source[:7], position), (offsets[:1], source, position), (offsets, source, position.t())):
        with pytest.raises(ValueError):
            ExpertOrder(*fields)
    with pytest.raises(ValueError, match="CUDA backend"), Device.fake() as device:
        gather_tokens(device, torch.zeros((4, 3)), order)


def test_null_arguments_are_rejected_without_a_device() -> None:
    library = _native.load()
    assert library.qpucuda_fp8_quantize_rows(None, ctypes.byref(_native.Fp8QuantizeDesc())) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_fp8_gemm(None, ctypes.byref(_native.Fp8GemmDesc())) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_fp8_quantize_blocks(None, None, 0, 0, 0, 0, 0, None, 0, None) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_expert_sort(None, ctypes.byref(_native.ExpertSortDesc())) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_expert_gather(None, ctypes.byref(_native.ExpertRowsDesc())) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_expert_combine(None, ctypes.byref(_native.ExpertRowsDesc())) == _native.Status.INVALID_ARGUMENT
    assert library.qpucuda_expert_combine_backward(None, ctypes.byref(_native.ExpertRowsDesc())) == _native.Status.INVALID_ARGUMENT


def test_sort_workspace_is_only_needed_past_one_cluster() -> None:
    size = _native.load().qpucuda_expert_sort_workspace
    assert size(1, 1, 1) == 0 and size(4096, 8, 64) == 0
    assert size(4097, 8, 64) > 0 and size(4097, 8, 64) % (4 * 64) == 0
    assert size(0, 8, 64) == 0 and size(8, 0, 64) == 0 and size(8, 8, 1025) == 0
    assert size(2**31, 2, 4) == 0


@pytest.mark.parametrize("structure", [_native.Fp8QuantizeDesc, _native.Fp8GemmDesc, _native.ExpertSortDesc, _native.ExpertRowsDesc])
def test_packed_descriptions_are_the_structures(structure) -> None:
    values = [i + 1 for i in range(len(structure._fields_))]
    assert _native.packer(structure)(*values) == bytes(structure(*values))


def test_matrices_have_31_bit_extents() -> None:
    meta = torch.device("meta")
    for shape in ((2**31, 1), (1, 2**31)):
        with pytest.raises(ValueError, match="2\\*\\*31"):
            check_matrix(torch.empty(shape, device=meta), meta, "x")
    assert check_matrix(torch.empty((2**31 - 1, 2), device=meta), meta, "x") == (2**31 - 1, 2, 2)


def meets_by_bytes(one: torch.Tensor, other: torch.Tensor) -> bool:
    def touched(t: torch.Tensor) -> set[int]:
        size = t.element_size()
        return {
            t.data_ptr() + r * t.stride(0) * size + c for r in range(t.shape[0]) for c in range(t.shape[1] * size)
        }

    return bool(touched(one) & touched(other))


def apart(out: torch.Tensor, read: torch.Tensor, what: str) -> None:
    strides = (check_matrix(t, t.device, "matrix")[2] for t in (out, read))
    check_apart(out, next(strides), read, next(strides), what)


def test_outputs_may_share_a_buffer_with_the_source_but_no_bytes() -> None:
    flat = torch.zeros(400)
    for rows in (1, 2, 5):
        for stride in (7, 12):
            for begin in range(0, 90, 3):
                for width in (1, 4, 7):
                    one = flat.as_strided((rows, width), (stride, 1), begin)
                    other = flat.as_strided((3, 5), (stride, 1), 30)
                    if meets_by_bytes(one, other):
                        with pytest.raises(ValueError, match="overlap"):
                            apart(one, other, "out")
                    else:
                        apart(one, other, "out")
    both = flat.as_strided((6, 12), (12, 1))
    apart(both[:, 5:], both[:, :5], "out")
    apart(both[:, :5], both[:, 5:], "out")
    apart(both[1:3, 5:], both[:, :5], "out")
    for out, source in ((both, both), (both[:, 4:], both[:, :5]), (both[:, :5], both[3:, 4:9]), (both.view(torch.bfloat16)[:, 8:], both[:, :5])):
        with pytest.raises(ValueError, match="overlap"):
            apart(out, source, "out")
    apart(both.view(torch.bfloat16)[:, 10:], both[:, :5], "out")
    apart(both[:0], both, "out")
