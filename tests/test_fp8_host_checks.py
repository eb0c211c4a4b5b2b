"""What the FP8 plans and the expert routing check and report on the host, around a library that only records
its calls."""

from __future__ import annotations

import random
from contextlib import nullcontext
from types import SimpleNamespace
from typing import Any

import pytest
import torch

from qpu_xla.errors import EventTimeoutError, NativeError
from qpu_xla.experts import ExpertOrder, FP8ExpertsFFN, combine_tokens, gather_tokens, gather_tokens_backward
from qpu_xla.fp8 import PreparedFP8Experts, PreparedFP8Linear, QuantizedRowsFP8, check_apart_from, quantize_blocks_fp8

E4M3 = torch.float8_e4m3fn


class RecordingDevice:
    """A device whose tensors lie in host memory and whose library records the entry points called."""

    is_cuda = True
    closed = False

    def __init__(self) -> None:
        self.calls: list[str] = []
        self.backend = SimpleNamespace(
            torch_device=torch.device("cpu"), current_stream_handle=0, call=lambda name, args, stream: self.calls.append(name)
        )


def plan_of(cls: type, device: RecordingDevice, n: int, k: int, experts: int = 0) -> Any:
    """A plan without its weight's copies."""
    plan = object.__new__(cls)
    plan.device, plan._torch_device, plan._closed, plan.gated, plan._pending = device, torch.device("cpu"), False, False, []
    plan.output_count, plan.input_count, plan.experts, plan._source_columns = n, k, experts, k
    plan._groups, plan._padded = -(-k // 128), -(-k // 16) * 16
    plan._values_address = plan._scales_address = plan._bias_address = 0
    return plan


def order_of(tokens: int, choices: int, experts: int, buffer: torch.Tensor | None = None) -> ExpertOrder:
    """Tables that follow one another in ``buffer`` (int32)."""
    total = tokens * choices
    buffer = torch.zeros(experts + 1 + 2 * total, dtype=torch.int32) if buffer is None else buffer
    parts = buffer[: experts + 1 + 2 * total].split_with_sizes([experts + 1, total, total])
    return ExpertOrder(parts[0], parts[1], parts[2].view(tokens, choices))


def touched(tensor: torch.Tensor) -> set[int]:
    size, places = tensor.element_size(), [tensor.data_ptr()]
    for extent, step in zip(tensor.shape, tensor.stride()):
        places = [place + i * step * size for place in places for i in range(extent)]
    return {place + byte for place in places for byte in range(size)}


def test_an_output_shares_no_bytes_with_anything_a_call_reads() -> None:
    """Rows, columns (a transposed table) and ranges of one buffer: refused exactly where bytes meet, except that
    layouts of different strides may be refused for the ranges they span."""
    flat = torch.zeros(400)
    rng = random.Random(5)
    refused = accepted = 0
    for _ in range(4000):
        stride = rng.choice((7, 12))
        out = flat.as_strided((rng.randint(0, 5), rng.randint(1, 7)), (stride, 1), rng.randint(0, 200))
        other, start = rng.choice((7, 12)), rng.randint(0, 200)
        read = rng.choice((
            flat.as_strided((rng.randint(1, 4), rng.randint(1, 7)), (other, 1), start),
            flat.as_strided((rng.randint(1, 7), rng.randint(1, 4)), (1, other), start),
            flat.as_strided((rng.randint(0, 9),), (1,), start),
            flat.as_strided((rng.randint(1, 3), 2), (0, 3), start),
        ))
        meet = bool(touched(out) & touched(read))
        try:
            check_apart_from(out, stride, (read,), "out")
            assert not meet
            accepted += 1
        except ValueError as error:
            assert "overlap" in str(error)
            assert meet or (stride != other or read.stride(0) == 0) and out.numel() and read.numel()
            refused += 1
    assert refused > 200 and accepted > 200


def test_row_scales_are_not_overwritten() -> None:
    device = RecordingDevice()
    plan = plan_of(PreparedFP8Linear, device, n=4, k=256)
    both = torch.zeros((6, 6))  # columns 0 to 3 the output, 4 and 5 the scales
    rows = QuantizedRowsFP8(torch.zeros((6, 256), dtype=E4M3), both[:, 4:])
    plan.forward_quantized(rows, out=both[:, :4])
    for scales in (both[:, 3:5], both[:, :2], both.view(-1)[:12].view(2, 6).t()):
        with pytest.raises(ValueError, match="overlap"):
            plan.forward_quantized(QuantizedRowsFP8(rows.values, scales), out=both[:, :4])
    assert device.calls == ["qpucuda_fp8_gemm"]


def test_offsets_and_order_are_not_overwritten() -> None:
    device = RecordingDevice()
    plan = plan_of(PreparedFP8Experts, device, n=4, k=16, experts=3)
    buffer = torch.zeros(64, dtype=torch.int32)
    order = order_of(4, 2, 3, buffer[32:])  # offsets, source and position at 32, 36 and 44
    tokens = torch.zeros((4, 16))

    def out(begin: int) -> torch.Tensor:
        return buffer.view(torch.float32)[begin : begin + 32].view(8, 4)

    for begin in (1, 4, 5):  # the last entry ends inside the offsets
        with pytest.raises(ValueError, match="overlap"):
            plan.forward(torch.zeros((8, 16)), order.offsets, out=out(begin))
        with pytest.raises(ValueError, match="overlap"):
            plan.forward_tokens(tokens, order, out=out(begin))
    moved = ExpertOrder(torch.zeros(4, dtype=torch.int32), buffer[24:32], order.position)
    with pytest.raises(ValueError, match="overlap"):
        plan.forward_tokens(tokens, moved, out=out(0))
    plan.forward(torch.zeros((8, 16)), order.offsets, out=out(0))
    plan.forward_tokens(tokens, order, out=out(0))
    assert device.calls == ["qpucuda_fp8_linear"] * 2


def test_positions_and_routing_weights_are_not_overwritten() -> None:
    device = RecordingDevice()
    buffer = torch.zeros(96)
    order = order_of(4, 2, 3, buffer[64:].view(torch.int32))  # offsets at 64, source 68, position 76 to 83
    tokens, rows, weights = torch.zeros((4, 8)), torch.zeros((8, 8)), torch.zeros((4, 2))
    for begin in (1, 17, 31):
        with pytest.raises(ValueError, match="overlap"):
            gather_tokens(device, tokens, order, out=buffer[begin : begin + 64].view(8, 8))
    for begin in (45, 60, 64):
        out = buffer[begin : begin + 32].view(4, 8)
        with pytest.raises(ValueError, match="overlap"):
            combine_tokens(device, rows, weights, order, out=out)
        with pytest.raises(ValueError, match="overlap"):
            gather_tokens_backward(device, rows, order, out=out)
        with pytest.raises(ValueError, match="overlap"):
            combine_tokens(device, rows, out.reshape(-1)[3:11].view(4, 2), order_of(4, 2, 3), out=out)
    assert device.calls == []
    gather_tokens(device, tokens, order, out=buffer[:64].view(8, 8))
    combine_tokens(device, rows, weights, order, out=buffer[:32].view(4, 8))
    gather_tokens_backward(device, rows, order, out=buffer[40:72].view(4, 8))  # its offsets and source are not read
    assert device.calls == ["qpucuda_expert_gather", "qpucuda_expert_combine", "qpucuda_expert_combine"]


class FakeNative:
    """The library's context: its error word, read by ``synchronize``."""

    def __init__(self) -> None:
        self.expired = self.poisoned = False
        self.waits: list[Any] = []

    def synchronize(self) -> None:
        if self.poisoned:
            raise NativeError(5, "CUDA context is poisoned after a wait failure")
        if self.expired:
            self.poisoned = True
            raise EventTimeoutError("a kernel barrier wait exceeded its bound")


@pytest.fixture
def waiting_device(monkeypatch: pytest.MonkeyPatch) -> RecordingDevice:
    device, native = RecordingDevice(), FakeNative()

    def launch(stream: Any, fn: Any) -> Any:
        native.waits.append("error word")
        return fn(native)

    device.backend.native, device.backend.launch = native, launch
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: native.waits.append("device"))
    current = SimpleNamespace(synchronize=lambda: native.waits.append("stream"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: current)
    monkeypatch.setattr(torch.cuda, "device", lambda device: nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return device


def test_an_expired_wait_of_a_stream_call_is_raised(waiting_device: RecordingDevice) -> None:
    """The kernels end without a CUDA error, so the plan has to ask: on request, and when it closes."""
    native = waiting_device.backend.native
    with plan_of(PreparedFP8Linear, waiting_device, n=4, k=16) as plan:
        plan.synchronize()
        assert native.waits == ["stream", "error word"]
        native.expired = True
        with pytest.raises(EventTimeoutError, match="exceeded its bound"):
            plan.synchronize()
        with pytest.raises(NativeError, match="poisoned"):
            plan.close()
    assert native.waits[-2:] == ["device", "error word"]  # everything has ended before the error word is read
    with pytest.raises(RuntimeError, match="closed"):
        plan.synchronize()


def test_close_reports_an_expired_wait_and_releases_the_weight(waiting_device: RecordingDevice) -> None:
    waiting_device.backend.native.expired = True
    plan = plan_of(PreparedFP8Linear, waiting_device, n=4, k=16)
    plan._values = plan._scales = torch.zeros(1)
    with pytest.raises(EventTimeoutError):
        plan.close()
    assert plan._closed and plan._values is None and plan._scales is None
    plan.close()  # once


def test_close_after_the_device_asks_it_nothing(waiting_device: RecordingDevice) -> None:
    waiting_device.closed = True
    waiting_device.backend.native.expired = True
    plan_of(PreparedFP8Linear, waiting_device, n=4, k=16).close()


def test_the_layer_closes_both_plans_and_raises(waiting_device: RecordingDevice) -> None:
    layer = object.__new__(FP8ExpertsFFN)
    layer.device = waiting_device
    layer.gate_up, layer.down = (plan_of(PreparedFP8Experts, waiting_device, n=4, k=16, experts=2) for _ in range(2))
    layer.synchronize()
    waiting_device.backend.native.expired = True
    with pytest.raises(EventTimeoutError):
        layer.synchronize()
    with pytest.raises(NativeError):
        layer.close()
    assert layer.gate_up._closed and layer.down._closed


def test_no_wait_while_a_graph_is_captured(waiting_device: RecordingDevice, monkeypatch: pytest.MonkeyPatch) -> None:
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        plan_of(PreparedFP8Linear, waiting_device, n=4, k=16).synchronize()
    assert waiting_device.backend.native.waits == []


@pytest.mark.parametrize("shape", [(1, 2**32 + 1), (2**31, 1), (2, 2**31, 1), (2**16, 1, 1)])
def test_weights_past_the_quantizers_extents_are_refused(shape: tuple[int, ...]) -> None:
    """A C extent has 32 bits (2**32 + 1 columns would pass as one), a grid 65535 matrices."""
    device = RecordingDevice()
    device.backend.torch_device = torch.device("meta")
    with pytest.raises(ValueError, match="fewer than"):
        quantize_blocks_fp8(device, torch.empty(shape, dtype=torch.float16, device="meta"))
    assert device.calls == []
