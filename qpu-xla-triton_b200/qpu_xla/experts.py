"""Tokens sorted by expert and back, and an FFN of FP8 experts, on CUDA.

Each token t makes ``choices`` choices of an expert; choice (t, j) has the flat
index ``t * choices + j``. Rows are ordered by expert, then by flat index; an id
outside ``[0, experts)`` drops the choice (a padding token). No counterpart in
the reference. The order and the sums never depend on timing: the sort counts
integers, a token's choices are added in their order, there are no atomics on
floating-point values.
An output that the caller gives shares no bytes with what the call reads (rows,
positions, offsets, weights); one that does is refused.

The functions run on the current stream of their device. There is no autograd:
each step's gradient is a function of its own (``gather_tokens_backward``,
``combine_tokens_backward``), and tensors that require grad are refused while
gradients are recorded (inside an ``autograd.Function`` they are not).
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Any, Self

import torch

from qpu_xla import _native
from qpu_xla.device import Device
from qpu_xla.fp8 import (
    MAX_EXPERTS,
    PreparedFP8Experts,
    QuantizedBlocksFP8,
    check_apart,
    check_apart_from,
    check_matrix,
    dtype_code,
    launch,
    made,
    new_matrix,
    require_cuda,
)


_pack_sort = _native.packer(_native.ExpertSortDesc)
_pack_rows = _native.packer(_native.ExpertRowsDesc)


@lru_cache(maxsize=256)
def _sort_workspace(tokens: int, choices: int, experts: int) -> int:
    return int(_native.load().qpucuda_expert_sort_workspace(tokens, choices, experts))


@dataclass(frozen=True, slots=True)
class ExpertOrder:
    """int32 CUDA tensors of one sort: ``offsets [experts + 1]`` (rows of expert e are ``offsets[e] ..
    offsets[e + 1]``), ``source [tokens * choices]`` (the flat index at each row, -1 from
    ``offsets[experts]`` on) and ``position [tokens, choices]`` (the row of each choice, -1 when
    dropped)."""

    offsets: Any
    source: Any
    position: Any

    def __post_init__(self: Self) -> None:
        fields = (self.offsets, self.source, self.position)
        if any(t.dtype != torch.int32 or not t.is_contiguous() for t in fields):
            raise ValueError("expert order tensors must be contiguous int32")
        if self.offsets.dim() != 1 or self.source.dim() != 1 or self.position.dim() != 2 or self.offsets.shape[0] < 2:
            raise ValueError("expert order needs offsets [experts + 1], source [rows] and position [tokens, choices]")
        if self.source.shape[0] != self.position.numel() or self.position.shape[1] == 0:
            raise ValueError("expert order needs one row per choice")
        if any(t.device != self.offsets.device for t in fields):
            raise ValueError("expert order tensors must be on one device")

    @property
    def experts(self: Self) -> int:
        return int(self.offsets.shape[0]) - 1

    @property
    def tokens(self: Self) -> int:
        return int(self.position.shape[0])

    @property
    def choices(self: Self) -> int:
        return int(self.position.shape[1])

    @property
    def rows(self: Self) -> int:
        return int(self.source.shape[0])

    def check(self: Self, torch_device: Any, *, tokens: int | None = None) -> None:
        if self.offsets.device != torch_device:
            raise ValueError(f"expert order must be on {torch_device}, the device it is used with")
        if tokens is not None and tokens != self.tokens:
            raise ValueError(f"expert order is of {self.tokens} tokens, not {tokens}")


def sort_tokens(device: Device, expert_ids: Any, experts: int) -> ExpertOrder:
    """Sort the choices ``[tokens, choices]`` (int32 or int64 expert ids) by expert, stably."""
    torch_device = require_cuda(device, "sort_tokens")
    if expert_ids.dtype not in (torch.int32, torch.int64) or expert_ids.dim() != 2 or expert_ids.shape[1] == 0:
        raise ValueError("sort_tokens requires int32 or int64 expert ids [tokens, choices]")
    if expert_ids.device != torch_device:
        raise ValueError(f"sort_tokens expert ids must be on {torch_device}")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"sort_tokens takes 1 to {MAX_EXPERTS} experts")
    if expert_ids.numel() >= 2**31:
        raise ValueError("sort_tokens takes fewer than 2**31 choices")
    ids = expert_ids.contiguous()
    tokens, choices = ids.shape
    total = tokens * choices
    # one allocation for the three tables
    offsets, source, position = torch.empty(experts + 1 + 2 * total, dtype=torch.int32, device=torch_device).split_with_sizes(
        [experts + 1, total, total]
    )
    needed = _sort_workspace(tokens, choices, experts)
    workspace = torch.empty(needed, dtype=torch.uint8, device=torch_device) if needed else None
    desc = _pack_sort(
        ids.data_ptr(), ids.dtype == torch.int64, tokens, choices, experts, offsets.data_ptr(), source.data_ptr(), position.data_ptr(),
        0 if workspace is None else workspace.data_ptr(), needed,
    )
    launch(device, "qpucuda_expert_sort", desc)
    return made(ExpertOrder, offsets=offsets, source=source, position=position.view(tokens, choices))


def _destination(
    out: Any, rows: int, width: int, read: Any, read_stride: int, reads: tuple[Any, ...], torch_device: Any, what: str
) -> tuple[Any, int]:
    """``out`` (or a new tensor) for rows of ``read``'s type, and its row stride."""
    if out is None:
        return new_matrix(rows, width, read.dtype, torch_device), max(width, 1)
    if out.dtype != read.dtype:
        raise ValueError(f"{what} must have the type of its source")
    stride = check_matrix(out, torch_device, what, rows, width)[2]
    check_apart(out, stride, read, read_stride, what)
    check_apart_from(out, stride, reads, what)
    return out, stride


def gather_tokens(device: Device, source: Any, order: ExpertOrder, out: Any = None) -> Any:
    """Tokens ``[T, H]`` (float32, bfloat16 or float16) copied into expert order, ``[T * choices, H]``:
    row ``order.position[t, j]`` is token t. Rows from ``offsets[experts]`` on become zero."""
    torch_device = require_cuda(device, "gather_tokens")
    code = dtype_code(source.dtype, "gather_tokens source")
    order.check(torch_device)
    tokens, choices = order.position.shape
    _, width, stride = check_matrix(source, torch_device, "gather_tokens source", tokens)
    reads = (order.position, order.offsets)
    out, out_stride = _destination(out, tokens * choices, width, source, stride, reads, torch_device, "gather_tokens out")
    if tokens and width:
        desc = _pack_rows(
            code, tokens, choices, width, order.experts, order.position.data_ptr(), order.offsets.data_ptr(), 0, source.data_ptr(), stride,
            0, 0, 0, out.data_ptr(), out_stride,
        )
        launch(device, "qpucuda_expert_gather", desc)
    return out


def _combine(device: Device, rows: Any, weights: Any, order: ExpertOrder, out: Any, torch_device: Any, name: str) -> Any:
    code = dtype_code(rows.dtype, name)
    order.check(torch_device)
    tokens, choices = order.position.shape
    _, width, stride = check_matrix(rows, torch_device, name, tokens * choices)
    reads = (order.position,) if weights is None else (order.position, weights)
    out, out_stride = _destination(out, tokens, width, rows, stride, reads, torch_device, name)
    if tokens and width:
        desc = _pack_rows(
            code, tokens, choices, width, order.experts, order.position.data_ptr(), 0, 0 if weights is None else weights.data_ptr(),
            rows.data_ptr(), stride, 0, 0, 0, out.data_ptr(), out_stride,
        )
        launch(device, "qpucuda_expert_combine", desc)
    return out


def _check_weights(weights: Any, order: ExpertOrder, torch_device: Any, name: str) -> None:
    if weights.dtype != torch.float32 or weights.shape != order.position.shape or not weights.is_contiguous():
        raise ValueError(f"{name} requires contiguous float32 weights [tokens, choices]")
    if weights.device != torch_device:
        raise ValueError(f"{name} weights must be on {torch_device}")
    if weights.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} weights require grad, and there is no autograd here")


def gather_tokens_backward(device: Device, grad_rows: Any, order: ExpertOrder, out: Any = None) -> Any:
    """The tokens' gradient ``[T, H]`` from the sorted rows' ``[T * choices, H]``: the sum over a
    token's choices in fp32, rounded once. Dropped choices add nothing."""
    return _combine(device, grad_rows, None, order, out, require_cuda(device, "gather_tokens_backward"), "gather_tokens_backward")


def combine_tokens(device: Device, rows: Any, weights: Any, order: ExpertOrder, out: Any = None) -> Any:
    """Sorted rows ``[T * choices, H]`` back to tokens: ``out[t] = sum_j weights[t, j] *
    rows[position[t, j]]`` in fp32, in the order of j, rounded once. A dropped choice adds nothing,
    whatever its weight."""
    torch_device = require_cuda(device, "combine_tokens")
    _check_weights(weights, order, torch_device, "combine_tokens")
    return _combine(device, rows, weights, order, out, torch_device, "combine_tokens")


def combine_tokens_backward(device: Device, rows: Any, weights: Any, grad: Any, order: ExpertOrder) -> tuple[Any, Any]:
    """The gradients of :func:`combine_tokens` from that of its result, ``grad [T, H]``: of the rows
    (``weights[t, j] * grad[t]`` at ``position[t, j]``, zero where no choice is) and of the weights
    (``<rows[position[t, j]], grad[t]>`` in fp32, zero where dropped)."""
    name = "combine_tokens_backward"
    torch_device = require_cuda(device, name)
    code = dtype_code(rows.dtype, name)
    if grad.dtype != rows.dtype:
        raise ValueError(f"{name} grad must have the type of the rows")
    order.check(torch_device)
    tokens, choices = order.position.shape
    _, width, stride = check_matrix(rows, torch_device, f"{name} rows", tokens * choices)
    grad_stride = check_matrix(grad, torch_device, f"{name} grad", tokens, width)[2]
    _check_weights(weights, order, torch_device, name)
    grad_rows = new_matrix(tokens * choices, width, rows.dtype, torch_device)
    grad_weights = new_matrix(tokens, choices, torch.float32, torch_device)
    if tokens and width:
        desc = _pack_rows(
            code, tokens, choices, width, order.experts, order.position.data_ptr(), order.offsets.data_ptr(), weights.data_ptr(),
            rows.data_ptr(), stride, grad.data_ptr(), grad_stride, grad_weights.data_ptr(), grad_rows.data_ptr(), width,
        )
        launch(device, "qpucuda_expert_combine_backward", desc)
    else:
        grad_weights.zero_()
    return grad_rows, grad_weights


class FP8ExpertsFFN:
    """A layer of experts: ``sum_j w[t, j] down_e(silu(gate_e(x_t)) * up_e(x_t))``, e = ids[t, j].

    ``gate_up`` ``[E, 2 I, H]`` stacks each expert's gate rows on its up rows, ``down`` is
    ``[E, H_out, I]``; both block-scaled e4m3. Per call: one sort, one quantization of the tokens in
    expert order, the gate/up product (kept in fp32), one gated quantization, the down product, the
    weighted sum.
    """

    def __init__(self: Self, device: Device, gate_up: QuantizedBlocksFP8, down: QuantizedBlocksFP8) -> None:
        if len(gate_up.shape) != 3 or len(down.shape) != 3 or gate_up.shape[0] != down.shape[0] or gate_up.shape[1] != 2 * down.shape[2]:
            raise ValueError("FP8ExpertsFFN requires gate_up [E, 2 * inner, inputs] and down [E, outputs, inner]")
        self.device = device
        self.gate_up = PreparedFP8Experts(device, gate_up)
        self.down = PreparedFP8Experts(device, down, gated=True)

    @property
    def experts(self: Self) -> int:
        return self.gate_up.experts

    def forward(self: Self, source: Any, expert_ids: Any, weights: Any) -> Any:
        """Tokens ``[T, H]``, their expert ids ``[T, choices]`` and float32 weights, to ``[T, H_out]``
        of the source's type."""
        order = sort_tokens(self.device, expert_ids, self.experts)
        hidden = self.gate_up.forward_tokens(source, order, dtype=torch.float32)
        rows = self.down.forward(hidden, order.offsets, dtype=source.dtype)
        return combine_tokens(self.device, rows, weights, order)

    def synchronize(self: Self) -> None:
        """Wait for the device's current stream and raise if a kernel's wait ran out (as a plan's ``synchronize``)."""
        self.gate_up.synchronize()

    def close(self: Self) -> None:
        """Close both plans (which wait for the device and raise what ``synchronize`` would)."""
        try:
            self.gate_up.close()
        finally:
            self.down.close()

    def __enter__(self: Self) -> Self:
        return self

    def __exit__(self: Self, exc_type: object, exc_value: object, traceback: object) -> None:
        self.close()


__all__ = [
    "ExpertOrder",
    "FP8ExpertsFFN",
    "combine_tokens",
    "combine_tokens_backward",
    "gather_tokens",
    "gather_tokens_backward",
    "sort_tokens",
]
