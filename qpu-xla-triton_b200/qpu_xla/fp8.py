"""Block-scaled FP8 (e4m3) linear plans on CUDA.

The W8A8 linear of :mod:`qpu_xla.quantization` for weights published as e4m3
values with one fp32 scale per 128 x 128 block; no counterpart in the reference.
Activation rows are quantized on the fly with one scale per 128 columns::

    s = max(RN(max|x| / 448), 2**-60)      q = e4m3(RN(x / s)), round to nearest even
    y[m, n] = sum_k (qx[m, k] sx[m, k // 128]) (qw[n, k] sw[n // 128, k // 128]) (+ bias[n])

summed in fp32 and rounded once to the output's type. A group of 128 columns
that holds a NaN or an infinity dequantizes to NaN, and so do that row's outputs.

An output that the caller gives may lie in a buffer with what the call reads
(source, scales, offsets), but one that shares bytes with it is refused.

Everything here runs on the current stream of the plan's device, allocates its
scratch from PyTorch per call (so calls on several streams, and several captured
CUDA graphs, share no workspace) and has no CPU path. There is no autograd: a
source that requires grad is refused while gradients are recorded.

The product's waits inside a kernel are bounded: one that runs out leaves outputs
unwritten or incomplete, records it on the device and ends without a CUDA error.
A plan's ``synchronize`` and ``close`` raise then, as a queue's event does;
results on a stream are certain once one of them has returned.
"""

from __future__ import annotations

from collections.abc import Iterable
from dataclasses import dataclass
from typing import Any, Self

import numpy as np
import torch

from qpu_xla import _native
from qpu_xla.device import Device
from qpu_xla.errors import DependencyError
from qpu_xla.kernel import Kernel
from qpu_xla.memory import AccessMode, Tensor
from qpu_xla.queue import Event, Queue

FP8_GROUP = 128
MAX_EXPERTS = 1024


_pack_quantize = _native.packer(_native.Fp8QuantizeDesc)
_pack_gemm = _native.packer(_native.Fp8GemmDesc)
_DTYPE_CODES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}


def dtype_code(dtype: Any, what: str) -> int:
    """``qpucuda_dtype`` of an activation or output type."""
    code = _DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16")
    return code


def groups_of(size: int) -> int:
    return (size + FP8_GROUP - 1) // FP8_GROUP


def require_cuda(device: Device, what: str) -> Any:
    """The torch device behind a CUDA ``Device``."""
    if not device.is_cuda:
        raise ValueError(f"{what} requires the CUDA backend (this build has no CPU path)")
    return device.backend.torch_device  # type: ignore[attr-defined]


def check_matrix(tensor: Any, torch_device: Any, what: str, rows: int | None = None, cols: int | None = None) -> tuple[int, int, int]:
    """A rank-2 tensor on ``torch_device`` with unit inner stride and the given extents: its rows,
    columns and row stride (a single row's stride is its width, whatever the tensor says)."""
    shape = tensor.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        raise ValueError(f"{what} must be [{'rows' if rows is None else rows}, {'columns' if cols is None else cols}], not {list(shape)}")
    if tensor.device != torch_device:
        raise ValueError(f"{what} must be on {torch_device}, the device it is used with")
    if tensor.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires grad, and there is no autograd here: call under torch.no_grad() or from an autograd.Function")
    have_rows, have_cols = shape
    if have_rows >= 2**31 or have_cols >= 2**31:
        raise ValueError(f"{what} must have fewer than 2**31 rows and columns")
    stride, inner = tensor.stride()
    if inner != 1 and have_cols > 1:
        raise ValueError(f"{what} must be row-major (unit inner stride)")
    if have_rows <= 1:
        return have_rows, have_cols, max(have_cols, 1)
    if stride < have_cols:
        raise ValueError(f"{what} must not have overlapping rows")
    return have_rows, have_cols, stride


def check_apart(out: Any, out_stride: int, read: Any, read_stride: int, what: str) -> None:
    """Refuse an ``out`` that shares bytes with the matrix the call reads (both with the row strides of
    :func:`check_matrix`): kernels read and write in no particular order. Column ranges of one buffer do
    not meet."""
    begin, read_begin = out.data_ptr(), read.data_ptr()
    size, read_size = out.element_size(), read.element_size()
    rows, cols = out.shape
    read_rows, read_cols = read.shape
    stride, read_stride = out_stride * size, read_stride * read_size
    if begin >= read_begin + read_rows * read_stride or read_begin >= begin + rows * stride:
        return
    if _meet((begin, rows, cols, stride, size), (read_begin, read_rows, read_cols, read_stride, read_size)):
        raise ValueError(f"{what} must not overlap its source")


def check_apart_from(out: Any, out_stride: int, reads: Iterable[Any], what: str) -> None:
    """Refuse an ``out`` that shares bytes with one of the other tensors the call reads (scales, offsets,
    positions, weights; rank 1 or 2)."""
    begin, size = out.data_ptr(), out.element_size()
    rows, cols = out.shape
    for read in reads:
        if _meet((begin, rows, cols, out_stride * size, size), _layout(read)):
            raise ValueError(f"{what} must not overlap what the call reads")


def _layout(tensor: Any) -> tuple[int, ...]:
    """A tensor as a row-major matrix for :func:`_meet`: its rows, its columns, or else the whole range of
    addresses it spans."""
    size, begin = tensor.element_size(), tensor.data_ptr()
    if tensor.dim() == 2 and not tensor.is_contiguous():
        (rows, cols), (stride, inner) = tensor.shape, tensor.stride()
        if inner == 1:
            return begin, rows, cols, stride * size, size
        if stride == 1:
            return begin, cols, rows, inner * size, size
    span = 0 if tensor.numel() == 0 else 1 + sum((extent - 1) * step for extent, step in zip(tensor.shape, tensor.stride()))
    return begin, 1, span, span * size, size


def _meet(one: tuple[int, ...], other: tuple[int, ...]) -> bool:
    """Whether two row-major matrices (address, rows, columns, row stride in bytes, element size) share
    bytes; of different row strides, whether their ranges of addresses do."""
    (begin, rows, cols, stride, size), (other_begin, other_rows, other_cols, other_stride, other_size) = one, other
    if 0 in (rows, cols, other_rows, other_cols):
        return False
    width, other_width = cols * size, other_cols * other_size
    if begin >= other_begin + (other_rows - 1) * other_stride + other_width or other_begin >= begin + (rows - 1) * stride + width:
        return False
    if rows == 1:
        stride = other_stride
    elif other_rows == 1:
        other_stride = stride
    if stride == other_stride and stride > 0:
        gap = (begin - other_begin) % stride
        return gap < other_width or gap + width > stride
    return True


def new_matrix(rows: int, cols: int, dtype: Any, torch_device: Any) -> Any:
    """An uninitialised row-major matrix (``empty_strided`` costs the host a third less than ``empty``)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=torch_device)


def launch(device: Device, name: str, *args: Any, stream: int | None = None) -> None:
    """Call one libqpucuda entry point on ``stream`` (a cudaStream_t; default: the device's current stream)."""
    backend = device.backend
    backend.call(name, args, backend.current_stream_handle if stream is None else stream)  # type: ignore[attr-defined]


def made(cls: type, **fields: Any) -> Any:
    """A frozen dataclass around tensors this package has just allocated, without its checks."""
    result = object.__new__(cls)
    for name, value in fields.items():
        object.__setattr__(result, name, value)
    return result


@dataclass(frozen=True, slots=True)
class QuantizedRowsFP8:
    """e4m3 rows ``[M, K]`` and their fp32 scales ``[M, ceil(K / 128)]`` (any strides)."""

    values: Any
    scales: Any

    def __post_init__(self: Self) -> None:
        if self.values.dim() != 2 or self.values.dtype != torch.float8_e4m3fn:
            raise ValueError("quantized rows must be rank-2 float8_e4m3fn")
        if tuple(self.scales.shape) != (self.values.shape[0], groups_of(self.values.shape[1])) or self.scales.dtype != torch.float32:
            raise ValueError("quantized rows need one float32 scale per row and 128 columns")
        if self.scales.device != self.values.device:
            raise ValueError("quantized rows and their scales must be on one device")

    @property
    def shape(self: Self) -> tuple[int, int]:
        return (int(self.values.shape[0]), int(self.values.shape[1]))

    def dequantize(self: Self) -> Any:
        """fp32 reconstruction ``[M, K]``."""
        spread = self.scales.repeat_interleave(FP8_GROUP, dim=1)[:, : self.values.shape[1]]
        return self.values.float() * spread


@dataclass(frozen=True, slots=True)
class QuantizedBlocksFP8:
    """e4m3 weights ``[N, K]`` with fp32 scales ``[ceil(N / 128), ceil(K / 128)]``, or one such matrix
    per expert (``[E, N, K]`` and ``[E, ceil(N / 128), ceil(K / 128)]``)."""

    values: Any
    scales: Any

    def __post_init__(self: Self) -> None:
        if self.values.dim() not in (2, 3) or self.values.dtype != torch.float8_e4m3fn or 0 in self.values.shape:
            raise ValueError("quantized weights must be non-empty rank-2 or rank-3 float8_e4m3fn")
        *batch, rows, cols = self.values.shape
        if tuple(self.scales.shape) != (*batch, groups_of(rows), groups_of(cols)) or self.scales.dtype != torch.float32:
            raise ValueError("quantized weights need one float32 scale per 128 x 128 block")
        if self.scales.device != self.values.device:
            raise ValueError("quantized weights and their scales must be on one device")

    @property
    def shape(self: Self) -> tuple[int, ...]:
        return tuple(int(extent) for extent in self.values.shape)

    def dequantize(self: Self) -> Any:
        """fp32 reconstruction, shaped as the values."""
        rows, cols = self.values.shape[-2:]
        spread = self.scales.repeat_interleave(FP8_GROUP, dim=-2)[..., :rows, :].repeat_interleave(FP8_GROUP, dim=-1)
        return self.values.float() * spread[..., :cols]


def quantize_blocks_fp8(device: Device, weight: Any) -> QuantizedBlocksFP8:
    """Quantize weights ``[N, K]`` or ``[E, N, K]`` (float32, bfloat16 or float16 CUDA tensor) per 128 x 128 block."""
    torch_device = require_cuda(device, "quantize_blocks_fp8")
    code = dtype_code(weight.dtype, "quantize_blocks_fp8 weight")
    if weight.dim() not in (2, 3) or 0 in weight.shape:
        raise ValueError("quantize_blocks_fp8 requires a non-empty rank-2 or rank-3 weight")
    if weight.device != torch_device:
        raise ValueError(f"quantize_blocks_fp8 weight must be on {torch_device}")
    *batch, rows, cols = weight.shape
    if rows > 65535 * FP8_GROUP or cols >= 2**31 or (batch and batch[0] > 65535):
        raise ValueError(f"quantize_blocks_fp8 takes fewer than 65536 matrices of fewer than {65535 * FP8_GROUP + 1} rows and 2**31 columns")
    weight = weight.contiguous()
    values = torch.empty(weight.shape, dtype=torch.float8_e4m3fn, device=torch_device)
    scales = torch.empty((*batch, groups_of(rows), groups_of(cols)), dtype=torch.float32, device=torch_device)
    launch(
        device, "qpucuda_fp8_quantize_blocks", weight.data_ptr(), code, cols, batch[0] if batch else 1, rows, cols,
        values.data_ptr(), cols, scales.data_ptr(),
    )
    return QuantizedBlocksFP8(values, scales)


def quantize_rows_fp8(device: Device, source: Any, *, gated: bool = False) -> QuantizedRowsFP8:
    """Quantize rows ``[M, K]`` (float32, bfloat16 or float16) with one scale per 128 columns.

    ``gated``: the source is ``[M, 2 K]``, gate then up, and ``silu(gate) * up`` is quantized,
    computed in fp32. The values are a view of rows padded to 16 bytes.
    """
    torch_device = require_cuda(device, "quantize_rows_fp8")
    code = dtype_code(source.dtype, "quantize_rows_fp8 source")
    rows, cols, stride = check_matrix(source, torch_device, "quantize_rows_fp8 source")
    if cols == 0 or (gated and cols % 2):
        raise ValueError("quantize_rows_fp8 source must have columns, an even number of them when gated")
    cols = cols // 2 if gated else cols
    q_stride = (cols + 15) // 16 * 16
    values = new_matrix(rows, q_stride, torch.float8_e4m3fn, torch_device)
    scales = new_matrix(rows, groups_of(cols), torch.float32, torch_device)
    if rows:
        desc = _pack_quantize(
            source.data_ptr(), code, stride, rows, cols, bool(gated), 0, 1, rows, values.data_ptr(), q_stride, scales.data_ptr(),
            groups_of(cols), 1,
        )
        launch(device, "qpucuda_fp8_quantize_rows", desc)
    return made(QuantizedRowsFP8, values=values if q_stride == cols else values[:, :cols], scales=scales)


class _PreparedFP8:
    """A weight (one matrix, or one per expert) resident on one GPU in the layout the product reads:
    e4m3 rows padded to 16 bytes, block scales, optional bias. The plan owns copies; calls only
    read them, so any number may be in flight. Keep the plan open until their work has finished
    (``close`` waits for the device, and raises what ``synchronize`` would)."""

    _name = "prepared FP8 linear"

    def __init__(self: Self, device: Device, weight: QuantizedBlocksFP8, bias: Any, gated: bool) -> None:
        self._torch_device = require_cuda(device, type(self).__name__)
        self.device = device
        self.gated = bool(gated)
        *batch, self.output_count, self.input_count = weight.shape
        self.experts = batch[0] if batch else 0
        self._source_columns = self.input_count * (2 if gated else 1)
        self._groups = groups_of(self.input_count)
        self._padded = padded = (self.input_count + 15) // 16 * 16
        self._values = torch.zeros((*batch, self.output_count, padded), dtype=torch.uint8, device=self._torch_device)
        self._values[..., : self.input_count].copy_(weight.values.view(torch.uint8))
        self._scales = weight.scales.to(self._torch_device).clone(memory_format=torch.contiguous_format)
        self._bias = None
        if bias is not None:
            bias = torch.as_tensor(bias)
            if tuple(bias.shape) != (self.output_count,):
                raise ValueError("bias must have one fp32 value per output feature")
            self._bias = bias.to(self._torch_device, torch.float32).clone(memory_format=torch.contiguous_format)
        self._values_address = self._values.data_ptr()
        self._scales_address = self._scales.data_ptr()
        self._bias_address = 0 if self._bias is None else self._bias.data_ptr()
        torch.cuda.current_stream(self._torch_device).synchronize()
        self._pending: list[Event] = []  # executions on queues that may not have been launched yet
        self._closed = False

    def __enter__(self: Self) -> Self:
        self._require_open()
        return self

    def __exit__(self: Self, exc_type: object, exc_value: object, traceback: object) -> None:
        self.close()

    def _require_open(self: Self) -> None:
        if self._closed:
            raise RuntimeError(f"{self._name} plan is closed")

    def synchronize(self: Self) -> None:
        """Wait for the device's current stream and raise if a kernel's wait ran out, in a call of any plan of the
        device: ``EventTimeoutError`` the first time, ``NativeError`` from then on."""
        self._require_open()
        with torch.cuda.device(self._torch_device):
            capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            raise RuntimeError(f"{self._name} calls cannot be waited for while a graph is captured")
        # without the launch lock, which other threads' calls need, and past the device's timeout if it takes that
        torch.cuda.current_stream(self._torch_device).synchronize()
        self._raise_device_errors()

    def _raise_device_errors(self: Self) -> None:
        stream = torch.cuda.current_stream(self._torch_device)
        self.device.backend.launch(stream, lambda native: native.synchronize())  # type: ignore[attr-defined]

    def close(self: Self) -> None:
        """Wait for queued executions and for the device, release the weight, and raise if a kernel's wait
        ran out (while the device is open; a closed one knows no more of it)."""
        if self._closed:
            return
        for event in self._pending:
            try:
                event.wait()
            except Exception:
                pass
        torch.cuda.synchronize(self._torch_device)
        self._values = self._scales = self._bias = None
        self._closed = True
        if not self.device.closed:
            self._raise_device_errors()

    @property
    def resident_bytes(self: Self) -> int:
        self._require_open()
        return sum(t.numel() * t.element_size() for t in (self._values, self._scales, self._bias) if t is not None)

    def _output(
        self: Self, rows: int, out: Any, dtype: Any, read: Any, read_stride: int, default: Any, *reads: Any
    ) -> tuple[Any, int]:
        if out is None:
            dtype = default if dtype is None else dtype
            dtype_code(dtype, f"{self._name} output")
            return new_matrix(rows, self.output_count, dtype, self._torch_device), self.output_count
        if dtype is not None and out.dtype != dtype:
            raise ValueError(f"{self._name} out and dtype differ")
        dtype_code(out.dtype, f"{self._name} output")
        stride = check_matrix(out, self._torch_device, f"{self._name} output", rows, self.output_count)[2]
        check_apart(out, stride, read, read_stride, f"{self._name} output")
        check_apart_from(out, stride, reads, f"{self._name} output")
        return out, stride

    def _gemm_desc(
        self: Self, a: int, a_stride: int, a_scales: int, scale_strides: tuple[int, int], rows: int, out_address: int, out_code: int,
        out_stride: int, offsets: int = 0, settled: bool = False,
    ) -> bytes:
        return _pack_gemm(
            a, a_stride, a_scales, *scale_strides, self._values_address, self._padded, self._scales_address, self._bias_address, rows,
            self.output_count, self.input_count, self.experts, offsets, out_address, out_code, out_stride, settled,
        )

    def _linear(
        self: Self, source: int, source_code: int, source_rows: int, stride: int, rows: int, out: int, out_code: int, out_stride: int,
        offsets: int = 0, row_source: int = 0, row_divisor: int = 1, stream: int | None = None,
    ) -> None:
        """Quantize and multiply. One scratch allocation, for this call alone: the quantized rows and,
        behind them, their scales, group-major (a warp of the product reads neighbouring rows' scales).
        The weight is older than the quantizer's launch, so the product may read it early; so are the
        offsets."""
        padded = self._padded
        scratch = new_matrix(rows, padded + 4 * self._groups, torch.uint8, self._torch_device)
        values = scratch.data_ptr()
        scales = values + rows * padded
        quantize = _pack_quantize(
            source, source_code, stride, rows, self.input_count, self.gated, row_source, row_divisor, source_rows, values, padded, scales, 1, rows
        )
        gemm = self._gemm_desc(values, padded, scales, (1, rows), rows, out, out_code, out_stride, offsets, True)
        launch(self.device, "qpucuda_fp8_linear", quantize, gemm, stream=stream)

    def _check_source(self: Self, source: Any) -> tuple[int, int, int]:
        """Rows, row stride and type code."""
        code = dtype_code(source.dtype, f"{self._name} source")
        rows, _, stride = check_matrix(source, self._torch_device, f"{self._name} source", None, self._source_columns)
        return rows, stride, code

    def _check_rows(self: Self, rows: QuantizedRowsFP8) -> tuple[int, int, tuple[int, int]]:
        values = rows.values
        count, _, stride = check_matrix(values, self._torch_device, f"{self._name} quantized rows", None, self.input_count)
        if count <= 1:
            stride = self._padded
        if stride % 16 or values.data_ptr() % 16:
            raise ValueError(f"{self._name} quantized rows must start on 16-byte boundaries")
        return count, stride, (int(rows.scales.stride(0)), int(rows.scales.stride(1)))


class PreparedFP8Linear(_PreparedFP8):
    """``y = x W^T (+ bias)`` with a resident block-scaled e4m3 weight ``[N, K]``.

    ``gated``: sources are ``[M, 2 K]``, gate then up (the output of one merged gate/up plan), and
    ``silu(gate) * up`` is what is quantized: an FFN's down projection.
    """

    def __init__(self: Self, device: Device, weight: QuantizedBlocksFP8, *, bias: Any = None, gated: bool = False) -> None:
        if len(weight.shape) != 2:
            raise ValueError("PreparedFP8Linear requires a rank-2 weight; PreparedFP8Experts takes one per expert")
        super().__init__(device, weight, bias, gated)

    def forward(self: Self, source: Any, out: Any = None, *, dtype: Any = None) -> Any:
        """Rows ``[M, K]`` (float32, bfloat16 or float16) to ``[M, N]`` of ``dtype`` (default: the
        source's type, or ``out``'s). ``out`` may share a buffer with the source, but no bytes."""
        self._require_open()
        rows, stride, code = self._check_source(source)
        out, out_stride = self._output(rows, out, dtype, source, stride, source.dtype)
        if rows:
            self._linear(source.data_ptr(), code, rows, stride, rows, out.data_ptr(), _DTYPE_CODES[out.dtype], out_stride)
        return out

    def forward_quantized(self: Self, rows: QuantizedRowsFP8, out: Any = None, *, dtype: Any = None) -> Any:
        """The product alone, over rows quantized before (:func:`quantize_rows_fp8`); ``dtype``
        defaults to float32."""
        self._require_open()
        count, stride, scale_strides = self._check_rows(rows)
        out, out_stride = self._output(count, out, dtype, rows.values, stride, torch.float32, rows.scales)
        if count:
            gemm = self._gemm_desc(
                rows.values.data_ptr(), stride, rows.scales.data_ptr(), scale_strides, count, out.data_ptr(), _DTYPE_CODES[out.dtype], out_stride
            )
            launch(self.device, "qpucuda_fp8_gemm", gemm)
        return out

    def execute(self: Self, destination: Tensor, source: Tensor, *, queue: Queue, wait_for: Iterable[Event] = ()) -> Event:
        """The same on a queue, float32 tensors of the plan's device (as ``PreparedW8A8Linear.execute``)."""
        self._require_open()
        if queue.device is not self.device or source.buffer.device is not self.device or destination.buffer.device is not self.device:
            raise DependencyError("prepared FP8 linear queue and tensors must belong to the plan device")
        if source.dtype != np.dtype(np.float32) or destination.dtype != np.dtype(np.float32):
            raise ValueError("prepared FP8 linear requires float32 source and destination")
        if len(source.shape) != 2 or source.shape[1] != self._source_columns or destination.shape != (source.shape[0], self.output_count):
            raise ValueError("prepared FP8 linear source and destination shapes do not align")
        if source.strides[1] != 4 or destination.strides[1] != 4:
            raise ValueError("prepared FP8 linear requires unit inner strides")
        if _meet(*((t.address, *t.shape, t.strides[0], 4) for t in (destination, source))):
            raise ValueError("prepared FP8 linear destination must not overlap its source")
        rows = int(source.shape[0])

        def executor(backend: Any, args: tuple[Any, ...], grid: tuple[int, int, int], stream: Any) -> None:
            with torch.cuda.stream(stream):  # the scratch belongs to the queue's stream
                self._linear(
                    source.address, _native.DTYPE_F32, rows, source.row_stride_elements, rows, destination.address, _native.DTYPE_F32,
                    destination.row_stride_elements, stream=stream.cuda_stream,
                )

        event = queue.submit(
            Kernel("cuda.fp8_linear", executor), (), wait_for=wait_for,
            buffers=(source.access(AccessMode.READ), destination.access(AccessMode.WRITE)),
        )
        with self.device.backend.launch_lock:  # type: ignore[attr-defined]
            self._pending = [*(pending for pending in self._pending if not pending.done), event]
        return event


class PreparedFP8Experts(_PreparedFP8):
    """One resident block-scaled e4m3 weight per expert, ``[E, N, K]``: rows sorted by expert (see
    :func:`qpu_xla.experts.sort_tokens`) meet their expert's matrix in one launch."""

    _name = "prepared FP8 experts"

    def __init__(self: Self, device: Device, weight: QuantizedBlocksFP8, *, gated: bool = False) -> None:
        if len(weight.shape) != 3:
            raise ValueError("PreparedFP8Experts requires a rank-3 weight [experts, outputs, inputs]")
        if weight.shape[0] > MAX_EXPERTS:
            raise ValueError(f"PreparedFP8Experts takes at most {MAX_EXPERTS} experts")
        super().__init__(device, weight, None, gated)

    def _check_offsets(self: Self, offsets: Any) -> None:
        if offsets.dtype != torch.int32 or tuple(offsets.shape) != (self.experts + 1,) or not offsets.is_contiguous():
            raise ValueError("prepared FP8 experts need contiguous int32 offsets [experts + 1]")
        if offsets.device != self._torch_device:
            raise ValueError(f"prepared FP8 experts offsets must be on {self._torch_device}")

    def forward(self: Self, source: Any, offsets: Any, out: Any = None, *, dtype: Any = None) -> Any:
        """Rows ``[R, K]``, those of expert e at ``offsets[e] .. offsets[e + 1]`` (ascending int32 on
        the GPU, clamped to ``[0, R]``), to ``[R, N]``. Rows from ``offsets[E]`` on become zero."""
        self._require_open()
        rows, stride, code = self._check_source(source)
        self._check_offsets(offsets)
        out, out_stride = self._output(rows, out, dtype, source, stride, source.dtype, offsets)
        if rows:
            self._linear(source.data_ptr(), code, rows, stride, rows, out.data_ptr(), _DTYPE_CODES[out.dtype], out_stride, offsets.data_ptr())
        return out

    def forward_tokens(self: Self, tokens: Any, order: Any, out: Any = None, *, dtype: Any = None) -> Any:
        """:meth:`forward` of the tokens ``[T, K]`` in expert order, without the sorted copy: row r is
        quantized straight from token ``order.source[r] // choices``. ``[T * choices, N]``."""
        self._require_open()
        tokens_count, stride, code = self._check_source(tokens)
        self._check_offsets(order.offsets)
        order.check(self._torch_device, tokens=tokens_count)
        rows = order.rows
        out, out_stride = self._output(rows, out, dtype, tokens, stride, tokens.dtype, order.offsets, order.source)
        if rows:
            self._linear(
                tokens.data_ptr(), code, tokens_count, stride, rows, out.data_ptr(), _DTYPE_CODES[out.dtype], out_stride, order.offsets.data_ptr(),
                order.source.data_ptr(), order.choices,
            )
        return out


__all__ = [
    "FP8_GROUP",
    "MAX_EXPERTS",
    "PreparedFP8Experts",
    "PreparedFP8Linear",
    "QuantizedBlocksFP8",
    "QuantizedRowsFP8",
    "quantize_blocks_fp8",
    "quantize_rows_fp8",
]
