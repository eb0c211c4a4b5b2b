"""Block-scaled FP8 on the GPU where it can go wrong: the widths of last tiles, signs and padding of quantized
rows, waits that ran out."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
from qpu_xla import Device, _native
from qpu_xla.errors import EventTimeoutError, NativeError
from qpu_xla.fp8 import PreparedFP8Experts, PreparedFP8Linear, dtype_code, quantize_blocks_fp8, quantize_rows_fp8
from test_gpu_fp8 import DTYPES, blocks, check_product, draw, expert_case

pytestmark = pytest.mark.gpu

# One box is 128 bytes of each of a warp's 32 rows and a tile's half has 128 columns, so widths that end in one
# whole box (16-bit: 64, fp32: 32) or three (fp32: 96) give an odd number; the others are their neighbours.
WIDTHS = [(torch.bfloat16, n) for n in (64, 192, 320, 576, 640)] + [(torch.float16, n) for n in (64, 192, 576)] + [
    (torch.float32, n) for n in (32, 96, 160, 224, 352, 384)
]


@pytest.mark.parametrize("dtype, n", WIDTHS)
@pytest.mark.parametrize("k", [128, 200])
def test_many_short_tiles_of_every_width(cuda_device, dtype, n, k) -> None:
    """65536 rows are 256 pairs' tiles per 256 columns, several to each pair of CTAs, and K of one or two blocks
    leaves next to no time between a tile's store and the next one's. The copy engine's rows equal the warps'
    (an output off its 16-byte boundary) bit for bit, and repeat."""
    rows = 65536
    weight = blocks(cuda_device, n, k)
    x = draw((rows, k), torch.bfloat16, seed=n)
    exact, magnitude = ref.product(*ref.quantize_rows(x), weight.values, weight.scales)
    wide = torch.full((rows, n + 3), 7.0, dtype=dtype, device="cuda")
    with PreparedFP8Linear(cuda_device, weight) as plan:
        y = plan.forward(x, dtype=dtype)
        check_product(y, exact, magnitude, k)
        for _ in range(5):
            assert torch.equal(plan.forward(x, dtype=dtype), y)
        plan.forward(x, out=wide[:, 1 : 1 + n])
        assert torch.equal(wide[:, 1 : 1 + n], y)


@pytest.mark.parametrize("dtype, n", WIDTHS)
@pytest.mark.parametrize("counts", [[700] * 16, [1100, 0, 900, 1300] * 4])
def test_many_short_tiles_of_every_width_with_experts(cuda_device, dtype, n, counts) -> None:
    """The same with a matrix per expert, in tiles of one CTA and of pairs: every expert has its own last tiles."""
    k = 128
    weight, x, offsets, exact, magnitude = expert_case(cuda_device, counts, n, k, trailing=5)
    wide = torch.full((x.shape[0], n + 3), 7.0, dtype=dtype, device="cuda")
    with PreparedFP8Experts(cuda_device, weight) as plan:
        y = plan.forward(x, offsets, dtype=dtype)
        check_product(y, exact, magnitude, k)
        for _ in range(5):
            assert torch.equal(plan.forward(x, offsets, dtype=dtype), y)
        plan.forward(x, offsets, out=wide[:, 1 : 1 + n])
        assert torch.equal(wide[:, 1 : 1 + n], y)


def test_an_expired_wait_reaches_the_caller_of_a_stream(cuda_device) -> None:
    """``synchronize`` and ``close`` read the error word after the stream's work: with the library's injected wait
    failure in place of a kernel's, on a context of its own."""
    weight = blocks(cuda_device, 64, 128)
    x = draw((4, 128))
    with Device.open(device_ordinal=0) as device:
        plan, other = PreparedFP8Linear(device, weight), PreparedFP8Linear(device, weight)
        y = plan.forward(x)
        plan.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            again = plan.forward(x)
            plan.synchronize()
            assert torch.equal(again, y)
        device.backend.native.set_failure_mask(int(_native.FailurePoint.WAIT))
        plan.forward(x)
        with pytest.raises(EventTimeoutError):
            plan.synchronize()
        device.backend.native.set_failure_mask(0)
        with pytest.raises(NativeError, match="poisoned"):
            other.forward(x)
        for each in (plan, other):
            with pytest.raises(NativeError, match="poisoned"):
                each.close()
            assert each._values is None
    with PreparedFP8Linear(cuda_device, weight) as plan:  # other contexts of the device go on
        assert torch.equal(plan.forward(x), y)
        plan.synchronize()


def signed(shape: tuple[int, int], dtype: torch.dtype, seed: int) -> torch.Tensor:
    """Values a third of which are zeros of either sign or so small that they end as one."""
    x = draw(shape, dtype, seed=seed)
    kind = torch.randint(0, 9, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    sign = torch.where(x < 0, -1.0, 1.0).to(dtype)
    x[kind == 0] = 0.0
    x[kind == 1] = -0.0
    return torch.where(kind == 2, sign * torch.finfo(dtype).tiny, x)


def as_bytes(values: torch.Tensor) -> torch.Tensor:
    """The bytes of float64 e4m3 values; a zero has its sign."""
    return values.float().to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (7, 129), (40, 1000), (1200, 1003)])
def test_quantized_bytes_keep_the_sign_of_zero(cuda_device, dtype, rows, cols) -> None:
    x = signed((rows, cols), dtype, seed=cols)
    x[0, 0] = -0.0
    assert torch.equal(quantize_rows_fp8(cuda_device, x).values.view(torch.uint8), as_bytes(ref.quantize_rows(x)[0]))
    assert torch.equal(quantize_blocks_fp8(cuda_device, x).values.view(torch.uint8), as_bytes(ref.quantize_blocks(x)[0]))
    wide = signed((rows, cols + 2), dtype, seed=cols)[:, 1 : cols + 1]
    assert torch.equal(quantize_rows_fp8(cuda_device, wide).values.view(torch.uint8), as_bytes(ref.quantize_rows(wide)[0]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(3, 128), (40, 1003)])
@pytest.mark.parametrize("far", [False, True])
def test_gated_bytes_have_the_sign_of_their_product(cuda_device, dtype, rows, cols, far) -> None:
    """silu(g) has g's sign at every size, zeros included; ``far``: beside gates below -87, which go another way."""
    x = signed((rows, 2 * cols), dtype, seed=cols)
    if far:
        x[:, 3::8] = -100.0
    sign = torch.signbit(x[:, :cols]) ^ torch.signbit(x[:, cols:])
    values = quantize_rows_fp8(cuda_device, x, gated=True).values
    assert torch.equal(values.view(torch.uint8) >= 0x80, sign)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(5, 1), (5, 13), (5, 130), (5, 255), (1300, 1003)])
@pytest.mark.parametrize("offset", [0, 1])
def test_bytes_behind_the_columns(cuda_device, dtype, rows, cols, offset) -> None:
    """Up to a vector's end (16 bytes of the source) they are quantized zeros, NaN in a last group that holds a NaN or
    an infinity; what lies behind that stays as it was."""
    x = draw((rows, cols + 8), dtype, seed=cols)[:, offset : cols + offset]
    x[1, cols - 1] = float("nan")
    x[2, (cols - 1) // 128 * 128] = -float("inf")
    stride = -(-cols // 16) * 16 + 16
    values = torch.full((rows, stride), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.empty((rows, -(-cols // 128)), device="cuda")
    desc = _native.Fp8QuantizeDesc(
        x.data_ptr(), dtype_code(dtype, "x"), x.stride(0), rows, cols, 0, None, 1, rows, values.data_ptr(), stride, scales.data_ptr(), scales.shape[1], 1
    )
    cuda_device.backend.call("qpucuda_fp8_quantize_rows", (bytes(desc),), cuda_device.backend.current_stream_handle)
    end = cols + -cols % (16 // x.element_size())
    assert (values[1:3, cols:end] == 0x7F).all() and (values[0, cols:end] == 0).all() and (values[3:, cols:end] == 0).all()
    assert (values[:, end:] == 0x55).all()
    quantized = quantize_rows_fp8(cuda_device, x)
    assert torch.equal(values[:, :cols], quantized.values.view(torch.uint8))
    assert quantized.values[1, cols - 1].isnan() and quantized.values[2, (cols - 1) // 128 * 128].isnan()
