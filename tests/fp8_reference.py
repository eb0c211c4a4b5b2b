"""Plain float64 restatements of the block-scaled FP8 linear and the expert routing (test oracle)."""

from __future__ import annotations

import torch

GROUP = 128
FLOOR = 2.0**-60


def groups(size: int) -> int:
    return -(-size // GROUP)


def e4m3(quotient: torch.Tensor) -> torch.Tensor:
    """fp32 quotients to the nearest e4m3 values (ties to even, at most 448), as float64."""
    return quotient.float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double()


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values [M, K] and scales [M, groups] as float64, quotients rounded to fp32 first."""
    x = x.double()
    values, scales = torch.empty_like(x), torch.empty((x.shape[0], groups(x.shape[1])), dtype=torch.float64, device=x.device)
    for g in range(scales.shape[1]):
        part = x[:, g * GROUP : (g + 1) * GROUP]
        scales[:, g] = (part.abs().amax(dim=1) / 448.0).float().double().clamp_min(FLOOR)
        values[:, g * GROUP : (g + 1) * GROUP] = e4m3(part / scales[:, g : g + 1])
    return values, scales


def quantize_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    w = w.double()
    rows, cols = w.shape
    values, scales = torch.empty_like(w), torch.empty((groups(rows), groups(cols)), dtype=torch.float64, device=w.device)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            block = (slice(i * GROUP, (i + 1) * GROUP), slice(j * GROUP, (j + 1) * GROUP))
            scales[i, j] = (w[block].abs().amax() / 448.0).float().double().clamp_min(FLOOR)
            values[block] = e4m3(w[block] / scales[i, j])
    return values, scales


def spread(scales: torch.Tensor, rows: int, cols: int, row_group: int) -> torch.Tensor:
    return scales.repeat_interleave(row_group, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]


def silu_gate(x: torch.Tensor) -> torch.Tensor:
    gate, up = x.double().chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up


def product(values: torch.Tensor, scales: torch.Tensor, w_values: torch.Tensor, w_scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """y and the sum of the products' magnitudes, float64."""
    left = values.double() * spread(scales.double(), *values.shape, 1)
    right = w_values.double() * spread(w_scales.double(), *w_values.shape, GROUP)
    return left @ right.t(), left.abs() @ right.abs().t()


def product_tolerance(exact: torch.Tensor, magnitude: torch.Tensor, k: int, dtype: torch.dtype) -> torch.Tensor:
    """Bound of |kernel - exact|. A block's 128 exact products are summed in fp32 with at most one
    step (2^-23) lost per addition: 256 units of 2^-24 of the block's magnitude. The factor sx * sw
    and the fma round once each, and each of the blocks' additions rounds once: (blocks + 2) units.
    A split sum adds at most 8 more, the bias one. Then one rounding to the output's type."""
    fp32 = (256 + groups(k) + 2 + 8 + 1) * 2.0**-24 * magnitude
    return fp32 + torch.finfo(dtype).eps / 2 * (exact.abs() + fp32) + torch.finfo(dtype).smallest_normal * 2.0**-8


def sort(ids: torch.Tensor, experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    flat = ids.reshape(-1).cpu().tolist()
    source = [i for e in range(experts) for i, have in enumerate(flat) if have == e] if experts <= 8 else None
    if source is None:
        buckets: list[list[int]] = [[] for _ in range(experts)]
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                buckets[e].append(i)
        source = [i for bucket in buckets for i in bucket]
    counts = [0] * experts
    for e in flat:
        if 0 <= e < experts:
            counts[e] += 1
    offsets = [0]
    for count in counts:
        offsets.append(offsets[-1] + count)
    position = [-1] * len(flat)
    for row, i in enumerate(source):
        position[i] = row
    source += [-1] * (len(flat) - len(source))
    as_int = [torch.tensor(v, dtype=torch.int32) for v in (offsets, source, position)]
    return as_int[0], as_int[1], as_int[2].view(ids.shape)
