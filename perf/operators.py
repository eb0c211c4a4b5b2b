"""Block-scaled FP8 linears and expert token routing: the cases these operators are measured on.

Four groups of calls, all on one GPU:

* ``quantize``  rows to e4m3 with one fp32 scale per 128 columns;
* ``linear``    ``y = x W^T (+ bias)``, both operands e4m3, x scaled per row and 128 columns, W per
  128 x 128 block; ``gated`` rows hold ``[gate | up]`` and enter as ``silu(gate) * up``;
* ``experts``   the same product with one W per expert over rows sorted by expert;
* ``dispatch`` / ``combine``  tokens sorted by expert and copied into that order, and the rows
  summed back per token with their routing weights; each with its gradient.

``run`` is either the plain form (elementary torch operations in fp32) or, with ``own`` set, the
calls a user makes of ``qpu_xla.fp8`` and ``qpu_xla.experts``. ``exact`` is the definition in 64 bits.

Definitions: a group's scale is ``s = max(fl32(max|x| / 448), 2^-60)``, its values
``e4m3(fl32(x / s))``, round to nearest even. A product's value is ``sum_k (q_x s_x)(q_w s_w)``. Rows
are ordered by expert, then by token, then by choice; an expert id outside ``[0, experts)`` drops
that choice, and rows that belong to no expert are zero.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 128
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0**-60
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ITEMSIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---- cases ------------------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # The activations of one 4096-token prompt entering the 70B FFN.
        {"name": "quantize-prompt", "op": "quantize", "rows": 4096, "cols": 8192, "dtype": "bfloat16"},
        # A short batch of an odd width in fp32: the last group of each row is partly filled.
        {"name": "quantize-odd", "op": "quantize", "rows": 700, "cols": 5001, "dtype": "float32"},
        # One token through a TinyLlama q projection: latency.
        {"name": "linear-one", "op": "linear", "rows": 1, "n": 2048, "k": 2048, "dtype": "bfloat16", "bias": False, "gated": False},
        # Four sequences decoding through the 70B gate projection: the weight's bytes.
        {"name": "linear-decode", "op": "linear", "rows": 4, "n": 28672, "k": 8192, "dtype": "bfloat16", "bias": False, "gated": False},
        # A mid-size batch through a down projection of odd width, from gate and up, with a bias.
        {"name": "linear-gated", "op": "linear", "rows": 333, "n": 5001, "k": 5632, "dtype": "float16", "bias": True, "gated": True},
        # The prompt through the 70B gate projection: the tensor cores.
        {"name": "linear-prompt", "op": "linear", "rows": 4096, "n": 28672, "k": 8192, "dtype": "bfloat16", "bias": False, "gated": False},
        # Eight tokens decoding, eight of 64 experts each: about one row per weight.
        {"name": "experts-decode", "op": "experts", "tokens": 8, "choices": 8, "experts": 64, "n": 2816, "k": 2048, "dtype": "bfloat16"},
        # A prompt of 4096 tokens, four of 32 experts each, of uneven popularity.
        {"name": "experts-prompt", "op": "experts", "tokens": 4096, "choices": 4, "experts": 32, "n": 5632, "k": 2048, "dtype": "bfloat16"},
        # That prompt's tokens into expert order, some of them padding.
        {"name": "dispatch-prompt", "op": "dispatch", "tokens": 4096, "choices": 4, "experts": 32, "width": 2048, "dtype": "bfloat16", "padding": 0.02},
        # The gradient of the tokens from the gradient of the sorted rows, in fp32, odd width.
        {"name": "dispatch-gradient", "op": "dispatch-gradient", "tokens": 1500, "choices": 2, "experts": 8, "width": 4099, "dtype": "float32", "padding": 0.0},
        # Eight decoding tokens summed back: latency.
        {"name": "combine-decode", "op": "combine", "tokens": 8, "choices": 8, "experts": 64, "width": 2048, "dtype": "bfloat16", "padding": 0.0},
        # The gradients of rows and routing weights for a prompt.
        {"name": "combine-gradient", "op": "combine-gradient", "tokens": 4096, "choices": 4, "experts": 32, "width": 2048, "dtype": "bfloat16", "padding": 0.02},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    op = rng.choice(["quantize", "linear", "linear", "experts", "dispatch", "dispatch-gradient", "combine", "combine-gradient"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])

    def size(low: int, high: int) -> int:
        value = _log_int(rng, low, high)
        return value if rng.random() < 0.4 else max(low, value // 128 * 128)

    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "cols": size(128, 16384), "dtype": dtype}
    if op == "linear":
        rows, n, k = _log_int(rng, 1, 4096), size(128, 28672), size(128, 28672)
        while n * k > 28672 * 8192:
            n, k = size(128, 28672), size(128, 28672)
        return {"op": op, "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3, "gated": rng.random() < 0.3}
    experts = _log_int(rng, 2, 128)
    choices = rng.randint(1, min(8, experts))
    tokens = _log_int(rng, 1, 8192)
    if op == "experts":
        n, k = size(128, 8192), size(128, 8192)
        while experts * n * k > 1 << 30:
            n, k = max(128, n * 3 // 4), max(128, k * 3 // 4)
        return {"op": op, "tokens": tokens, "choices": choices, "experts": experts, "n": n, "k": k, "dtype": dtype}
    width = size(128, 8192)
    return {"op": op, "tokens": tokens, "choices": choices, "experts": experts, "width": width, "dtype": dtype, "padding": rng.choice([0.0, 0.05])}


def work(case: dict) -> dict:
    op, item = case["op"], ITEMSIZE[case["dtype"]]
    if op == "quantize":
        elements = case["rows"] * case["cols"]
        return {"bytes": elements * (item + 1) + 4 * case["rows"] * _groups(case["cols"]), "flops": 3 * elements}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        inputs = m * k * item * (2 if case["gated"] else 1)
        weight = n * k + 4 * _groups(n) * _groups(k) + (4 * n if case["bias"] else 0)
        return {"bytes": inputs + weight + m * n * item, "flops": 2 * m * n * k}
    t, c, e = case["tokens"], case["choices"], case["experts"]
    if op == "experts":
        rows, n, k = t * c, case["n"], case["k"]
        active = e * (1.0 - (1.0 - c / e) ** t)  # experts that get a row, were all equally popular
        weight = active * (n * k + 4 * _groups(n) * _groups(k))
        return {"bytes": int(rows * (k + n) * item + weight + 4 * (e + 1)), "flops": 2 * rows * n * k}
    width, tables = case["width"], 4 * t * c
    if op == "dispatch":
        return {"bytes": (t + t * c) * width * item + 3 * tables + 4 * (e + 1), "flops": t * c}
    if op == "dispatch-gradient":
        return {"bytes": (t + t * c) * width * item + tables, "flops": t * c * width}
    if op == "combine":
        return {"bytes": (t + t * c) * width * item + 2 * tables, "flops": 2 * t * c * width}
    return {"bytes": (t + 2 * t * c) * width * item + 3 * tables, "flops": 3 * t * c * width}


def _groups(size: int) -> int:
    return (size + GROUP - 1) // GROUP


# ---- inputs -----------------------------------------------------------------------------------


def _generator(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(shape: tuple[int, int], dtype: torch.dtype, generator):
    """Normal activations with a few loud channels, as hidden states have them."""
    x = torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32)
    loud = torch.rand(shape[1], generator=generator, device="cuda") < 0.01
    x *= torch.where(loud, 12.0, 1.0)
    return x.to(dtype)


def _weight(rows: int, cols: int, generator):
    """A trained matrix's e4m3 values and block scales, as a checkpoint holds them."""
    w = torch.randn((rows, cols), generator=generator, device="cuda", dtype=torch.float32) * 0.02
    padded = torch.zeros((_groups(rows) * GROUP, _groups(cols) * GROUP), device="cuda", dtype=torch.float32)
    padded[:rows, :cols] = w
    blocks = padded.view(_groups(rows), GROUP, _groups(cols), GROUP)
    scales = (blocks.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    values = (blocks / scales[:, None, :, None]).view(padded.shape)[:rows, :cols]
    return values.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).contiguous(), scales


def _routing(case: dict, generator):
    """Each token's choices (distinct experts of uneven popularity) and its weights (summing to 1);
    a padding token has the id -1 everywhere."""
    tokens, choices, experts = case["tokens"], case["choices"], case["experts"]
    popularity = torch.randn(experts, generator=generator, device="cuda") * 0.5
    scores = torch.randn((tokens, experts), generator=generator, device="cuda") + popularity
    top, ids = torch.topk(scores, choices, dim=1)
    weights = torch.softmax(top, dim=1)
    ids = ids.to(torch.int32)
    if case.get("padding", 0.0) > 0.0:
        ids[torch.rand(tokens, generator=generator, device="cuda") < case["padding"]] = -1
    return ids.contiguous(), weights.contiguous()


def _inputs(case: dict, seed: int) -> dict:
    g, dtype, op = _generator(seed), DTYPES[case["dtype"]], case["op"]
    if op == "quantize":
        return {"x": _activations((case["rows"], case["cols"]), dtype, g)}
    if op == "linear":
        x = _activations((case["rows"], case["k"] * (2 if case["gated"] else 1)), dtype, g)
        values, scales = _weight(case["n"], case["k"], g)
        bias = torch.randn(case["n"], generator=g, device="cuda") * 0.1 if case["bias"] else None
        return {"x": x, "values": values, "scales": scales, "bias": bias}
    ids, weights = _routing(case, g)
    rows = case["tokens"] * case["choices"]
    if op == "experts":
        x = _activations((rows, case["k"]), dtype, g)
        parts = [_weight(case["n"], case["k"], g) for _ in range(case["experts"])]
        offsets = _order(ids, case["experts"])[0]
        return {"x": x, "values": torch.stack([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn),
                "scales": torch.stack([p[1] for p in parts]), "offsets": offsets}
    if op == "dispatch":
        return {"ids": ids, "x": _activations((case["tokens"], case["width"]), dtype, g)}
    offsets, source, position = _order(ids, case["experts"])
    state = {"offsets": offsets, "source": source, "position": position, "weights": weights}
    state["rows"] = _activations((rows, case["width"]), dtype, g)
    if op == "combine-gradient":
        state["grad"] = torch.randn((case["tokens"], case["width"]), generator=g, device="cuda").to(dtype)
    return state


def _device():
    root = Path(__file__).resolve().parents[1] / "qpu-xla-triton_b200"
    if str(root) not in sys.path:
        sys.path.insert(0, str(root))
    from qpu_xla import Device

    if not hasattr(_device, "opened"):
        _device.opened = Device.open()
    return _device.opened


def _plan(state: dict) -> None:
    """What a program makes once and keeps: the plan that owns the weight, the order of the forward pass."""
    device, op = _device(), state["case"]["op"]
    from qpu_xla import experts, fp8

    if op == "linear":
        weight = fp8.QuantizedBlocksFP8(state["values"], state["scales"])
        state["plan"] = fp8.PreparedFP8Linear(device, weight, bias=state["bias"], gated=state["case"]["gated"])
    elif op == "experts":
        weight = fp8.QuantizedBlocksFP8(state["values"], state["scales"])
        state["plan"] = fp8.PreparedFP8Experts(device, weight)
    elif "position" in state:
        state["plan"] = experts.ExpertOrder(state["offsets"], state["source"], state["position"])
    else:
        state["plan"] = None


def prepare(case: dict, seed: int) -> dict:
    state = {"case": dict(case), **_inputs(case, seed)}
    if own:
        _plan(state)
    return state


# ---- the framework's calls ----------------------------------------------------------------------


def _run_own(state: dict):
    if "plan" not in state:
        _plan(state)
    device, case, op = _device(), state["case"], state["case"]["op"]
    from qpu_xla import experts, fp8

    if op == "quantize":
        rows = fp8.quantize_rows_fp8(device, state["x"])
        return [rows.values, rows.scales]
    if op == "linear":
        return state["plan"].forward(state["x"])
    if op == "experts":
        return state["plan"].forward(state["x"], state["offsets"])
    if op == "dispatch":
        order = experts.sort_tokens(device, state["ids"], case["experts"])
        return [order.offsets, order.source, order.position, experts.gather_tokens(device, state["x"], order)]
    if op == "dispatch-gradient":
        return experts.gather_tokens_backward(device, state["rows"], state["plan"])
    if op == "combine":
        return experts.combine_tokens(device, state["rows"], state["weights"], state["plan"])
    return list(experts.combine_tokens_backward(device, state["rows"], state["weights"], state["grad"], state["plan"]))


# ---- the plain form ------------------------------------------------------------------------------


def _quantize(x):
    rows, cols = x.shape
    padded = torch.zeros((rows, _groups(cols) * GROUP), device=x.device, dtype=torch.float32)
    padded[:, :cols] = x
    groups = padded.view(rows, _groups(cols), GROUP)
    # A divisor on the GPU: torch multiplies by the reciprocal of a Python number, which is not the quotient.
    scales = (groups.abs().amax(dim=2) / torch.full((), E4M3_MAX, device=x.device)).clamp_min(SCALE_FLOOR)
    values = (groups / scales[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).float()
    return values, scales


def _spread(scales, rows: int, cols: int):
    return scales.repeat_interleave(GROUP, dim=0)[:rows].repeat_interleave(GROUP, dim=1)[:, :cols]


def _gate(x, gated: bool):
    x = x.float()
    if not gated:
        return x
    gate, up = x.chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _product(x, values, scales):
    quantized, row_scales = _quantize(x)
    left = (quantized * row_scales[:, :, None]).view(x.shape[0], -1)[:, : x.shape[1]]
    right = values.float() * _spread(scales, *values.shape)
    return left @ right.t()


def _order(ids, experts: int):
    """Offsets [experts + 1], the choice (token * choices + j) at each row, the row of each choice;
    dropped choices come last in ``source``, as -1, and have position -1."""
    flat = ids.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    by_expert = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.cumsum(counts, 0).to(torch.int32)
    rank = torch.arange(flat.numel(), dtype=torch.int32, device=ids.device)
    kept = rank < offsets[-1]
    source = torch.where(kept, by_expert.to(torch.int32), torch.full_like(rank, -1))
    position = torch.empty_like(rank)
    position[by_expert] = torch.where(kept, rank, torch.full_like(rank, -1))
    return offsets, source, position.view(ids.shape)


def _picked(rows, position):
    """fp32 rows of each token's choices [tokens, choices, width], zero where dropped."""
    kept = position >= 0
    picked = rows[position.clamp_min(0).long().reshape(-1)].float().view(*position.shape, -1)
    return torch.where(kept[:, :, None], picked, torch.zeros_like(picked)), kept


def _run_plain(state: dict):
    case, op = state["case"], state["case"]["op"]
    dtype = DTYPES[case["dtype"]]
    if op == "quantize":
        values, scales = _quantize(state["x"])
        return [values.view(case["rows"], -1)[:, : case["cols"]].to(torch.float8_e4m3fn), scales]
    if op == "linear":
        y = _product(_gate(state["x"], case["gated"]), state["values"], state["scales"])
        return (y if state["bias"] is None else y + state["bias"]).to(dtype)
    if op == "experts":
        bounds = state["offsets"].tolist()
        out = torch.zeros((state["x"].shape[0], case["n"]), device="cuda", dtype=dtype)
        for e, (begin, end) in enumerate(zip(bounds, bounds[1:])):
            if end > begin:
                out[begin:end] = _product(state["x"][begin:end].float(), state["values"][e], state["scales"][e]).to(dtype)
        return out
    if op == "dispatch":
        offsets, source, position = _order(state["ids"], case["experts"])
        token = torch.div(source.clamp_min(0), case["choices"], rounding_mode="floor").long()
        rows = torch.where((source >= 0)[:, None], state["x"][token], torch.zeros((), device="cuda", dtype=dtype))
        return [offsets, source, position, rows]
    if op == "dispatch-gradient":
        return _picked(state["rows"], state["position"])[0].sum(dim=1).to(dtype)
    picked, kept = _picked(state["rows"], state["position"])
    if op == "combine":
        return (picked * state["weights"][:, :, None]).sum(dim=1).to(dtype)
    grad = state["grad"].float()
    grad_weights = torch.where(kept, (picked * grad[:, None, :]).sum(dim=2), torch.zeros_like(state["weights"]))
    grad_rows = torch.zeros_like(state["rows"])
    scaled = (state["weights"][:, :, None] * grad[:, None, :]).to(dtype)
    grad_rows[state["position"][kept].long()] = scaled[kept]
    return [grad_rows, grad_weights]


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------------


def _exact_groups(x64):
    """Column groups of a float64 matrix: their e4m3 values (float64) and scales, group by group."""
    for begin in range(0, x64.shape[1], GROUP):
        part = x64[:, begin : begin + GROUP]
        scale = (part.abs().max(dim=1).values / E4M3_MAX).float().double().clamp(min=SCALE_FLOOR)
        quotient = (part / scale[:, None]).float().clamp(-E4M3_MAX, E4M3_MAX)
        yield begin, quotient.to(torch.float8_e4m3fn).double(), scale


def _exact_product(x64, values, scales):
    out = torch.zeros((x64.shape[0], values.shape[0]), device="cuda", dtype=torch.float64)
    row_block = torch.arange(values.shape[0], device="cuda") // GROUP
    for begin, q, scale in _exact_groups(x64):
        w = values[:, begin : begin + GROUP].double() * scales[row_block, begin // GROUP].double()[:, None]
        out += (q * scale[:, None]) @ w.t()
    return out


def exact(case: dict, seed: int):
    inputs, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        parts = list(_exact_groups(inputs["x"].double()))
        return [torch.cat([p[1] for p in parts], dim=1), torch.stack([p[2] for p in parts], dim=1)]
    if op == "linear":
        x = inputs["x"].double()
        if case["gated"]:
            x = x[:, : case["k"]] * torch.sigmoid(x[:, : case["k"]]) * x[:, case["k"] :]
        y = _exact_product(x, inputs["values"], inputs["scales"])
        return y if inputs["bias"] is None else y + inputs["bias"].double()
    if op == "experts":
        bounds = inputs["offsets"].cpu().tolist()
        out = torch.zeros((inputs["x"].shape[0], case["n"]), device="cuda", dtype=torch.float64)
        for e in range(case["experts"]):
            begin, end = bounds[e], bounds[e + 1]
            if begin < end:
                out[begin:end] = _exact_product(inputs["x"][begin:end].double(), inputs["values"][e], inputs["scales"][e])
        return out
    choices, width = case["choices"], case["width"]
    if op == "dispatch":
        ids = inputs["ids"].cpu().reshape(-1).tolist()
        lists: list[list[int]] = [[] for _ in range(case["experts"])]
        for index, expert in enumerate(ids):
            if 0 <= expert < case["experts"]:
                lists[expert].append(index)
        source = [index for chosen in lists for index in chosen]
        offsets = [0]
        for chosen in lists:
            offsets.append(offsets[-1] + len(chosen))
        position = [-1] * len(ids)
        for row, index in enumerate(source):
            position[index] = row
        rows = torch.zeros((len(ids), width), device="cuda", dtype=torch.float64)
        tokens = torch.tensor([index // choices for index in source], device="cuda", dtype=torch.long)
        rows[: len(source)] = inputs["x"].double()[tokens]
        source += [-1] * (len(ids) - len(source))
        integers = [torch.tensor(v, device="cuda", dtype=torch.int32) for v in (offsets, source, position)]
        return [integers[0], integers[1], integers[2].view(case["tokens"], choices), rows]
    rows, position, weights = inputs["rows"].double(), inputs["position"].long(), inputs["weights"].double()
    out = torch.zeros((case["tokens"], width), device="cuda", dtype=torch.float64)
    grad_rows, grad_weights = torch.zeros_like(rows), torch.zeros_like(weights)
    for j in range(choices):
        tokens = torch.nonzero(position[:, j] >= 0)[:, 0]
        at = position[tokens, j]
        if op == "dispatch-gradient":
            out[tokens] += rows[at]
        elif op == "combine":
            out[tokens] += weights[tokens, j][:, None] * rows[at]
        else:
            grad = inputs["grad"].double()[tokens]
            grad_rows[at] = weights[tokens, j][:, None] * grad
            grad_weights[tokens, j] = torch.einsum("tw,tw->t", rows[at], grad)
    return [grad_rows, grad_weights] if op == "combine-gradient" else out
