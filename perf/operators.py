"""The 8-bit operators of the decoder's projections: plain forms, and the framework's own calls.

Rows in 8 bits are e4m3 values [rows, width] with one power of two per row and block of 128
columns: element c of a row stands for values[c] * scales[c // 128]. The power is the smallest with
which the block's largest magnitude does not pass 448, the largest e4m3 value.

  round    fp16 rows rounded to 8 bits (quantize_fp8): attention outputs, long prompts' activations,
           weights.
  norm     residual add and root-mean-square norm, the norm's output in 8 bits (add_rms_norm_fp8);
           the residual's delta is fp16, or fp32 partial sums of a split projection.
  project  a projection of 8-bit rows by an 8-bit weight (gemm_fp8): fp32 partial sums of K splits (a
           decode step's rows, up to 128), fp16, or SwiGLU of a stacked [gate | up] weight in fp16 or in
           8 bits. Up to 128 rows the input may also be fp16 rows, rounded to 8 bits on the way in.
  qkv      the q|k|v projection with RoPE, K and V written to their slots of the paged pool
           (qkv_rope_append_fp8).

Sizes are the TinyLlama architecture of the decoder (hidden 2048, 32 query and 4 kv heads of 64, MLP
5632) at decode steps of 1 to 128 rows and prompts of up to 2048 tokens, and ragged sizes around them.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
LAYERS, HIDDEN, MLP, QKV = 22, 2048, 5632, 2560
Q_HEADS, KV_HEADS, DIM, SLOTS = 32, 4, 64, 16
BLOCK, LARGEST, EPS = 128, 448.0, 1e-5


def listed():
    return [
        # One token's attention output, and a full-length prompt's MLP activations, rounded.
        {"name": "round_1", "kind": "round", "rows": 1, "width": HIDDEN},
        {"name": "round_2048", "kind": "round", "rows": 2048, "width": MLP},
        # The norms of a decode step of one row and of 128 rows (the deltas are partial sums), and of
        # a full-length prompt (an fp16 delta).
        {"name": "norm_1", "kind": "norm", "rows": 1, "width": HIDDEN, "splits": 4},
        {"name": "norm_128", "kind": "norm", "rows": 128, "width": HIDDEN, "splits": 8},
        {"name": "norm_2048", "kind": "norm", "rows": 2048, "width": HIDDEN, "splits": 0},
        # Decode steps: the SwiGLU projection of one row and of a serving batch, the down projection
        # of the full batch from fp16 activations.
        {"name": "project_swiglu_1", "kind": "project", "m": 1, "n": 2 * MLP, "k": HIDDEN, "out": "swiglu", "splits": 1, "half_x": False},
        {"name": "project_swiglu_64", "kind": "project", "m": 64, "n": 2 * MLP, "k": HIDDEN, "out": "swiglu", "splits": 1, "half_x": False},
        {"name": "project_down_128", "kind": "project", "m": 128, "n": HIDDEN, "k": MLP, "out": "partials", "splits": 4, "half_x": True},
        # A ragged product: no size a multiple of a tile, the last block of 128 cut.
        {"name": "project_ragged", "kind": "project", "m": 333, "n": 1004, "k": 1328, "out": "half", "splits": 1, "half_x": False},
        # A full-length prompt: the SwiGLU projection, its output in 8 bits for the down projection.
        {"name": "project_swiglu_2048", "kind": "project", "m": 2048, "n": 2 * MLP, "k": HIDDEN, "out": "swiglu_fp8", "splits": 1, "half_x": False},
        # q|k|v with RoPE and the cache write: a decode step of 37 sequences, a prompt of 2048 tokens.
        {"name": "qkv_37", "kind": "qkv", "m": 37, "k": HIDDEN},
        {"name": "qkv_2048", "kind": "qkv", "m": 2048, "k": HIDDEN},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over its logarithm."""
    value = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(hi, max(lo, value))


def draw(rng):
    kind = rng.choice(("round", "norm", "project", "project", "project", "qkv"))
    if kind == "round":
        return {"kind": kind, "rows": _log(rng, 1, 2048), "width": _log(rng, 64, MLP, 16)}
    if kind == "norm":
        splits = rng.choice((0, 1, 2, 3, 4, 8))
        return {"kind": kind, "rows": _log(rng, 1, 2048 if splits < 2 else 256), "width": _log(rng, 64, 4096, 16), "splits": splits}
    if kind == "qkv":
        return {"kind": kind, "m": _log(rng, 1, 2048), "k": _log(rng, 256, HIDDEN, 16)}
    out = rng.choice(("partials", "half", "swiglu", "swiglu_fp8"))
    case = {"kind": kind, "m": _log(rng, 1, 2048), "out": out}
    if out == "partials":  # a decode step's rows
        case["m"] = min(case["m"], _log(rng, 1, 128))
    case["n"] = _log(rng, 128, 2 * MLP if out.startswith("swiglu") else QKV, 32 if out == "swiglu_fp8" else 8)
    case["k"] = _log(rng, 128, HIDDEN if out.startswith("swiglu") else MLP, 16)
    case["splits"] = rng.choice((1, 2, 3, 4)) if out == "partials" and case["k"] >= 1024 else 1
    case["half_x"] = case["m"] <= 128 and out != "swiglu_fp8" and rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------------------


def _normal(gen, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float16, device=DEVICE).normal_(0.0, std, generator=gen)


def _activations(gen, rows, width):
    """N(0, 1) rows in which some channels are ten times as large, as in a model's residual stream."""
    channel = 1.0 + 9.0 * (torch.rand(width, device=DEVICE, generator=gen) < 0.01)
    return (_normal(gen, (rows, width)) * channel).half()


def _blocks(width):
    return -(-width // BLOCK)


def _eight_bits(x):
    """fp16 rows as an 8-bit row's values and scales, scales padded to a multiple of four a row."""
    values, powers = _round_plain(x.float())
    scales = torch.zeros((x.shape[0], (powers.shape[1] + 3) // 4 * 4), dtype=torch.uint8, device=DEVICE)
    scales[:, : powers.shape[1]] = powers
    return values, scales.view(torch.float8_e8m0fnu)


def _rope_table():
    angles = torch.arange(2048).float().unsqueeze(-1) * (1.0 / (10000.0 ** (torch.arange(0, DIM, 2).float() / DIM)))
    return torch.stack((angles.cos().half(), angles.sin().half()), dim=1).contiguous().to(DEVICE)


def _empty_eight_bits(rows, width):
    values = torch.empty((rows, width), dtype=torch.float8_e4m3fn, device=DEVICE)
    return values, torch.zeros((rows, (_blocks(width) + 3) // 4 * 4), dtype=torch.uint8, device=DEVICE).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    state = {"case": dict(case)}
    if kind == "round":
        state["x"] = _activations(gen, case["rows"], case["width"])
        state["values"], state["scales"] = _empty_eight_bits(case["rows"], case["width"])
    elif kind == "norm":
        rows, width, splits = case["rows"], case["width"], case["splits"]
        state["hidden"] = _activations(gen, rows, width)
        if splits:
            state["delta"] = torch.empty((splits, rows, width), device=DEVICE).normal_(0.0, 0.5 / math.sqrt(splits), generator=gen)
        else:
            state["delta"] = _normal(gen, (rows, width), 0.5)
        state["weight"] = (1.0 + 0.1 * _normal(gen, (width,)).float()).half()
        state["sum"] = torch.empty_like(state["hidden"])
        state["values"], state["scales"] = _empty_eight_bits(rows, width)
    else:
        m, k, n = case["m"], case["k"], case.get("n", QKV)
        x = _activations(gen, m, k)
        state["x"], state["x_scales"] = (x, None) if case.get("half_x") else _eight_bits(x)
        state["w"], state["w_scales"] = _eight_bits(_normal(gen, (n, k), 0.02))
        if kind == "qkv":
            blocks = m // SLOTS + 8
            state["pool"] = _normal(gen, (LAYERS, 2, blocks, SLOTS, KV_HEADS, DIM))
            state["slots"] = torch.randperm(blocks * SLOTS, device=DEVICE, generator=gen)[:m].contiguous()
            state["positions"] = torch.randint(0, 2048, (m,), device=DEVICE, generator=gen)
            state["table"] = _rope_table()
            state["layer"] = seed % LAYERS
            state["query"] = torch.empty((m, Q_HEADS, DIM), dtype=torch.float16, device=DEVICE)
        elif case["out"] == "partials":
            state["y"] = torch.empty((case["splits"], m, n), device=DEVICE)
        elif case["out"] == "swiglu_fp8":
            state["y"], state["y_scales"] = _empty_eight_bits(m, n // 2)
        else:
            state["y"] = torch.empty((m, n if case["out"] == "half" else n // 2), dtype=torch.float16, device=DEVICE)
    return state


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------


def _round_plain(y):
    """fp32 rows to e4m3 values and the biased exponents of their blocks' powers of two."""
    rows, width = y.shape
    padded = torch.zeros((rows, _blocks(width) * BLOCK), device=y.device)
    padded[:, :width] = y
    padded = padded.view(rows, -1, BLOCK)
    largest = padded.abs().amax(-1).double()  # next to a power of two, 32 bits of a logarithm are too few
    power = torch.ceil(torch.log2(largest / LARGEST)).clamp(min=-126.0)
    power = power + (largest > LARGEST * torch.exp2(power)).double()
    power = torch.where((largest <= LARGEST * torch.exp2(power - 1.0)) & (power > -126.0), power - 1.0, power)
    values = (padded * torch.exp2(-power).float().unsqueeze(-1)).view(rows, -1)[:, :width]
    return values.to(torch.float8_e4m3fn), (power + 127.0).to(torch.uint8)


def _values(eight, scales):
    """What 8-bit rows stand for, in fp32."""
    rows, width = eight.shape
    power = scales.view(torch.uint8)[:, : _blocks(width)].float() - 127.0
    return eight.float() * torch.exp2(power.double()).float().repeat_interleave(BLOCK, dim=1)[:, :width]


def _rounded(values, power):
    return {"values": values, "scales": power.view(torch.float8_e8m0fnu)}


def _split(case):
    """The columns at which the K splits begin, and the end: whole blocks, as even as they go."""
    blocks, splits = _blocks(case["k"]), case["splits"]
    return [min(case["k"], BLOCK * (s * blocks // splits)) for s in range(splits + 1)]


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "round":
        return _rounded(*_round_plain(state["x"].float()))
    if kind == "norm":
        delta = state["delta"]
        delta = delta.sum(0).half() if delta.ndim == 3 else delta
        total = (state["hidden"].float() + delta.float()).half()
        h = total.float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * state["weight"].float()
        return {"sum": total, **_rounded(*_round_plain(y))}
    x, x_scales = state["x"], state["x_scales"]
    if x_scales is None:
        x, power = _round_plain(x.float())
        x_scales = power
    x, w = _values(x, x_scales), _values(state["w"], state["w_scales"])
    if kind == "qkv":
        return _plain_qkv(state, x @ w.t())
    if case["out"] == "partials":
        at = _split(case)
        return torch.stack([x[:, a:b] @ w[:, a:b].t() for a, b in zip(at, at[1:])])
    y = x @ w.t()
    if case["out"] == "half":
        return y.half()
    gate, up = y.chunk(2, dim=1)
    y = gate / (1.0 + torch.exp(-gate)) * up
    return y.half() if case["out"] == "swiglu" else _rounded(*_round_plain(y))


def _plain_qkv(state, y):
    m = y.shape[0]
    heads = y.view(m, Q_HEADS + 2 * KV_HEADS, DIM)
    cos, sin = (state["table"].float()[state["positions"], i].unsqueeze(1) for i in range(2))
    rotated = heads[:, : Q_HEADS + KV_HEADS]
    low, high = rotated.chunk(2, dim=-1)
    rotated = torch.cat((low * cos - high * sin, high * cos + low * sin), dim=-1)
    cache = state["pool"][state["layer"]].view(2, -1, KV_HEADS, DIM)
    cache[0, state["slots"]] = rotated[:, Q_HEADS:].half()
    cache[1, state["slots"]] = heads[:, Q_HEADS + KV_HEADS :].half()
    return {"query": rotated[:, :Q_HEADS].half(), "cache": cache}


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------


def _own(state):
    from pagedcore_amd import _hip

    case = state["case"]
    kind = case["kind"]
    if kind == "round":
        _hip.quantize_fp8(state["values"], state["scales"], state["x"])
        return {"values": state["values"], "scales": state["scales"][:, : _blocks(case["width"])]}
    if kind == "norm":
        _hip.add_rms_norm_fp8(state["values"], state["scales"], state["sum"], state["hidden"], state["delta"], state["weight"], EPS)
        return {"sum": state["sum"], "values": state["values"], "scales": state["scales"][:, : _blocks(case["width"])]}
    if kind == "qkv":
        _hip.qkv_rope_append_fp8(
            state["query"], state["x"], state["x_scales"], state["w"], state["w_scales"], state["positions"], state["table"],
            pool=state["pool"], layer=state["layer"], slot_mapping=state["slots"],
        )
        return {"query": state["query"], "cache": state["pool"][state["layer"]].view(2, -1, KV_HEADS, DIM)}
    args = (state["y"], state["x"], state["x_scales"], state["w"], state["w_scales"])
    if case["out"] == "partials":
        _hip.gemm_fp8(*args, splits=case["splits"])
    elif case["out"] == "half":
        _hip.gemm_fp8(*args, epilogue=_hip.GEMM_HALF)
    elif case["out"] == "swiglu":
        _hip.gemm_fp8(*args, epilogue=_hip.GEMM_SWIGLU)
    else:
        _hip.gemm_fp8(*args, out_scales=state["y_scales"], epilogue=_hip.GEMM_SWIGLU_FP8)
        return {"values": state["y"], "scales": state["y_scales"][:, : _blocks(case["n"] // 2)]}
    return state["y"]


def run(state):
    with torch.inference_mode():
        return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------
# What a pass has to do, and its outputs in 64 bits
# ---------------------------------------------------------------------------------------


def work(case):
    eight = lambda rows, width: rows * (width + _blocks(width))  # noqa: E731
    if case["kind"] == "round":
        elements = case["rows"] * case["width"]
        return {"bytes": 2 * elements + eight(case["rows"], case["width"]), "flops": 3 * elements}
    if case["kind"] == "norm":
        elements = case["rows"] * case["width"]
        delta = 4 * case["splits"] if case["splits"] else 2
        return {
            "bytes": (4 + delta) * elements + 2 * case["width"] + eight(case["rows"], case["width"]),
            "flops": (8 + case["splits"]) * elements,
        }
    m, k, n = case["m"], case["k"], case.get("n", QKV)
    read = eight(n, k) + (2 * m * k if case.get("half_x") else eight(m, k))
    if case["kind"] == "qkv":
        written = m * (2 * QKV + 16 + 2 * DIM)  # outputs, and the token's position, slot and table row
    elif case["out"] == "partials":
        written = 4 * case["splits"] * m * n
    elif case["out"] == "swiglu_fp8":
        written = eight(m, n // 2)
    else:
        written = 2 * m * (n if case["out"] == "half" else n // 2)
    return {"bytes": read + written, "flops": 2 * m * n * k}


def _exact_round(y):
    """The definition in 64 bits: values on e4m3's grid, and the powers of two themselves."""
    rows, width = y.shape
    found, powers = torch.empty_like(y), torch.empty((rows, _blocks(width)), dtype=torch.float64, device=y.device)
    for b in range(_blocks(width)):
        part = y[:, BLOCK * b : BLOCK * (b + 1)]
        fraction, exponent = torch.frexp(part.abs().amax(1))  # fraction in [0.5, 1); 448 = 0.875 * 2^9
        exponent = torch.where(fraction == 0, -126, torch.clamp(exponent - 9 + (fraction > 0.875).int(), min=-126)).double()
        scaled = part / torch.exp2(exponent).unsqueeze(1)
        step = torch.exp2(torch.clamp(torch.frexp(scaled.abs())[1] - 1, min=-6).double() - 3.0)
        found[:, BLOCK * b : BLOCK * (b + 1)] = torch.round(scaled / step) * step
        powers[:, b] = torch.exp2(exponent)
    return {"values": found, "scales": powers}


def _exact_values(eight, scales):
    rows, width = eight.shape
    out = eight.double()
    power = torch.exp2(scales.view(torch.uint8).double() - 127.0)
    for b in range(_blocks(width)):
        out[:, BLOCK * b : BLOCK * (b + 1)] *= power[:, b : b + 1]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "round":
        return _exact_round(state["x"].double())
    if kind == "norm":
        delta = state["delta"].double()
        delta = delta.sum(0).half().double() if delta.ndim == 3 else delta
        total = (state["hidden"].double() + delta).half().double()
        y = total / torch.sqrt((total * total).sum(1, keepdim=True) / case["width"] + EPS) * state["weight"].double()
        return {"sum": total, **_exact_round(y)}
    if state["x_scales"] is None:
        rounded = _exact_round(state["x"].double())
        x = rounded["values"] * rounded["scales"].repeat_interleave(BLOCK, dim=1)[:, : case["k"]]
    else:
        x = _exact_values(state["x"], state["x_scales"])
    w = _exact_values(state["w"], state["w_scales"])
    if kind == "project" and case["out"] == "partials":
        at = _split(case)
        return torch.stack([torch.mm(x[:, a:b].contiguous(), w[:, a:b].t().contiguous()) for a, b in zip(at, at[1:])])
    y = torch.mm(x, w.t().contiguous())
    if kind == "qkv":
        m = case["m"]
        y = y.view(m, -1, DIM)
        c, s = state["table"].double()[state["positions"]].unbind(1)
        turned = y.clone()
        for head in range(Q_HEADS + KV_HEADS):
            a, b = y[:, head, : DIM // 2], y[:, head, DIM // 2 :]
            turned[:, head, : DIM // 2] = a * c - b * s
            turned[:, head, DIM // 2 :] = b * c + a * s
        cache = state["pool"][state["layer"]].double().view(2, -1, KV_HEADS, DIM)
        cache[0].index_copy_(0, state["slots"], turned[:, Q_HEADS : Q_HEADS + KV_HEADS])
        cache[1].index_copy_(0, state["slots"], turned[:, Q_HEADS + KV_HEADS :])
        return {"query": turned[:, :Q_HEADS], "cache": cache}
    if case["out"] == "half":
        return y
    half = case["n"] // 2
    y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y if case["out"] == "swiglu" else _exact_round(y)
