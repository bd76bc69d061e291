"""The 8-bit rows' oracle, and what the 8-bit entry points refuse, without a GPU."""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd import decoder as dec
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import KVAllocator


def _every_e4m3() -> torch.Tensor:
    return torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn)


def test_oracle_rounding_is_torchs_cast_up_to_448():
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16).double()
    x = x[x.abs() <= 448]
    assert torch.equal(ref.round_e4m3(x), x.to(torch.float8_e4m3fn).double())


def test_oracle_keeps_every_e4m3_value():
    v = _every_e4m3().double()
    kept = ref.round_e4m3(v)
    assert torch.equal(kept.nan_to_num(nan=1e9), v.nan_to_num(nan=1e9))


@pytest.mark.parametrize("most,s", [(448.0, 127), (448.0 + 2**-40, 128), (449.0, 128), (896.0, 128), (0.0, 1), (1.75, 119),
                                    (1.7500001, 120), (2.0**-24, 95), (65504.0, 135), (2.0**-126, 1)])
def test_oracle_exponents(most, s):
    assert ref.exponents(torch.tensor([most], dtype=torch.float64)).item() == s
    assert most <= 448 * 2.0 ** (s - 127) and (s == 1 or most > 448 * 2.0 ** (s - 128))


def test_oracle_splits_are_whole_blocks():
    assert ref.split_columns(5632, 8) == [128 * b for b in (0, 5, 11, 16, 22, 27, 33, 38, 44)]
    assert ref.split_columns(400, 3) == [0, 128, 256, 400]


@pytest.mark.parametrize("width", [1, 16, 127, 128, 129, 512, 513, 2048, 5632, 1 << 22])
def test_scale_stride(width):
    stride = _hip.load().pc_fp8_scale_stride(width)
    assert stride == _hip.fp8_scale_stride(width)
    assert stride % 4 == 0 and stride >= ref.blocks(width) > stride - 4


@pytest.mark.parametrize("width", [0, -1, (1 << 22) + 1])
def test_scale_stride_of_no_width(width):
    assert _hip.load().pc_fp8_scale_stride(width) == 0


P = 4096  # an aligned address that is never read: every call below is refused


def _refused(status: int, needle: bytes) -> None:
    text = _hip.load().pc_last_error()
    assert status == 1 and needle in text, (status, text)


@pytest.mark.parametrize("change,needle", [
    ({"values": None}, b"null pointer"), ({"scales": None}, b"null pointer"), ({"x": None}, b"null pointer"),
    ({"width": 0}, b"width"), ({"width": 24}, b"multiple of 16"), ({"width": (1 << 22) + 16}, b"width"),
    ({"rows": -1}, b"negative"), ({"stride": 48}, b"x_stride"), ({"stride": 68}, b"x_stride"),
    ({"x": P + 8}, b"aligned"), ({"values": P + 8}, b"aligned"), ({"scales": P + 2}, b"aligned"),
    ({"rows": 1 << 60}, b"too large"), ({"rows": 1 << 29}, b"too large"),
])
def test_quantize_refuses(change, needle):
    a = {"values": P, "scales": P, "x": P, "stride": 64, "rows": 1, "width": 64, **change}
    _refused(_hip.load().pc_quantize_fp8(a["values"], a["scales"], a["x"], a["stride"], a["rows"], a["width"], None), needle)


def test_no_rows_are_no_work():
    lib = _hip.load()
    assert lib.pc_quantize_fp8(None, None, None, 64, 0, 64, None) == 0
    assert lib.pc_add_rms_norm_fp8(None, None, None, None, None, None, 0, 64, 1e-5, None) == 0
    assert lib.pc_add_rms_norm_parts_fp8(None, None, None, None, None, 2, None, 0, 64, 1e-5, None) == 0


@pytest.mark.parametrize("change,needle", [
    ({"values": None}, b"null pointer"), ({"scales": None}, b"null pointer"), ({"hidden": None}, b"null pointer"),
    ({"weight": None}, b"null pointer"), ({"hidden_out": None}, b"hidden_out"), ({"width": 24}, b"multiple of 16"),
    ({"width": 8208}, b"width"), ({"width": 0}, b"width"), ({"rows": -1}, b"rows"), ({"rows": 1 << 24}, b"rows"),
    ({"eps": -1.0}, b"eps"), ({"eps": float("nan")}, b"eps"), ({"hidden": P + 2}, b"aligned"), ({"delta": P + 4}, b"aligned"),
    ({"hidden_out": P + 8}, b"aligned"), ({"scales": P + 1}, b"aligned"), ({"values": P + 4}, b"aligned"),
])
@pytest.mark.parametrize("parts", [False, True])
def test_norm_refuses(change, needle, parts):
    a = {"values": P, "scales": P, "hidden_out": P, "hidden": P, "delta": P, "weight": P, "rows": 1, "width": 64, "eps": 1e-5, **change}
    head = (a["values"], a["scales"], a["hidden_out"], a["hidden"], a["delta"])
    tail = (a["weight"], a["rows"], a["width"], a["eps"], None)
    lib = _hip.load()
    _refused(lib.pc_add_rms_norm_parts_fp8(*head, 2, *tail) if parts else lib.pc_add_rms_norm_fp8(*head, *tail), needle)


@pytest.mark.parametrize("delta,splits,needle", [(None, 2, b"null pointer"), (P, 0, b"splits"), (P, 65, b"splits")])
def test_norm_parts_refuses(delta, splits, needle):
    _refused(_hip.load().pc_add_rms_norm_parts_fp8(P, P, P, P, delta, splits, P, 1, 64, 1e-5, None), needle)


@pytest.mark.parametrize("change,needle", [
    ({"out": None}, b"null pointer"), ({"x": None}, b"null pointer"), ({"w": None}, b"null pointer"), ({"w_scales": None}, b"null pointer"),
    ({"m": 0}, b"m = 0"), ({"m": 65537}, b"m = 65537"), ({"n": 0}, b"n must"), ({"n": -4}, b"n must"),
    ({"k": 0}, b"k = 0"), ({"k": 24}, b"k = 24"), ({"k": (1 << 22) + 16}, b"k = "),
    ({"n": 6}, b"multiple of 4"), ({"n": 4, "epilogue": 2}, b"multiple of 8"), ({"n": 48, "epilogue": 4, "out_scales": P}, b"multiple of 32"),
    ({"m": 129, "epilogue": 0}, b"partial sums take up to 128"), ({"m": 129, "x_scales": None}, b"fp16 x takes up to 128"),
    ({"epilogue": 4, "x_scales": None, "out_scales": P}, b"8-bit x"),
    ({"epilogue": 3}, b"unknown epilogue"), ({"epilogue": 5}, b"unknown epilogue"), ({"epilogue": -1}, b"unknown epilogue"),
    ({"epilogue": 4}, b"out_scales"), ({"out_scales": P}, b"out_scales"),
    ({"splits": 2}, b"only partial sums"), ({"splits": 0}, b"only partial sums"),
    ({"epilogue": 0, "splits": 0}, b"splits"), ({"epilogue": 0, "splits": 65}, b"splits"), ({"epilogue": 0, "splits": 3, "k": 256}, b"2 blocks"),
    ({"out": P + 8}, b"aligned"), ({"x": P + 8}, b"aligned"), ({"w": P + 4}, b"aligned"), ({"x_scales": P + 2}, b"aligned"),
    ({"w_scales": P + 1}, b"aligned"), ({"n": 1 << 20, "k": 4096}, b"too large"), ({"m": 65536, "k": 65536}, b"too large"),
    ({"epilogue": 0, "splits": 17, "k": 2048}, b"16 blocks"), ({"m": 65536, "n": 1 << 16, "k": 16}, b"too large"),
])
def test_gemm_refuses(change, needle):
    a = {"out": P, "out_scales": None, "x": P, "x_scales": P, "w": P, "w_scales": P, "m": 8, "n": 64, "k": 128, "splits": 1,
         "epilogue": 1, **change}
    _refused(_hip.load().pc_gemm_fp8(*(a[name] for name in ("out", "out_scales", "x", "x_scales", "w", "w_scales", "m", "n", "k",
                                                             "splits", "epilogue")), None), needle)


@pytest.mark.parametrize("change,needle", [
    ({"query": None}, b"null pointer"), ({"x": None}, b"null pointer"), ({"w": None}, b"null pointer"), ({"positions": None}, b"null pointer"),
    ({"table": None}, b"null pointer"), ({"m": 0}, b"m = 0"), ({"m": 129, "x_scales": None}, b"fp16 x"), ({"k": 40}, b"k = 40"),
    ({"k": (1 << 18) + 16}, b"k = "), ({"table_rows": 0}, b"rope_positions"), ({"slots": None}, b"both"), ({"pool": None}, b"both"),
    ({"blocks": 0}, b"num_blocks"), ({"blocks": 1 << 31}, b"num_blocks"), ({"layer": 22}, b"layer"), ({"layer": -1}, b"layer"),
    ({"query": P + 8}, b"aligned"), ({"key": P + 8}, b"aligned"), ({"pool": P + 8}, b"aligned"), ({"w": P + 8}, b"aligned"),
    ({"x_scales": P + 2}, b"aligned"),
])
def test_qkv_refuses(change, needle):
    a = {"query": P, "key": P, "value": P, "x": P, "x_scales": P, "w": P, "w_scales": P, "m": 2, "k": 64, "positions": P, "table": P,
         "table_rows": 16, "pool": P, "blocks": 4, "layer": 0, "slots": P, **change}
    _refused(_hip.load().pc_qkv_rope_append_fp8(*(a[name] for name in (
        "query", "key", "value", "x", "x_scales", "w", "w_scales", "m", "k", "positions", "table", "table_rows", "pool", "blocks",
        "layer", "slots")), None), needle)


def test_the_binding_takes_gpu_tensors_only():
    values, scales = _hip.empty_fp8(2, 64, torch.device("cpu"))
    assert values.shape == (2, 64) and scales.shape == (2, 4)
    x = torch.zeros((2, 64), dtype=torch.float16)
    with pytest.raises(Exception, match="GPU|CUDA|HIP|NVIDIA|device"):
        _hip.quantize_fp8(values, scales, x)


def test_layers_of_both_kinds_are_refused():
    """Half a model in 8 bits is no model: refused before anything is staged."""
    weights = dec.random_weights(device="cpu", layers=2, vocab=8, intermediate=16)
    some = torch.zeros((1, 16), dtype=torch.float16)
    rows = dec.Fp8Rows(some, some)
    eight = dec.Fp8LayerWeights(weights.layers[0].input_norm, rows, rows, weights.layers[0].post_attention_norm, rows, rows)
    mixed = dec.TinyLlamaWeights(weights.embedding, weights.layers[:1] * 21 + (eight,), weights.final_norm, weights.lm_head)
    allocator = KVAllocator(torch.zeros((22, 2, 2, 16, 4, 64), dtype=torch.float16))
    allocator.create(KVReservation(RequestId("a"), 1))
    with pytest.raises(ValueError, match="all in 8 bits"):
        dec.prefill_paged(torch.ones((1, 3), dtype=torch.int64), mixed, allocator, RequestId("a"))
    with pytest.raises(ValueError, match="all in 8 bits"):
        dec.decode_paged(torch.ones((1, 1), dtype=torch.int64), mixed, allocator, (RequestId("a"),))
