"""Every kernel of the 8-bit projections against the definition in 64 bits, at the sizes of tests/fp8_sizes.py.

Tolerances. The operands are whole numbers times powers of two, chosen so that every sum is exact in fp32 in any order and
no product of eight lies 2^-13 below another: products are compared bit for bit. SwiGLU in fp32 is
then off by, in steps of 2^-24 relative: two each for the hardware's exponential and reciprocal (one ulp), one each for
1 + e, gate * r and * up, and |gate| each for log2(e)'s own rounding and that of its product with the gate: 8 + 2 |gate| holds
them. Its outputs add half a step: 2^-11 relative (fp16; 2^-25 below its normals), 2^-4 (e4m3).
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp8_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd import decoder as dec
from tests.fp8_sizes import HALF, PARTIALS, ROPE, SWIGLU, SWIGLU_FP8, sizes
from tests.test_gpu_fp8 import STEP32, _check_rounded, _gen, _guarded, _intact

pytestmark = pytest.mark.gpu


def _eight_rows(device, rows, width, seed, power=0):
    """8-bit rows of whole numbers from -4 to 4 times 2^power, 2^(power - 1) or 2^(power + 1), by block (random bytes past the
    blocks)."""
    gen = _gen(device, seed)
    values = torch.randint(-4, 5, (rows, width), device=device, generator=gen).half().to(torch.float8_e4m3fn)
    scales = torch.randint(126 + power, 129 + power, (rows, _hip.fp8_scale_stride(width)), device=device, generator=gen)
    return values, scales.to(torch.uint8).view(torch.float8_e8m0fnu)


def _half_rows(device, rows, width, seed):
    """fp16 rows, and what they stand for once rounded: magnitudes from 16 to 31 (five bits, e4m3 keeps four) times a power
    of two per row, one in eight 0, and some blocks of zeros."""
    gen = _gen(device, seed)
    draw = lambda lo, hi, *shape: torch.randint(lo, hi, shape, device=device, generator=gen)  # noqa: E731
    x = draw(16, 32, rows, width) * (2 * draw(0, 2, rows, width) - 1) * (draw(0, 8, rows, width) > 0)
    for row in range(0, rows, 5):
        x[row, : min(128, width // 2)] = 0
    x = (x * torch.exp2(draw(-3, 4, rows, 1).float())).half()
    values, s = ref.round_rows(x.cpu().double())
    assert not torch.equal(values * ref.spread(s, width), x.cpu().double())
    return x, ref.stands_for(values, s).to(device)


def _stands(values, scales):
    return ref.stands_for(values, scales.view(torch.uint8).long())


def _operands(device, half_x, m, n, k, unit):
    """(x, its scales or None, w, its scales, x and w in 64 bits); unit: scaled so that outputs are about 1."""
    rms = (24.0 * 2.7 * 1.3 if half_x else 6.7 * 1.75) * math.sqrt(k)
    w, ws = _eight_rows(device, n, k, seed=n + k, power=-round(math.log2(rms)) if unit else 0)
    if half_x:
        x, x64 = _half_rows(device, m, k, seed=m)
        return x, None, w, ws, x64, _stands(w, ws)
    x, xs = _eight_rows(device, m, k, seed=m)
    return x, xs, w, ws, _stands(x, xs), _stands(w, ws)


def _cases(form):
    return [pytest.param(h, *size, id="-".join(map(str, size)) + "-fp16" * h)
            for h in (0, 1) if (form, h) != (SWIGLU_FP8, 1) for size in sizes(form, h)]


@pytest.mark.parametrize("half_x,m,n,k,splits", _cases(PARTIALS))
def test_partial_sums_are_exact(device, half_x, m, n, k, splits):
    x, xs, w, ws, x64, w64 = _operands(device, half_x, m, n, k, unit=False)
    out, store = _guarded((splits, m, n), torch.float32, device)
    _hip.gemm_fp8(out, x, xs, w, ws, splits=splits)
    at = ref.split_columns(k, splits)
    for s, (a, b) in enumerate(zip(at, at[1:])):
        assert torch.equal(out[s].double(), x64[:, a:b] @ w64[:, a:b].t()), s
    _intact(store)


@pytest.mark.parametrize("half_x,m,n,k,splits", _cases(HALF))
def test_fp16_products_are_exact(device, half_x, m, n, k, splits):
    x, xs, w, ws, x64, w64 = _operands(device, half_x, m, n, k, unit=True)
    out, store = _guarded((m, n), torch.float16, device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    assert torch.equal(out, (x64 @ w64.t()).half())
    _intact(store)


def _swiglu(x64, w64):
    """silu(gate) * up in 64 bits, and how far fp32 may be off."""
    gate, up = (x64 @ w64.t()).chunk(2, dim=1)
    exact = gate / (1.0 + torch.exp(-gate)) * up
    return exact, exact.abs() * (8.0 + 2.0 * gate.abs()) * STEP32


@pytest.mark.parametrize("half_x,m,n,k,splits", _cases(SWIGLU))
def test_swiglu(device, half_x, m, n, k, splits):
    x, xs, w, ws, x64, w64 = _operands(device, half_x, m, n, k, unit=True)
    exact, slack = _swiglu(x64, w64)
    out, store = _guarded((m, n // 2), torch.float16, device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_SWIGLU)
    assert ((out.double() - exact).abs() <= slack + (exact.abs() + slack) * 2.0**-11 + 2.0**-25).all()
    _intact(store)


@pytest.mark.parametrize("half_x,m,n,k,splits", _cases(SWIGLU_FP8))
def test_swiglu_to_eight_bits(device, half_x, m, n, k, splits):
    x, xs, w, ws, x64, w64 = _operands(device, half_x, m, n, k, unit=True)
    exact, slack = _swiglu(x64, w64)
    out, store = _guarded((m, n // 2), torch.float8_e4m3fn, device)
    scales, scale_store = _guarded((m, _hip.fp8_scale_stride(n // 2)), torch.float8_e8m0fnu, device)
    _hip.gemm_fp8(out, x, xs, w, ws, out_scales=scales, epilogue=_hip.GEMM_SWIGLU_FP8)
    _check_rounded(out, scales, exact.cpu(), slack.cpu())
    _intact(store)
    _intact(scale_store)
    assert (scales.view(torch.uint8)[:, ref.blocks(n // 2) :] == 0x5A).all()


def _same(a, b):
    """Equal, NaN for NaN."""
    assert torch.equal(a.isnan(), b.isnan())
    assert torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


@pytest.mark.parametrize("half_x,m,n,k,splits", _cases(ROPE))
def test_q_k_v_is_rotated_and_written(device, half_x, m, n, k, splits):
    """The exact product's fp16 values through rope_kv_append, bit for bit: positions from the first to the last of the
    table, some outside it (NaN q and k, nothing written to the pool), slots from the first to the last and some outside it."""
    x, xs, w, ws, x64, w64 = _operands(device, half_x, m, n, k, unit=True)
    table = dec.rope_table(device)
    gen = _gen(device, m)
    positions = torch.randint(0, 2048, (m,), device=device, generator=gen)
    blocks = m // 16 + 2
    slots = torch.randperm(blocks * 16, device=device, generator=gen)[:m].contiguous()
    positions[0], slots[0] = 2047, blocks * 16 - 1
    slots[1:][slots[1:] == blocks * 16 - 1] = 0 if not (slots == 0).any() else -1
    positions[m - 1] = 2048
    if m > 8:
        positions[1], positions[3] = -1, 1 << 40
        slots[5], slots[6], slots[7] = -1, blocks * 16, 1 << 40
        positions[8] = 0
    pools = [torch.full((22, 2, blocks, 16, 4, 64), 3.0, dtype=torch.float16, device=device) for _ in range(2)]
    outs, stores = zip(*(_guarded((m, heads, 64), torch.float16, device) for heads in (32, 4, 4)))
    _hip.qkv_rope_append_fp8(outs[0], x, xs, w, ws, positions, table, key_out=outs[1], value_out=outs[2], pool=pools[0], layer=21,
                             slot_mapping=slots)
    expected = [torch.empty_like(out) for out in outs]
    qkv = (x64 @ w64.t()).half()
    _hip.rope_kv_append(expected[0], qkv, positions, table, key_out=expected[1], value_out=expected[2], pool=pools[1], layer=21,
                        slot_mapping=slots)
    for got, want, store in zip(outs, expected, stores):
        _same(got, want)
        _intact(store)
    assert torch.equal(pools[0].view(torch.int16), pools[1].view(torch.int16))
    outside = (positions < 0) | (positions >= 2048)
    assert outside.any() and torch.equal(outs[0].isnan().flatten(1).all(1), outside) and torch.equal(outs[1].isnan().flatten(1).all(1), outside)
    assert not outs[2].isnan().any()
    written = (pools[0][21, 0].view(-1, 256) != 3.0).any(1).sum()
    assert written == (~outside & (slots >= 0) & (slots < blocks * 16)).sum()
    assert (pools[0][:21] == 3.0).all()


def test_norms_leave_what_lies_around_their_outputs(device):
    gen = _gen(device, 3)
    for rows, width, splits in ((3, 112, 0), (5, 2064, 2), (1, 2048, 4), (2, 8192, 11)):
        hidden = torch.randn((rows, width), device=device, generator=gen).half()
        delta = torch.randn((splits, rows, width), device=device, generator=gen) if splits else hidden.clone()
        weight = torch.ones(width, dtype=torch.float16, device=device)
        values, store = _guarded((rows, width), torch.float8_e4m3fn, device)
        scales, scale_store = _guarded((rows, _hip.fp8_scale_stride(width)), torch.float8_e8m0fnu, device)
        total, sum_store = _guarded((rows, width), torch.float16, device)
        _hip.add_rms_norm_fp8(values, scales, total, hidden, delta, weight)
        for around in (store, scale_store, sum_store):
            _intact(around)
        assert (scales.view(torch.uint8)[:, ref.blocks(width) :] == 0x5A).all()
        assert (total.double() - hidden.double() - (delta.double().sum(0) if splits else delta.double())).abs().max() < 0.1


def test_graphs_replayed_on_two_streams_at_once(device):
    """Two captured chains of a layer's 8-bit launches, replayed side by side on new inputs: each replay equals its eager calls."""
    def chain(m, width, seed):
        make = lambda *shape: torch.empty(shape, dtype=torch.float16, device=device)  # noqa: E731
        hidden, weight = make(m, 2048), torch.ones(2048, dtype=torch.float16, device=device)
        gate_up, down = _eight_rows(device, 2 * width, 2048, seed, -9), _eight_rows(device, 2048, width, seed + 1, -7)

        def run():
            x, xs = _hip.empty_fp8(m, 2048, device)
            _hip.add_rms_norm_fp8(x, xs, None, hidden, None, weight)
            a, a_s = _hip.empty_fp8(m, width, device)
            _hip.gemm_fp8(a, x, xs, *gate_up, out_scales=a_s, epilogue=_hip.GEMM_SWIGLU_FP8)
            y, total = make(m, 2048), make(m, 2048)
            _hip.gemm_fp8(y, a, a_s, *down, epilogue=_hip.GEMM_HALF)
            _hip.add_rms_norm_fp8(x, xs, total, hidden, y, weight)
            return y, total, x.view(torch.uint8)
        return hidden, run

    sides = [chain(150, 272, 40), chain(333, 1024, 50)]
    for hidden, run in sides:
        hidden.normal_()
        run()
    graphs = [dec.capture_graph(run, device) for _, run in sides]
    streams = [torch.cuda.Stream() for _ in sides]
    for turn in range(4):
        for i, (hidden, _) in enumerate(sides):
            hidden.normal_(generator=_gen(device, 10 * turn + i))
        torch.cuda.synchronize()
        for _ in range(3):
            for stream, (graph, _) in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, run), (_, held) in zip(sides, graphs):
            for got, expected in zip(held, run()):
                assert torch.equal(got.view(torch.uint8), expected.view(torch.uint8))
