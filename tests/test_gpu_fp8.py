"""The 8-bit rows and their projections on the GPU against their definition in 64 bits.

Tolerances. Rounding rows that are given is exact, so it is compared bit for bit. A projection's
fp32 sums are compared exactly where every partial sum is exact (small whole numbers), in any order;
on normal data a sum of k products is off by at most k roundings of 2^-24 of S = sum |x||w|. The 8-bit matrix
instruction (every form but the fp32 partial sums) aligns eight products to the largest, 2^e <= |p|, and
drops each one's bits below 2^(e - 13): at most 7 * 2^-13 of the group's largest product, added over the groups.
Outputs add half a step: 2^-11 relative (fp16; 2^-25 below its normals), 2^-4 (e4m3; 2^-10 of the
scale below its normals).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd.decoder import rope_table

pytestmark = pytest.mark.gpu

STEP32 = 2.0**-24


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _normal(device, shape, seed, std=1.0):
    return torch.empty(shape, dtype=torch.float16, device=device).normal_(0.0, std, generator=_gen(device, seed))


def _eight(x):
    """x (fp16, on the GPU) as the kernel rounds it."""
    values, scales = _hip.empty_fp8(x.shape[0], x.shape[1], x.device)
    _hip.quantize_fp8(values, scales, x)
    return values, scales


def _stands(values, scales):
    return ref.stands_for(values.cpu(), scales.cpu().view(torch.uint8).long())


def _same(got, expected):
    """Equal, NaN for NaN."""
    got, expected = got.cpu().double(), expected.cpu().double()
    assert torch.equal(got.isnan(), expected.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), expected.nan_to_num(nan=0.0))


def _same_bits(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _check_rows(values, scales, x):
    """values, scales are x (float64, CPU) rounded, exactly."""
    expected, s = ref.round_rows(x)
    assert torch.equal(scales.cpu().view(torch.uint8)[:, : s.shape[1]].long(), s)
    _same(values, expected)


def _check_rounded(values, scales, y, slack):
    """values, scales are rows within `slack` (absolute, per element) of y rounded to 8 bits."""
    s = scales.cpu().view(torch.uint8)[:, : ref.blocks(y.shape[1])].long()
    power = torch.exp2(s.double() - 127.0)
    most, least = ref.largest(y.abs() + slack), ref.largest((y.abs() - slack).clamp(min=0.0))
    assert (power * 448.0 >= least).all() and ((power * 224.0 < most) | (s == 1)).all()
    spread = ref.spread(s, y.shape[1])
    got = values.cpu().double() * spread
    half = ref.step((y.abs() + slack) / spread) / 2 * spread
    assert ((got - y).abs() <= half + slack).all(), ((got - y).abs() - half - slack).max()


# ---------------------------------------------------------------------------------------
# Rounding rows
# ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,width", [(1, 16), (1, 2048), (3, 128), (5, 144), (2, 112), (37, 640), (7, 5632), (1, 32768), (300, 272)])
def test_quantize_is_exact(device, rows, width):
    x = _normal(device, (rows, width), seed=rows + width)
    x *= torch.exp2(torch.randint(-20, 12, (rows, 1), device=device, generator=_gen(device, 1)).half())
    values, scales = _eight(x)
    _check_rows(values, scales, x.cpu().double())


def test_quantize_every_fp16(device):
    """Every fp16 value beside each power of two that sets another scale; infinities and NaN become NaN
    and leave the rest alone."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    finite = every[torch.isfinite(every)]
    lists = [every.view(512, 128)]
    for top in (2.0**-24, 2.0**-10, 0.25, 1.0, 448.0, 449.0, 65504.0):
        small = finite[finite.abs() <= top]
        small = small[: small.numel() // 112 * 112].view(-1, 112)
        lists.append(torch.cat((torch.full((small.shape[0], 16), top, dtype=torch.float16), small), dim=1))
    x = torch.cat(lists).to(device)
    values, scales = _eight(x)
    _check_rows(values, scales, x.cpu().double())


def test_quantize_zero_and_nonfinite_blocks(device):
    x = torch.zeros((4, 256), dtype=torch.float16)
    x[1, 3], x[1, 130] = float("inf"), 2.0
    x[2, :128] = float("nan")
    x[3, 200], x[3, 201] = -float("inf"), -7.0
    values, scales = _eight(x.to(device))
    _check_rows(values, scales, x.double())
    assert scales.cpu().view(torch.uint8)[0, :2].tolist() == [1, 1]


def test_quantize_strided_rows_and_untouched_neighbours(device):
    wide = _normal(device, (6, 400), seed=2)
    x = wide[:, 8:280]
    store = torch.full((8, 272), 0x55, dtype=torch.uint8, device=device)
    scale_store = torch.full((8, 4), 0xAA, dtype=torch.uint8, device=device)
    values, scales = store[1:7].view(torch.float8_e4m3fn), scale_store[1:7].view(torch.float8_e8m0fnu)
    _hip.quantize_fp8(values, scales, x)
    _check_rows(values, scales, x.cpu().double())
    assert (store[[0, 7]] == 0x55).all() and (scale_store[[0, 7]] == 0xAA).all()
    assert (scale_store[:, 3] == 0xAA).all()  # the bytes past the blocks are not written


def test_no_rows(device):
    values, scales = _eight(torch.empty((0, 64), dtype=torch.float16, device=device))
    assert values.shape == (0, 64) and scales.shape == (0, 4)


# ---------------------------------------------------------------------------------------
# Residual add + RMSNorm
# ---------------------------------------------------------------------------------------


def _norm(hidden, delta, weight, hidden_out, eps=1e-5):
    values, scales = _hip.empty_fp8(*hidden.shape, hidden.device)
    _hip.add_rms_norm_fp8(values, scales, hidden_out, hidden, delta, weight, eps)
    return values, scales


@pytest.mark.parametrize("rows,width", [(1, 16), (1, 2048), (3, 112), (37, 2048), (5, 2064), (2, 4096), (3, 5632), (2, 8192), (130, 256)])
@pytest.mark.parametrize("splits", [None, 0, 1, 2, 3, 4, 8, 11])
def test_norm(device, rows, width, splits):
    hidden = _normal(device, (rows, width), seed=rows)
    weight = (1 + 0.1 * _normal(device, (width,), seed=5).float()).half()
    before = hidden.clone()
    if splits is None:
        delta, added, out = None, None, None
    elif splits == 0:
        delta = _normal(device, (rows, width), seed=6)
        added, out = delta.cpu(), torch.empty_like(hidden)
    else:
        delta = torch.empty((splits, rows, width), device=device).normal_(generator=_gen(device, 7))
        added, out = delta[0].cpu(), torch.empty_like(hidden)
        for s in range(1, splits):
            added = added + delta[s].cpu()  # fp32, in split order
        added = added.half()
    values, scales = _norm(hidden, delta, weight, out)
    total, y = ref.add_rms_norm(before.cpu(), added, weight.cpu(), 1e-5)
    if out is not None:
        assert torch.equal(out.cpu().double(), total)
    assert torch.equal(hidden, before)
    # fp32: a sum of `width` squares in a tree of at most 32 + 10 additions, then four more roundings of
    # the norm and three of the product; the root halves what lies under it.
    _check_rounded(values, scales, y, y.abs() * 30 * STEP32)
    # in place
    again = hidden.clone()
    values2, scales2 = _norm(again, delta, weight, None if delta is None else again)
    _same_bits(values2, values)
    assert torch.equal(again, hidden if out is None else out)


def test_norm_edges(device):
    """A row of zeros, a single large element, rows with infinities and NaN (all NaN, and no other row)."""
    hidden = torch.zeros((5, 256), dtype=torch.float16)
    hidden[1, 77] = 60000.0
    hidden[2, 1], hidden[3, 200] = float("inf"), float("nan")
    hidden[4] = 2.0**-24
    weight = torch.ones(256, dtype=torch.float16)
    out = torch.empty((5, 256), dtype=torch.float16, device=device)
    values, scales = _norm(hidden.to(device), None, weight.to(device), out)
    assert torch.equal(out.cpu().view(torch.int16), hidden.view(torch.int16))
    _, y = ref.add_rms_norm(hidden, None, weight, 1e-5)
    keep = [0, 1, 4]
    _check_rounded(values[keep], scales[keep], y[keep], y[keep].abs() * 30 * STEP32)
    assert values[3].float().isnan().all()
    assert values[2].float().isnan()[1] and (values[2].float().nan_to_num(nan=0.0) == 0).all()


# ---------------------------------------------------------------------------------------
# Projections
# ---------------------------------------------------------------------------------------

SIZES = [  # (m, n, k): rows of every tile's edge, columns and K that end inside a tile, a block, a 16-byte chunk
    (1, 4, 16), (1, 64, 128), (2, 36, 112), (15, 100, 144), (16, 32, 256), (17, 132, 640), (32, 96, 1328), (33, 260, 512),
    (48, 64, 2048), (64, 320, 1024), (65, 68, 400), (127, 128, 272), (128, 256, 1152), (129, 128, 128), (130, 4, 16),
    (160, 260, 144), (200, 132, 1328), (257, 384, 640), (300, 1004, 400),
]


def _whole_rows(device, rows, width, seed):
    """8-bit rows of whole numbers from -4 to 4 with scales of 1/2, 1 and 2 (random bytes past the blocks)."""
    gen = _gen(device, seed)
    values = torch.randint(-4, 5, (rows, width), device=device, generator=gen).float().to(torch.float8_e4m3fn)
    scales = torch.randint(126, 129, (rows, _hip.fp8_scale_stride(width)), device=device, generator=gen).to(torch.uint8)
    return values, scales.view(torch.float8_e8m0fnu)


def _guarded(shape, dtype, device):
    """(an output, the storage around it): eight rows' worth of marked bytes on both sides."""
    size = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    store = torch.full((size + 2048,), 0x5A, dtype=torch.uint8, device=device)
    return store[1024 : 1024 + size].view(dtype).view(shape), store


def _intact(store):
    assert (store[:1024] == 0x5A).all() and (store[-1024:] == 0x5A).all()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_of_whole_numbers_are_exact(device, m, n, k):
    """|sums| < 2^24 quarters: exact in fp32 in any order, on the 8-bit instruction too (products of 2^-2 to
    2^6 within its 13 bits)."""
    x, xs = _whole_rows(device, m, k, seed=m)
    w, ws = _whole_rows(device, n, k, seed=n + 1000)
    expected = _stands(x, xs) @ _stands(w, ws).t()
    out, store = _guarded((m, n), torch.float16, device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    assert torch.equal(out.cpu(), expected.half())
    _intact(store)
    if m > _hip.FP8_STREAM_ROWS:
        return
    for splits in sorted({1, 2, 3, 5, ref.blocks(k)}):
        if splits > min(ref.blocks(k), 64):
            continue
        parts, store = _guarded((splits, m, n), torch.float32, device)
        _hip.gemm_fp8(parts, x, xs, w, ws, splits=splits)
        at = ref.split_columns(k, splits)
        for s in range(splits):
            span = slice(at[s], at[s + 1])
            # blocks stay whole, so a split's columns keep their scales
            first = at[s] // ref.BLOCK
            xe = ref.stands_for(x[:, span].cpu(), xs.cpu().view(torch.uint8)[:, first:].long())
            we = ref.stands_for(w[:, span].cpu(), ws.cpu().view(torch.uint8)[:, first:].long())
            assert torch.equal(parts[s].cpu().double(), xe @ we.t()), (splits, s)
        _intact(store)


def _aligned_loss(x, w):
    """Bound of what the 8-bit instruction drops: over groups of eight columns, 7 * 2^-13 of the largest product."""
    m, k = x.shape
    pad = -k % 8
    xa = torch.nn.functional.pad(x.abs(), (0, pad)).view(m, -1, 8).float()
    wa = torch.nn.functional.pad(w.abs(), (0, pad)).view(w.shape[0], -1, 8).float()
    total = torch.zeros((m, w.shape[0]))
    for i in range(0, m, 16):
        total[i : i + 16] = (xa[i : i + 16, None] * wa[None]).amax(-1).sum(-1)
    return total.double() * 7 * 2.0**-13


def _sum_slack(x, w):
    """Bound of a product's error in fp32."""
    return (x.abs() @ w.abs().t()) * x.shape[1] * STEP32


@pytest.mark.parametrize("m,n,k", [s for s in SIZES if s[1] * s[2] >= 8000])
def test_products_of_normal_data(device, m, n, k):
    x, xs = _eight(_normal(device, (m, k), seed=m + 1))
    w, ws = _eight(_normal(device, (n, k), seed=n + 2, std=0.02))
    x64, w64 = _stands(x, xs), _stands(w, ws)
    y = x64 @ w64.t()
    exact = _sum_slack(x64, w64)
    slack = exact + _aligned_loss(x64, w64)
    out = torch.empty((m, n), dtype=torch.float16, device=device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    assert ((out.cpu().double() - y).abs() <= slack + (y.abs() + slack) * 2.0**-11 + 2.0**-25).all()
    if m <= _hip.FP8_STREAM_ROWS:
        parts = torch.empty((1, m, n), device=device)
        _hip.gemm_fp8(parts, x, xs, w, ws)
        assert ((parts[0].cpu().double() - y).abs() <= exact).all()
        # fp32 sums: the matrix instruction's 13 bits would show here (1.5e-5)
        assert (parts[0].cpu().double() - y).norm() <= 2e-6 * y.norm()


SWIGLU_SIZES = [(1, 8, 16), (3, 64, 128), (16, 72, 400), (33, 256, 1152), (64, 544, 272), (100, 320, 512), (128, 64, 640),
                (129, 264, 144), (150, 512, 1328), (260, 96, 256), (300, 736, 400)]


def _swiglu_slack(x64, w64, y):
    """Error of silu(gate) * up in fp32 for the products' errors: |silu'| <= 1.1; five roundings and expf's two ulp."""
    slack = _sum_slack(x64, w64) + _aligned_loss(x64, w64)
    gate, up = y.chunk(2, dim=1)
    eg, eu = slack.chunk(2, dim=1)
    active = gate / (1.0 + torch.exp(-gate))
    exact = active * up
    return exact, 1.1 * eg * (up.abs() + eu) + (active.abs() + 1.1 * eg) * eu + exact.abs() * 16 * STEP32


@pytest.mark.parametrize("m,n,k", SWIGLU_SIZES)
def test_swiglu(device, m, n, k):
    x, xs = _eight(_normal(device, (m, k), seed=m + 3))
    w, ws = _eight(_normal(device, (n, k), seed=n + 4, std=2.0 / k**0.5))
    x64, w64 = _stands(x, xs), _stands(w, ws)
    exact, slack = _swiglu_slack(x64, w64, x64 @ w64.t())
    out, store = _guarded((m, n // 2), torch.float16, device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_SWIGLU)
    assert ((out.cpu().double() - exact).abs() <= slack + (exact.abs() + slack) * 2.0**-11 + 2.0**-25).all()
    _intact(store)


@pytest.mark.parametrize("m,n,k", [s for s in SWIGLU_SIZES if s[1] % 32 == 0] + [(1, 32, 16), (5, 288, 2048), (70, 1056, 640)])
def test_swiglu_to_eight_bits(device, m, n, k):
    x, xs = _eight(_normal(device, (m, k), seed=m + 5))
    w, ws = _eight(_normal(device, (n, k), seed=n + 6, std=2.0 / k**0.5))
    x64, w64 = _stands(x, xs), _stands(w, ws)
    exact, slack = _swiglu_slack(x64, w64, x64 @ w64.t())
    out, store = _guarded((m, n // 2), torch.float8_e4m3fn, device)
    scales, scale_store = _guarded((m, _hip.fp8_scale_stride(n // 2)), torch.float8_e8m0fnu, device)
    _hip.gemm_fp8(out, x, xs, w, ws, out_scales=scales, epilogue=_hip.GEMM_SWIGLU_FP8)
    _check_rounded(out, scales, exact, slack)
    _intact(store)
    _intact(scale_store)
    past = scales.cpu().view(torch.uint8)[:, ref.blocks(n // 2) :]
    assert (past == 0x5A).all()


@pytest.mark.parametrize("m", [5, 200])
def test_swiglu_to_eight_bits_past_fp32(device, m):
    """Activations past fp32's range become NaN and leave the scale to the block's others: the even columns, whose
    weights are zero where x is huge."""
    x, xs = _eight(_normal(device, (m, 256), seed=21))
    xs.view(torch.uint8)[1::2, 0] = 127 + 80  # 2^80: gate and up far past 2^64, or the gate below -2^64 and the output 0
    weight = _normal(device, (320, 256), seed=22, std=0.125)
    weight[::2, :128] = 0.0
    w, ws = _eight(weight)
    x64, w64 = _stands(x, xs), _stands(w, ws)
    exact, slack = _swiglu_slack(x64, w64, x64 @ w64.t())
    lost = torch.zeros((m, 160), dtype=torch.bool)
    lost[1::2, 1::2] = (x64 @ w64.t())[1::2, 1:160:2] > 0.0
    empty = torch.zeros_like(lost)
    empty[1::2, 1::2] = True
    assert (exact[lost].abs() > 2.0**130).all() and lost.any()
    out, scales = _hip.empty_fp8(m, 160, device)
    _hip.gemm_fp8(out, x, xs, w, ws, out_scales=scales, epilogue=_hip.GEMM_SWIGLU_FP8)
    got = out.cpu().double()
    assert torch.equal(got.isnan(), lost)
    zero = torch.zeros((), dtype=torch.float64)
    _check_rounded(got.nan_to_num(nan=0.0), scales, torch.where(empty, zero, exact), torch.where(empty, zero, slack))


@pytest.mark.parametrize("m,n,k", [(1, 64, 2048), (5, 36, 112), (16, 128, 1328), (31, 64, 5632), (64, 96, 400), (65, 32, 144), (128, 72, 272)])
def test_fp16_rows_are_rounded_as_quantize_does(device, m, n, k):
    x = _normal(device, (m, k), seed=m + 7)
    x *= torch.exp2(torch.randint(-8, 8, (m, 1), device=device, generator=_gen(device, 8)).half())
    x[0, 1] = 0.0
    if m > 2:
        x[2, :] = 0.0
    eight, xs = _eight(x)
    w, ws = _eight(_normal(device, (n, k), seed=n + 9, std=0.02))
    splits = min(3, ref.blocks(k))
    for epilogue, shape, dtype in ((_hip.GEMM_PARTIALS, (splits, m, n), torch.float32), (_hip.GEMM_HALF, (m, n), torch.float16),
                                   (_hip.GEMM_SWIGLU, (m, n // 2), torch.float16)):
        if epilogue == _hip.GEMM_SWIGLU and n % 8:
            continue
        a, b = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
        count = splits if epilogue == _hip.GEMM_PARTIALS else 1
        _hip.gemm_fp8(a, x, None, w, ws, splits=count, epilogue=epilogue)
        _hip.gemm_fp8(b, eight, xs, w, ws, splits=count, epilogue=epilogue)
        _same_bits(a, b)


@pytest.mark.parametrize("m,splits", [(3, 1), (20, 2), (70, 3)])
def test_nonfinite_fp16_rows_are_rounded_as_quantize_does(device, m, splits):
    """Infinities and NaN in fp16 x, beside values that set the scale and beside none: the rows become NaN, others keep
    their bits, whatever forms the products take."""
    x = _normal(device, (m, 400), seed=70)
    x[0, 5], x[1, 399] = float("inf"), float("nan")
    x[1, 130:140] = -float("inf")
    x[2, 128:256] = float("inf")
    eight, xs = _eight(x)
    w, ws = _eight(_normal(device, (72, 400), seed=71))
    for epilogue, shape, dtype, count in ((_hip.GEMM_PARTIALS, (splits, m, 72), torch.float32, splits), (_hip.GEMM_HALF, (m, 72), torch.float16, 1)):
        a, b = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        _hip.gemm_fp8(a, x, None, w, ws, splits=count, epilogue=epilogue)
        _hip.gemm_fp8(b, eight, xs, w, ws, splits=count, epilogue=epilogue)
        assert torch.equal(a.isnan(), b.isnan())
        bad = a.isnan().any(0) if a.ndim == 3 else a.isnan()
        assert bad[:3].all() and not bad[3:].any()


@pytest.mark.parametrize("m", [4, 140])
def test_nan_stays_in_its_row_and_column(device, m):
    x = _normal(device, (m, 272), seed=11)
    x[1, 260] = float("nan")
    x[2, 3] = float("inf")
    w = _normal(device, (64, 272), seed=12)
    w[5, 271] = float("nan")
    (xe, xs), (we, ws) = _eight(x), _eight(w)
    out = torch.empty((m, 64), dtype=torch.float16, device=device)
    _hip.gemm_fp8(out, xe, xs, we, ws, epilogue=_hip.GEMM_HALF)
    bad = torch.zeros((m, 64), dtype=torch.bool)
    bad[1:3], bad[:, 5] = True, True
    assert torch.equal(out.isnan().cpu(), bad)


@pytest.mark.parametrize("m", [3, 150])
def test_far_scales(device, m):
    """Scales at both ends: one block's power times another's stays in range where the result does."""
    x, xs = _whole_rows(device, m, 256, seed=20)
    w, ws = _whole_rows(device, 32, 256, seed=21)
    xs.view(torch.uint8)[:, 0], ws.view(torch.uint8)[:, 0] = 220, 30
    xs.view(torch.uint8)[:, 1], ws.view(torch.uint8)[:, 1] = 10, 244
    expected = (_stands(x, xs) @ _stands(w, ws).t()).half()
    out = torch.empty((m, 32), dtype=torch.float16, device=device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    assert torch.equal(out.cpu(), expected)


QKV_SIZES = [(1, 2048), (2, 144), (16, 512), (17, 2048), (50, 400), (64, 2048), (100, 256), (128, 1328), (129, 2048), (200, 400),
             (260, 272)]


@pytest.mark.parametrize("m,k,half_x", [(m, k, h) for m, k in QKV_SIZES for h in (False, True) if not h or m <= 128])
def test_qkv_is_the_half_product_rotated_and_written(device, m, k, half_x):
    x = _normal(device, (m, k), seed=m + 13)
    eight, xs = (x, None) if half_x else _eight(x)
    w, ws = _eight(_normal(device, (2560, k), seed=14, std=0.05))
    table = rope_table(device)
    gen = _gen(device, 15)
    positions = torch.randint(0, 2048, (m,), device=device, generator=gen)
    blocks = m // 16 + 3
    slots = torch.randperm(blocks * 16, device=device, generator=gen)[:m].contiguous()
    slots[m // 2] = -1
    pools = [torch.full((22, 2, blocks, 16, 4, 64), 3.0, dtype=torch.float16, device=device) for _ in range(2)]
    outs = [[torch.empty((m, h, 64), dtype=torch.float16, device=device) for h in (32, 4, 4)] for _ in range(2)]
    _hip.qkv_rope_append_fp8(outs[0][0], eight, xs, w, ws, positions, table, key_out=outs[0][1], value_out=outs[0][2], pool=pools[0],
                             layer=7, slot_mapping=slots)
    qkv = torch.empty((m, 2560), dtype=torch.float16, device=device)
    _hip.gemm_fp8(qkv, eight, xs, w, ws, epilogue=_hip.GEMM_HALF)
    _hip.rope_kv_append(outs[1][0], qkv, positions, table, key_out=outs[1][1], value_out=outs[1][2], pool=pools[1], layer=7, slot_mapping=slots)
    for a, b in zip(outs[0] + [pools[0]], outs[1] + [pools[1]]):
        _same_bits(a, b)
    only = torch.empty((m, 32, 64), dtype=torch.float16, device=device)
    _hip.qkv_rope_append_fp8(only, eight, xs, w, ws, positions, table)  # no pool, no copies
    _same_bits(only, outs[0][0])


# ---------------------------------------------------------------------------------------
# Large buffers, graphs, refusals of the binding
# ---------------------------------------------------------------------------------------


def test_rows_past_32_bit_offsets(device):
    """More than 2^31 elements, read and written: the last rows are those of a small call."""
    rows, width = 1_100_000, 2048
    x = torch.zeros((rows, width), dtype=torch.float16, device=device)
    x[-5:] = _normal(device, (5, width), seed=30)
    values, scales = _eight(x)
    few = _eight(x[-5:].clone())
    _same_bits(values[-5:], few[0])
    _same_bits(scales[-5:], few[1])
    weight = torch.ones(width, dtype=torch.float16, device=device)
    out = torch.empty_like(x)
    _hip.add_rms_norm_fp8(values, scales, out, x, x, weight)
    few_out = torch.empty_like(x[-5:])
    few = _hip.empty_fp8(5, width, device)
    _hip.add_rms_norm_fp8(*few, few_out, x[-5:].clone(), x[-5:].clone(), weight)
    _same_bits(values[-5:], few[0])
    _same_bits(scales[-5:], few[1])
    assert torch.equal(out[-5:], few_out)


def test_products_at_the_largest_operands(device):
    """n * k = 2^31 for one row, and 65536 rows: the ends hold what products of their own rows hold, exactly (whole numbers)."""
    k = 2048
    w, ws = _whole_rows(device, 1 << 20, k, seed=31)
    x, xs = _whole_rows(device, 2, k, seed=32)
    out = torch.empty((2, 1 << 20), dtype=torch.float16, device=device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    for part in (slice(0, 40), slice(-40, None)):
        expected = _stands(x, xs) @ _stands(w[part], ws[part]).t()
        assert torch.equal(out[:, part].cpu(), expected.half())
    del w, ws
    x, xs = _whole_rows(device, 65536, k, seed=33)
    w, ws = _whole_rows(device, 132, k, seed=34)
    out = torch.empty((65536, 132), dtype=torch.float16, device=device)
    _hip.gemm_fp8(out, x, xs, w, ws, epilogue=_hip.GEMM_HALF)
    for part in (slice(0, 40), slice(-40, None)):
        assert torch.equal(out[part].cpu(), (_stands(x[part], xs[part]) @ _stands(w, ws).t()).half())


def test_captured_chain_replays_on_new_inputs(device):
    """norm, SwiGLU to 8 bits and down projection in one graph, inputs changed in place between replays with eager
    work and synchronizations: every replay equals the eager calls, bit for bit."""
    from pagedcore_amd.decoder import capture_graph

    m, width = 150, 272
    weight = torch.ones(2048, dtype=torch.float16, device=device)
    gate_up, down = _eight(_normal(device, (2 * width, 2048), 40, 0.05)), _eight(_normal(device, (2048, width), 41, 0.05))
    hidden, delta = torch.empty((m, 2048), dtype=torch.float16, device=device), torch.empty((3, m, 2048), device=device)

    def fill(turn):
        hidden.copy_(_normal(device, (m, 2048), 50 + turn))
        delta.normal_(generator=_gen(device, 60 + turn))

    def chain():
        x, xs = _hip.empty_fp8(m, 2048, device)
        total = torch.empty_like(hidden)
        _hip.add_rms_norm_fp8(x, xs, total, hidden, delta, weight)
        a, a_s = _hip.empty_fp8(m, width, device)
        _hip.gemm_fp8(a, x, xs, *gate_up, out_scales=a_s, epilogue=_hip.GEMM_SWIGLU_FP8)
        y = torch.empty((m, 2048), dtype=torch.float16, device=device)
        _hip.gemm_fp8(y, a, a_s, *down, epilogue=_hip.GEMM_HALF)
        return total, y

    fill(0)
    chain()
    graph, held = capture_graph(chain, device)
    for turn in range(1, 5):
        fill(turn)
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        for a, b in zip(got, chain()):
            _same_bits(a, b)


def test_the_binding_refuses(device):
    x = torch.zeros((4, 64), dtype=torch.float16, device=device)
    values, scales = _hip.empty_fp8(4, 64, device)
    for call, needle in [
        (lambda: _hip.quantize_fp8(values, scales, x.float()), "float16"),
        (lambda: _hip.quantize_fp8(values, scales, x.t()), "unit column stride|float8_e4m3fn"),
        (lambda: _hip.quantize_fp8(values[:3], scales[:3], x), "float8_e4m3fn"),
        (lambda: _hip.quantize_fp8(values, scales[:, :0], x), "scales"),
        (lambda: _hip.quantize_fp8(values, scales.cpu(), x), "scales"),
        (lambda: _hip.quantize_fp8(values, scales.view(torch.uint8), x), "scales"),
        (lambda: _hip.quantize_fp8(values, scales, x.cpu()), "not the current GPU"),
        (lambda: _hip.quantize_fp8(values, scales, x[:1].expand(4, 64)), "x_stride"),
        (lambda: _hip.add_rms_norm_fp8(values, scales, None, x, x, x[0].clone()), "hidden_out"),
        (lambda: _hip.add_rms_norm_fp8(values, scales, x, x, x[:3], x[0].clone()), "delta"),
        (lambda: _hip.add_rms_norm_fp8(values, scales, x, x, torch.zeros((2, 4, 32), device=device), x[0].clone()), "partial sums"),
        (lambda: _hip.add_rms_norm_fp8(values, scales, x, x, None, x[0, :32].clone()), "weight"),
        (lambda: _hip.gemm_fp8(x, values, None, values, scales, epilogue=_hip.GEMM_HALF), "without scales"),
        (lambda: _hip.gemm_fp8(x, values, scales, values, scales, epilogue=_hip.GEMM_HALF), "out must be"),
        (lambda: _hip.gemm_fp8(x, values, scales, values, scales, epilogue=9), "unknown"),
        (lambda: _hip.gemm_fp8(torch.empty((1, 4, 4), device=device), values, scales, values, scales, splits=2), "out must be"),
        (lambda: _hip.gemm_fp8(torch.empty((2, 4, 4), device=device), values, scales, values, scales, splits=2), "1 blocks"),
        (lambda: _hip.qkv_rope_append_fp8(x, values, scales, values, scales, x, x), "2560"),
    ]:
        with pytest.raises(_hip.HipExtensionError, match=needle):
            call()


def test_streams_at_once(device):
    """Calls of two streams, interleaved, give what they give alone: no entry point has a buffer of its own."""
    def chain(m, seed, outputs):
        hidden, weight = _normal(device, (m, 512), seed=seed), _normal(device, (512,), seed=seed + 1)
        w, ws = _eight(_normal(device, (384, 512), seed=seed + 2, std=0.05))
        down, ds = _eight(_normal(device, (512, 192), seed=seed + 3, std=0.05))

        def run():
            rows = _hip.empty_fp8(m, 512, device)
            _hip.add_rms_norm_fp8(*rows, None, hidden, None, weight)
            active = torch.empty((m, 192), dtype=torch.float16, device=device)
            _hip.gemm_fp8(active, *rows, w, ws, epilogue=_hip.GEMM_SWIGLU)
            parts = torch.empty((2, m, 512), device=device)
            _hip.gemm_fp8(parts, active, None, down, ds, splits=2)
            eight = _hip.empty_fp8(m, 192, device)
            _hip.quantize_fp8(*eight, active)
            half = torch.empty((m, 512), dtype=torch.float16, device=device)
            _hip.gemm_fp8(half, *eight, down, ds, epilogue=_hip.GEMM_HALF)
            outputs.append((active, parts, *eight, half))
        return run

    alone, together = ([], []), ([], [])
    sides = [(chain(37, 80, alone[0]), chain(37, 80, together[0])), (chain(100, 90, alone[1]), chain(100, 90, together[1]))]
    for first, _ in sides:
        first()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    for _ in range(10):
        for stream, (_, again) in zip(streams, sides):
            with torch.cuda.stream(stream):
                again()
    torch.cuda.synchronize()
    for expected, got in zip(alone, together):
        assert len(got) == 10
        for outputs in got:
            for a, b in zip(expected[0], outputs):
                if a.dtype == torch.float8_e8m0fnu:  # a row's bytes past its blocks are not written
                    a, b = a[:, :2], b[:, :2]
                _same_bits(a, b)
