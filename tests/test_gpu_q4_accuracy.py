"""What decode attention over the 4-bit pool loses in its sums, where the output's rounding to fp16 does not hide it.

The values cancel exactly: tokens come in pairs of the same key, whose values are the negatives of each other and lie on the
levels (s (n - 7.5) and s ((15 - n) - 7.5)). Both have one score, one weight p and one step s, so that every output is 0, and what
the kernel writes is its error alone."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from tests.support import flags_clear

pytestmark = pytest.mark.gpu


def _cancelling_rows(tokens, device, seed):
    """K and V rows float16 [tokens, 4, 64], tokens 2 i and 2 i + 1 a pair."""
    gen = torch.Generator(device=device).manual_seed(seed)
    pairs = tokens // 2
    key = torch.randn(pairs, 4, 64, dtype=torch.float16, device=device, generator=gen)
    step = torch.randint(64, 128, (pairs, 4, 1), device=device, generator=gen).double() * 2.0**-9
    level = torch.randint(0, 16, (pairs, 4, 64), device=device, generator=gen)
    level[..., 5], level[..., 38] = 0, 15  # a row has both ends, so it is quantised to these levels
    value = (step * (level - 7.5)).half()  # 7 bits of the step times 4 of 2 n - 15: exact
    return key.repeat_interleave(2, dim=0), torch.stack((value, -value), dim=1).view(tokens, 4, 64)


@pytest.mark.parametrize("batch,length", [(256, 2048), (512, 2048), (64, 512), (8, 2048)])
def test_sums_of_values_that_cancel(device, batch, length):
    """Root mean square of the outputs against that of the roundings. Of an accumulated sum that grows evenly to A over n products the
    roundings, r in each, are independent, uniform and at most 2^-24 of what is held then: their variance is at most r n (2^-24 A)^2 / 9.
    n: 32 tokens a product, a wave's share of the bin, and 16 joins; r: 4 (the instruction's own additions). The sums
    held: (16 + n) p s of the levels, 16 p s of the offset that is taken off, 7.5 p s of the minima. p s is held in 16 bits: 2^-17 of
    15 p s a pair, independent between pairs. The output is rounded to a multiple of fp16's smallest, 2^-24, at most."""
    blocks, layer = batch * length // 16, 3
    tables = np.random.default_rng(batch).permutation(blocks).astype(np.int32).reshape(batch, length // 16)
    pool = torch.empty((22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device)
    steps = []
    for b in range(batch):
        key, value = _cancelling_rows(length, device, 1000 * batch + b)
        slots = torch.from_numpy((tables[b].astype(np.int64)[:, None] * 16 + np.arange(16)).reshape(-1)).to(device)
        _hip.kv_append_q4(pool, layer, key[None], value[None], slots)
        if b < 8:
            steps.append((key, value.abs().amax(-1).double() / 7.5))
    query = torch.randn(batch, 32, 64, dtype=torch.float16, device=device, generator=torch.Generator(device=device).manual_seed(batch))
    out = torch.full_like(query, 3.0)
    lens = np.full(batch, length, dtype=np.int32)
    plan = _hip.decode_plan(lens, tables)
    workspace = torch.zeros(_hip.workspace_bytes(batch, tables.shape[1]), dtype=torch.uint8, device=device)
    _hip.planned_decode_attention_q4(out, query, pool, layer, torch.from_numpy(lens).to(device), torch.from_numpy(plan).to(device), tables.shape[1], workspace)
    torch.cuda.synchronize()
    _hip.check_attention_faults(workspace, "test")
    assert flags_clear(workspace) and torch.isfinite(out).all()
    longest = int(plan[:, 1].max())  # blocks of a bin, which one wave takes of a head, or two in halves
    n = longest * 16 / 32 / (1 if batch <= 8 and batch * tables.shape[1] <= 2048 else 2) + 16
    for b, (key, step) in enumerate(steps):
        scores = torch.einsum("hgd,thd->hgt", query[b].double().view(4, 8, 64), key.double()) / 8.0
        p = torch.softmax(scores, -1)
        ps = p * step.t()[:, None]
        total = ps.sum(-1)
        sums = total * ((16 + 7.5) ** 2 + 16**2 + 7.5**2) ** 0.5
        variance = 4 * n / 9 * (2.0**-24 * sums) ** 2 + (2.0**-17 * 15 * ps[..., ::2]).square().sum(-1) / 3 + (2.0**-25) ** 2 / 3
        got = out[b].double().view(4, 8, 64).square().mean().sqrt().item()
        bound = variance.mean().sqrt().item()
        print(f"{batch} x {length}, sequence {b}: {got:.3g}, bound {bound:.3g}, bins of up to {longest} blocks")
        assert got <= bound
