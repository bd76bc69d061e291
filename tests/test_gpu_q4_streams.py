"""Calls over the 4-bit pool on two streams at once, each with a workspace of its own: cut sequences on one XCD and spread over all, the
fused append, rows written and read beside them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from tests.support import flags_clear

pytestmark = pytest.mark.gpu

BATCHES = {"ragged": [1 + 331 * i % 2048 for i in range(64)], "few": [2048, 3, 1500], "long": [20000, 700], "full": [2048] * 64}


def _case(device, lengths, seed):
    rng = np.random.default_rng(seed)
    need = -(-np.asarray(lengths) // 16)
    tables = np.zeros((len(lengths), int(need.max())), dtype=np.int32)
    tables[np.arange(tables.shape[1]) < need[:, None]] = rng.permutation(int(need.sum()))
    gen = torch.Generator(device=device).manual_seed(seed)
    pool = torch.zeros((22, int(need.sum()), 4, ref.UNIT), dtype=torch.uint8, device=device)
    slots = torch.arange(16 * pool.shape[1], device=device)
    rows = [torch.randn(1, slots.shape[0], 4, 64, dtype=torch.float16, device=device, generator=gen) for _ in range(2)]
    for layer in range(4):
        _hip.kv_append_q4(pool, layer, *[x.roll(layer, dims=1) for x in rows], slots)
    lens = np.asarray(lengths, dtype=np.int32)
    return {
        "pool": pool, "layers": range(4), "width": tables.shape[1], "lens": torch.from_numpy(lens).to(device),
        "plan": torch.from_numpy(_hip.decode_plan(lens, tables)).to(device),
        "workspace": torch.zeros(_hip.workspace_bytes(len(lens), tables.shape[1]), dtype=torch.uint8, device=device),
        "query": torch.randn(len(lens), 32, 64, dtype=torch.float16, device=device, generator=gen),
        "new": [torch.randn(len(lens), 4, 64, dtype=torch.float16, device=device, generator=gen) for _ in range(2)],
    }


def _run(case, fused):
    out = [torch.zeros_like(case["query"]) for _ in case["layers"]]
    new = case["new"] if fused else (None, None)
    for layer in case["layers"]:
        _hip.planned_decode_attention_q4(
            out[layer], case["query"], case["pool"], layer, case["lens"], case["plan"], case["width"], case["workspace"],
            new_key=new[0], new_value=new[1],
        )
    return out


@pytest.mark.parametrize("first,second", [("ragged", "ragged"), ("ragged", "few"), ("long", "ragged"), ("full", "long"), ("few", "few")])
def test_two_streams(device, first, second):
    cases = [_case(device, BATCHES[name], seed) for seed, name in enumerate((first, second))]
    alone = []
    for case, fused in zip(cases, (False, True)):
        alone.append(_run(case, fused))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        torch.cuda.synchronize()
        outs = [[], []]
        for _ in range(3):
            for i, (case, fused) in enumerate(zip(cases, (False, True))):
                with torch.cuda.stream(streams[i]):
                    outs[i].append(_run(case, fused))
        torch.cuda.synchronize()
        for i in range(2):
            _hip.check_attention_faults(cases[i]["workspace"], f"stream {i}")
            assert flags_clear(cases[i]["workspace"])
            for run in outs[i]:
                for got, expected in zip(run, alone[i]):
                    assert torch.equal(got.view(torch.int16), expected.view(torch.int16))
