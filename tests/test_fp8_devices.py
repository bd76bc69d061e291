"""The 8-bit calls on a GPU that is not the current one, without a GPU: the library and torch's device state are
stand-ins, the checks and the call are the binding's own."""

from __future__ import annotations

from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

from pagedcore_amd import _hip


class OnGpu:
    """A CPU tensor that says it lies on GPU `index`."""

    def __init__(self, tensor: torch.Tensor, index: int) -> None:
        self._tensor, self._index = tensor, index

    def get_device(self) -> int:
        return self._index

    def __getattr__(self, name):
        return getattr(self._tensor, name)


@pytest.fixture
def calls(monkeypatch):
    """(entry point, GPU that is current in it, stream it is given) of each call; GPU 0 is current."""
    made, current = [], [0]

    @contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    class Library:
        def __getattr__(self, name):
            return lambda *args: made.append((name, current[0], args[-1])) or 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_hip, "_raw_stream", lambda index: 7000 + index)
    library = Library()
    monkeypatch.setattr(_hip, "load", lambda: library)
    yield made
    assert current[0] == 0


def _operands(gpu):
    on = lambda *shape, dtype=torch.float16: OnGpu(torch.zeros(shape, dtype=dtype), gpu)  # noqa: E731
    eight = lambda rows, width: (on(rows, width, dtype=torch.uint8).view(torch.float8_e4m3fn),  # noqa: E731
                                 on(rows, _hip.fp8_scale_stride(width), dtype=torch.uint8).view(torch.float8_e8m0fnu))
    place = lambda pair: tuple(OnGpu(t, gpu) for t in pair)  # noqa: E731
    x, w = place(eight(2, 64)), place(eight(2560, 64))
    return SimpleNamespace(half=on(2, 64), x=x, w=w, out=on(2, 2560), weight=on(64), query=on(2, 32, 64), table=on(8, 2, 32),
                           positions=on(2, dtype=torch.int64), parts=on(3, 2, 64, dtype=torch.float32))


@pytest.mark.parametrize("gpu", [0, 1])
def test_calls_run_on_the_tensors_gpu(calls, gpu):
    """On its current stream, with it made current for the call, as the library's launches need."""
    t = _operands(gpu)
    _hip.quantize_fp8(*t.x, t.half)
    _hip.add_rms_norm_fp8(*t.x, t.half, t.half, t.half, t.weight)
    _hip.add_rms_norm_fp8(*t.x, t.half, t.half, t.parts, t.weight)
    _hip.gemm_fp8(t.out, *t.x, *t.w, epilogue=_hip.GEMM_HALF)
    _hip.qkv_rope_append_fp8(t.query, *t.x, *t.w, t.positions, t.table)
    assert calls == [(name, gpu, 7000 + gpu) for name in (
        "pc_quantize_fp8", "pc_add_rms_norm_fp8", "pc_add_rms_norm_parts_fp8", "pc_gemm_fp8", "pc_qkv_rope_append_fp8")]


def test_tensors_of_two_gpus_are_refused(calls):
    here, there = _operands(1), _operands(0)
    for call in (lambda: _hip.quantize_fp8(*there.x, here.half), lambda: _hip.add_rms_norm_fp8(*here.x, None, here.half, None, there.weight),
                 lambda: _hip.gemm_fp8(there.out, *here.x, *here.w, epilogue=_hip.GEMM_HALF),
                 lambda: _hip.gemm_fp8(here.out, *here.x, *there.w, epilogue=_hip.GEMM_HALF),
                 lambda: _hip.qkv_rope_append_fp8(here.query, *here.x, *here.w, there.positions, here.table)):
        with pytest.raises(_hip.HipExtensionError, match="on GPU 1"):
            call()
    assert not calls


def test_host_tensors_are_refused(calls):
    cpu = _operands(-1)
    with pytest.raises(_hip.HipExtensionError, match="not the current GPU"):
        _hip.quantize_fp8(*cpu.x, cpu.half)
    assert not calls
