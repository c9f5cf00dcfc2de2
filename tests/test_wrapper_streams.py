"""CPU tests of the stream that the Python binding passes: torch's current stream
of the context's device (of the destination's for an upload), whichever device is
current; the caller's own where one is given.  The library is replaced by a
recorder, the tensors live on the CPU."""
import types

import pytest
import torch

import rlxq


def _u8(*s):
    return torch.zeros(s, dtype=torch.uint8)


X, XB = torch.zeros((2, 64)), torch.zeros((2, 64), dtype=torch.bfloat16)
IDS = torch.zeros((2, 1), dtype=torch.int32)

CALLS = {
    "reserve_workspace": lambda c, **k: c.reserve_workspace(64, **k),
    "workspace_bytes": lambda c, **k: c.workspace_bytes(**k),
    "workspace_retired_bytes": lambda c, **k: c.workspace_retired_bytes(**k),
    "peak_probe": lambda c, **k: c.peak_probe(0, 1, sink=X, **k),
    "release_stream": lambda c, **k: c.release_stream(**k),
    "dequant_matmul": lambda c, **k: c.dequant_matmul(X, _u8(8 * 40), rlxq.GGUF_Q4_1, 8, **k),
    "dequant_matmul_noalloc": lambda c, **k: c.dequant_matmul_noalloc(X, _u8(8 * 40), rlxq.GGUF_Q4_1, 8,
                                                                      y=torch.zeros((2, 8)), **k),
    "dequantize": lambda c, **k: c.dequantize(_u8(8 * 40), rlxq.GGUF_Q4_1, 8, 64, **k),
    "grouped_matmul": lambda c, **k: c.grouped_matmul(X, _u8(2 * 8 * 40), torch.zeros(2), rlxq.GGUF_Q4_1, 8, 2, **k),
    "moe_grouped": lambda c, **k: c.moe_grouped(X, _u8(2 * 8 * 40), IDS, None, rlxq.GGUF_Q4_1, rlxq.MOE_EXPAND, 8, 2, **k),
    "moe_layer": lambda c, **k: c.moe_layer(X, torch.zeros((2, 64)), _u8(2 * 64 * 40), _u8(2 * 64 * 20), rlxq.GGUF_Q4_1,
                                            rlxq.GGUF_Q4_1, 1, 32, 2, **k),
    "moe_route": lambda c, **k: c.moe_route(torch.zeros((2, 4)), 2, True, **k),
    "swiglu": lambda c, **k: c.swiglu(torch.zeros((2, 8)), 4, **k),
    "quantize_act_int8": lambda c, **k: c.quantize_act_int8(X, **k),
    "quantize_mxfp4": lambda c, **k: c.quantize_mxfp4(X, **k),
    "mxfp4_gemm": lambda c, **k: c.mxfp4_gemm(X, _u8(8 * 32), _u8(16), 8, **k),
    "w8a8_gemm": lambda c, **k: c.w8a8_gemm(X, torch.zeros((64, 8), dtype=torch.int8), torch.ones(8), 8, **k),
}


@pytest.fixture(params=["handle", "object", "first"])
def recorder(request, monkeypatch):
    """Calls of the library as {name: arguments}, on streams 1000 + device: torch
    gives the handle alone, or a Stream object (where it has no such function, or
    has not used the GPU yet: the handle alone would be an error then)."""
    got = {}

    class Lib:
        def __getattr__(self, name):
            if not name.startswith("rlxq_"):
                raise AttributeError(name)

            def call(*args):
                got[name] = args
                return b"" if name.endswith("_error") else 0

            return call

    monkeypatch.setattr(rlxq, "lib", Lib)
    monkeypatch.setattr(rlxq, "_on_device", lambda device, **t: None)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: request.param != "first")
    if request.param == "handle":
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 1000 + d, raising=False)
    else:
        monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=1000 + d))
    if request.param == "object":
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    return got


def _context(device):
    c = rlxq.Context.__new__(rlxq.Context)
    c.h, c.device = None, device
    return c


@pytest.mark.parametrize("name", CALLS)
def test_stream_of_the_contexts_device(recorder, name):
    c = _context(3)
    for kw, want in (({}, 1003), ({"stream": 77}, 77)):
        recorder.clear()
        CALLS[name](c, **kw)
        (args,) = [a for n, a in recorder.items() if n == "rlxq_" + name or n.startswith("rlxq_dequant_grouped")]
        assert args[1 if "workspace" in name or name == "release_stream" else -1] == want


def test_every_method_with_a_stream_is_here():
    import inspect

    have = {n for n, f in inspect.getmembers(rlxq.Context, inspect.isfunction) if "stream" in inspect.signature(f).parameters}
    assert have - {"bind_dequant_matmul"} == set(CALLS)


@pytest.mark.parametrize("kind", ["GgufFile", "MlxFile"])
def test_upload_stream_of_the_destinations_device(recorder, kind):
    cls = getattr(rlxq, kind)
    f = cls.__new__(cls)
    f.h = None
    dst = types.SimpleNamespace(numel=lambda: 4, element_size=lambda: 1, data_ptr=lambda: 64, get_device=lambda: 2)
    f.upload("t", dst)
    (args,) = [a for n, a in recorder.items() if n.endswith("_upload")]
    assert args[-1] == 1002
