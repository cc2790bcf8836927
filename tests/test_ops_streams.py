"""Where the wrappers take the current stream and device from, on the CPU."""
from __future__ import annotations

import importlib.util
import types

import pytest
import torch


def second_copy():
    """littlellm_b200.ops as it loads under the torch of the moment, beside the
    loaded module."""
    from littlellm_b200 import build
    build.build()
    import littlellm_b200.ops as ops
    spec = importlib.util.spec_from_file_location("littlellm_b200._ops_copy", ops.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("missing", [("_cuda_getCurrentRawStream",), ("_cuda_getDevice",),
                                     ("_cuda_getCurrentRawStream", "_cuda_getDevice")])
def test_public_functions_serve_where_torch_lacks_the_raw_ones(monkeypatch, missing):
    for name in missing:
        monkeypatch.delattr(torch._C, name, raising=False)
    asked = []

    def current_stream(device=None):
        asked.append(device)
        return types.SimpleNamespace(cuda_stream=0x1234)

    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    ops = second_copy()
    got = []
    assert ops._stream(torch.device("cuda", 2)) == 0x1234
    ops._call(torch.device("cuda", 2), lambda *args: got.append(args) or 0, 7, 8)
    assert got == [(7, 8, 0x1234)] and asked == [2, 2]
