"""The status word is never created inside a CUDA-graph capture by the training entries."""

from __future__ import annotations

import pytest


def test_the_first_call_on_a_device_is_refused_inside_a_capture(b200, monkeypatch):
    import torch

    monkeypatch.setattr(b200, "_status_words", {})
    monkeypatch.setattr(b200, "_status_addresses", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        b200.status_address(3)
    assert not b200._status_words and not b200._status_addresses
    b200._status_words[3] = torch.zeros(1, dtype=torch.int32)  # made by an earlier call
    assert b200.status_address(3) == b200._status_words[3].data_ptr()


@pytest.mark.gpu
def test_a_refused_capture_leaves_the_device_usable(b200, monkeypatch):
    import importlib.util
    import sys

    import torch

    name = "avo_b200_training_binding"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, b200.HERE / "b200_training.py")
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    training = sys.modules[name]
    q = torch.randn(1, 2, 70, 128, device="cuda").bfloat16()
    want = training.grouped_attention(q, q, q, True)
    with monkeypatch.context() as patch:
        patch.setattr(b200, "_status_words", {})
        patch.setattr(b200, "_status_addresses", {})
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for call in (lambda: training.grouped_attention(q, q, q, True),
                         lambda: training.attention_backward(q, q, q, q, *want, True)):
                with pytest.raises(RuntimeError, match="first call on device 0 cannot be captured"):
                    call()
        del graph
    got = training.grouped_attention(q, q, q, True)
    torch.cuda.synchronize()
    b200.check_status(q.device)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
