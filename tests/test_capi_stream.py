"""The current stream that the tensor helpers launch on, with and without torch's inner functions for it."""
import pytest


@pytest.fixture
def capi():
    from peregrine_b200 import capi
    capi._torch_current.cache_clear()
    yield capi
    capi._torch_current.cache_clear()


@pytest.mark.parametrize("missing", ["_cuda_getDevice", "_cuda_getCurrentRawStream"])
def test_without_torchs_inner_functions(capi, monkeypatch, missing):
    import torch
    monkeypatch.delattr(torch._C, missing, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)

    class Stream:
        cuda_stream = 1234

    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: Stream if d == 3 else None)
    assert capi._stream(None) == 1234
    assert capi._stream(Stream) == 1234 and capi._stream(77) == 77


@pytest.mark.gpu
def test_current_stream(cuda, capi, monkeypatch):
    import torch
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            assert capi._stream(None) == stream.cuda_stream
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")
    capi._torch_current.cache_clear()
    with torch.cuda.stream(side):
        assert capi._stream(None) == side.cuda_stream
