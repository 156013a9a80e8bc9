"""Tensors of a device that is not the current one, without a GPU."""

import pytest
import torch

from pir2_b200 import ops


def test_streams_of_the_current_device_alone(monkeypatch):
    streams = []
    monkeypatch.setattr(ops, "_current_device", lambda: 1)
    monkeypatch.setattr(ops, "_current_raw_stream", lambda index: streams.append(index) or 16 * index)
    assert ops._raw_stream(1) == 16 and ops._stream(torch.device("cuda", 1)) == 16
    for call in (lambda: ops._raw_stream(0), lambda: ops._stream(torch.device("cuda", 0)), lambda: ops._raw_stream(2)):
        with pytest.raises(ValueError, match="current device"):
            call()
    assert streams == [1, 1]
