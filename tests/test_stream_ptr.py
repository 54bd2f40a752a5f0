"""CPU: which stream a call launches on: the current one, also on a torch without the direct query for its
handle, or the given one."""
from __future__ import annotations

from importlib import import_module
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def stream_ptr(pkg, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=77))
    return import_module(pkg.__name__ + "._lib").stream_ptr


def test_the_current_stream_of_the_current_device(stream_ptr, monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    assert stream_ptr() == 103


def test_without_the_direct_query(stream_ptr, monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    assert stream_ptr() == 77


def test_a_given_stream(stream_ptr):
    assert stream_ptr(SimpleNamespace(cuda_stream=5)) == 5
