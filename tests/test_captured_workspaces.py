"""A workspace that a captured graph has stays when a larger call outgrows it: the graph
writes there with every replay (the extension's bookkeeping, without a GPU)."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from uma_qmoe_amd import native_backend
from uma_qmoe_amd.native_backend import HipExtension

SIZES = (2048, 1408, 5632, 60, 4)


@pytest.fixture
def ext(monkeypatch):
    """An extension whose streams are a number and whose captures a flag, with workspaces on the host."""
    state = {"stream": 1, "capturing": False}
    monkeypatch.setattr(native_backend, "_stream_handle", lambda _torch, _device: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    ext = HipExtension()
    return ext, state


def take(ext, tokens):
    """A weak reference to the workspace of a call of ``tokens`` tokens."""
    return weakref.ref(ext._workspace("cpu", tokens, *SIZES))


def alive(ref):
    gc.collect()
    return ref() is not None


def test_a_captured_workspace_outlives_a_larger_call(ext):
    ext, state = ext
    small = take(ext, 1)
    state["capturing"] = True
    assert take(ext, 1)() is small()
    state["capturing"] = False
    large = take(ext, 64)
    assert large() is not small() and alive(small) and alive(large)
    assert take(ext, 64)() is large() and take(ext, 1)() is large()


def test_a_workspace_of_eager_calls_is_given_up(ext):
    ext, state = ext
    small = take(ext, 1)
    assert alive(take(ext, 64)) and not alive(small)
    # also where another stream's is captured
    state["stream"] = 2
    take(ext, 1)
    state["capturing"] = True
    other = take(ext, 1)
    state["capturing"], state["stream"] = False, 1
    first = take(ext, 64)
    second = take(ext, 128)
    assert alive(other) and alive(second) and not alive(first)


def test_errors_of_captured_workspaces_are_seen(ext, monkeypatch):
    ext, state = ext
    take(ext, 1)
    state["capturing"] = True
    small = take(ext, 1)
    state["capturing"] = False
    large = take(ext, 64)
    seen = []
    monkeypatch.setattr(ext, "workspace_status", seen.append)
    ext.status()
    assert len(seen) == 2 and {id(w) for w in seen} == {id(small()), id(large())}
