"""Scratch that calls share: per stream outside of captures, per capture and stream inside (no GPU)."""
import types

import pytest
import torch


@pytest.fixture()
def now(tq, monkeypatch):
    state = types.SimpleNamespace(stream=5, capture=0)
    monkeypatch.setattr(tq._lib, "_workspaces", {})
    monkeypatch.setattr(tq._lib, "_captured", {}, raising=False)
    monkeypatch.setattr(tq._lib, "stream_handle", lambda device=None: state.stream)
    monkeypatch.setattr(tq._lib, "capture_id", lambda stream: state.capture, raising=False)
    return state


def test_workspaces_of_captures(tq, now):
    """Two graphs captured on one stream may be replayed at the same time, and the zero fill of a capture happens only in
    its graph's replays: neither another graph nor an eager call on the stream uses that scratch."""
    dev = torch.device("cpu")
    get = lambda tag="flash8", n=100: tq._lib.workspace(n, dev, tag=tag)
    eager = get()
    assert eager is get() and eager.numel() >= 100 and not eager.any()
    now.capture = 7
    first = get()
    assert first is not eager and first is get() and not first.any()
    assert get("prefill") is not first
    assert get(n=3 << 20).numel() >= 3 << 20                # grows inside the capture
    now.capture = 8
    second = get()
    assert second is not first and second.data_ptr() != first.data_ptr()
    now.stream = 6                                          # another branch of the same capture
    assert get() is not second
    now.stream, now.capture = 5, 0
    assert get() is eager
    now.stream = 9
    assert get() is not eager


def test_first_use_of_a_stream_in_a_capture(tq, now):
    now.capture = 3
    inside = tq._lib.workspace(16, torch.device("cpu"), tag="prefill")
    now.capture = 0
    assert tq._lib.workspace(16, torch.device("cpu"), tag="prefill") is not inside
