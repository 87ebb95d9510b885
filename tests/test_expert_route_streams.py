"""A route used on another stream than the one that prepared it, with the library
and the streams replaced by recorders (no GPU): its memory, which the caller holds
no tensor of, waits for the calls queued there."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from flagsparse_amd.expert import PreparedExpertRoute


@pytest.fixture
def stream(monkeypatch):
    """The handle of the current stream, to be set; and what was called and recorded."""
    events, handle = [], [11]

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0 if name.endswith("bytes") else events.append((name, args[-1])) or 0

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: events.append(("kept", t.data_ptr(), s)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: f"stream {handle[0]}")
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "stream_handle", lambda device: handle[0])
    return handle, events


def test_calls_on_another_stream_keep_the_places(stream):
    handle, events = stream
    route = fs.prepare_expert_route(torch.zeros((4, 1), dtype=torch.int32), 2)
    assert isinstance(route, PreparedExpertRoute) and events == [("fs_expert_route", 11)]
    x, w, m = torch.ones(4, 8), torch.ones(4, 1), torch.ones(2, 8, 8)
    calls = {
        "fs_expert_dispatch": lambda: fs.flagsparse_expert_dispatch(x, route),
        "fs_expert_combine": lambda: fs.flagsparse_expert_combine(x, route, w),
        "fs_expert_combine_grad": lambda: fs.flagsparse_expert_combine_grad(x, x, route, w),
        "fs_expert_product": lambda: fs.flagsparse_expert_product(x, m, route),
        "fs_expert_product_grad_matrices": lambda: fs.flagsparse_expert_product_grad(x, x, m, route),
    }
    for name, call in calls.items():
        for handle[0] in (11, 12, 11, 13):
            events.clear()
            call()
            assert events[-1] == (name, handle[0])
            kept = [e for e in events if e[0] == "kept"]
            if handle[0] == 11:
                assert kept == []
            else:
                assert events[0] == ("kept", route.order.data_ptr(), f"stream {handle[0]}")
