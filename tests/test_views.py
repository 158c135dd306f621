"""The Python binding's views of what a call is given."""
import sys

import pytest

import h3attn as H


def test_a_view_is_taken_as_it_is():
    """Without an exception raised and caught on the way, which costs four times the call."""
    v, raised = H.raw_view(0x1000, 64), []

    def trace(frame, event, arg):
        if event == "exception":
            raised.append(arg)
        return trace

    sys.settrace(trace)
    try:
        got = H.view(v)
    finally:
        sys.settrace(None)
    assert got is v and not raised


def test_what_is_no_tensor_is_refused():
    class Wider(H.View):
        pass

    wider = Wider(0x1000, 64)
    assert H.view(wider) is wider
    assert H.view(None).bytes == 0
    with pytest.raises(TypeError, match="cannot bind"):
        H.view([1, 2])
