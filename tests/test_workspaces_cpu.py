"""Which memory the token operators' workspaces hand out, without a GPU."""
import pytest
import torch

from sketchpad_b200 import _torch


@pytest.fixture
def host(monkeypatch):
    """Workspaces in host memory; state["capturing"] says whether the stream is being captured."""
    state = {"capturing": False}
    zeros = torch.zeros
    monkeypatch.setattr(_torch.torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    return state


def test_calls_of_a_stream_share_one_that_grows(host):
    w = _torch.Workspaces()
    a = w.get(0, 7, 100)
    assert a[2] >= 100 and not a[0].any()
    assert w.get(0, 7, 60)[1] == a[1]
    assert w.get(0, 8, 60)[1] != a[1] and w.get(1, 7, 60)[1] != a[1]
    b = w.get(0, 7, 1000)
    assert b[2] >= 1000 and w.get(0, 7, 100)[1] == b[1]


def test_a_capture_never_gets_the_streams_workspace(host):
    # warm up on a stream, capture on it, make a larger call on it: the stream's workspace is
    # replaced and its memory freed, so the graph must not have it
    w = _torch.Workspaces()
    kept = w.get(0, 7, 100)
    host["capturing"] = True
    inside = w.get(0, 7, 100)
    assert inside[1] != kept[1] and not inside[0].any()
    host["capturing"] = False
    assert w.get(0, 7, 100)[1] == kept[1]  # nor does the stream get the graph's
    larger = w.get(0, 7, 1000)
    assert larger[1] not in (kept[1], inside[1])


def test_a_given_workspace_is_contiguous():
    # its bytes are counted from its values, which must not lie further apart
    t = torch.zeros(64, 4, dtype=torch.int32)
    assert _torch.given_workspace(t)[1:] == (t.data_ptr(), 1024)
    for bad in (t[:, :2], t[::2], t.t()):
        with pytest.raises(ValueError):
            _torch.given_workspace(bad)


class OnDevice:
    def __init__(self, index):
        self.index = index

    def get_device(self):
        return self.index


def test_operators_run_on_the_current_device(monkeypatch):
    # a default stream's handle is the same on every device: the kernel would run on the current
    # one, with addresses of another
    monkeypatch.setattr(_torch, "_current_device", lambda: 1, raising=False)
    assert _torch.cuda_index(OnDevice(1), None, OnDevice(1)) == 1
    with pytest.raises(ValueError):
        _torch.cuda_index(OnDevice(0), OnDevice(0))
    with pytest.raises(ValueError):
        _torch.cuda_index(OnDevice(-1))
