"""Whose a stream's scratch is, with a stand-in for captures and for the device's memory."""
import pytest
import torch

from hidet_b200 import native, runtime

DEVICE = torch.device('cuda', 0)
SIZE = 1 << 20


class Workspaces(runtime._Workspaces):
    capture = 0

    def _capture(self, stream):
        return self.capture

    @staticmethod
    def _allocate(how, index, size):
        return how(size, dtype=torch.uint8)

    def during(self, capture, nbytes=SIZE):
        """The address that a call gets inside a capture, 0: outside."""
        self.capture = capture
        try:
            return self.get(DEVICE, nbytes)[0]
        finally:
            self.capture = 0


@pytest.fixture
def told(monkeypatch):
    """What the native host path was told last, by stream."""
    last = {}
    monkeypatch.setattr(native, 'set_scratch', lambda device, stream, address, nbytes: last.__setitem__(stream, address))
    monkeypatch.setattr(native, 'clear_scratch', last.clear)
    monkeypatch.setattr(runtime, 'current_stream_ptr', lambda device: 77)
    return last


def test_a_graphs_scratch_stays_its_own_after_it_was_put_aside(told):
    """As CudaGraph does on a stream that a plain capture had: what it finds there it puts back."""
    w = Workspaces()
    first = w.during(1)
    assert told[77] == 0
    around = w.swap(DEVICE, 77, None)
    assert around.data_ptr() == first and told[77] == 0
    w.during(0)
    mine = w.swap(DEVICE, 77, around)
    assert mine.data_ptr() != first
    assert told[77] == 0            # not what calls outside use, on neither path
    keep = [around, mine]           # no address is handed out twice while they live
    second, outside = w.during(2), w.during(0)
    assert len({first, second, outside, mine.data_ptr()}) == 4 and told[77] == outside
    assert w.during(0) == outside and len(keep) == 2


def test_scratch_made_outside_comes_back_as_such(told):
    w = Workspaces()
    outside = w.during(0)
    around = w.swap(DEVICE, 77, None)
    assert told[77] == 0
    assert w.swap(DEVICE, 77, around) is None
    assert w.during(0) == outside and told[77] == outside


def test_one_capture_uses_what_it_made(told):
    w = Workspaces()
    assert w.during(1) == w.during(1)
    large = w.during(1, 4 * SIZE)
    assert w.during(1) == large and w.during(1, 4 * SIZE) == large
