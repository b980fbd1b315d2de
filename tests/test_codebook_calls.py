"""CPU checks of the host side of the codebook operators: which device, stream and tensors a call hands to
the library, with a fake in the library's place, and what it does not hand over."""
import contextlib

import pytest

torch = pytest.importorskip("torch")


class FakeLib:
    """Stands in for the library: records the calls and answers 0."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.startswith("__"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


class FakeDevices:
    """The current device, and a stream per device (handle 100 + index)."""

    def __init__(self, monkeypatch, current=0):
        from hds_b200 import native

        self.current, self.seen = current, []
        monkeypatch.setattr(native, "on_device", self.on_device)
        monkeypatch.setattr(native, "stream_of", lambda device: 100 + device.index)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)

    @contextlib.contextmanager
    def on_device(self, device):
        before, self.current = self.current, device.index
        yield
        self.current = before


@pytest.mark.parametrize("device, index", [(None, 0), ("cuda", 0), (torch.device("cuda"), 0), ("cuda:1", 1), (1, 1),
                                           (torch.device("cuda", 0), 0), (torch.device("cuda", 1), 1)])
def test_the_status_is_read_on_its_own_device(monkeypatch, device, index):
    """Each device has its own status word, which the library finds through the current device: reading
    that of another device makes it current, with a stream of that device."""
    from hds_b200 import native

    devices = FakeDevices(monkeypatch)

    class Lib:
        def hds_device_status(self, out, stream):
            devices.seen.append((devices.current, stream))
            out._obj.value = devices.current + 1  # each device's word, as it were
            return 0

    monkeypatch.setattr(native, "lib", Lib())
    assert native.device_status(device) == index + 1
    assert devices.seen == [(index, 100 + index)]
    assert devices.current == 0
