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


F32, BF16, F16, I32, I64 = range(5)
HALF = 32768  # a dropout threshold of 0.5


@pytest.mark.parametrize("scale, threshold", [(1e39, 0), (-1e39, 0), (3.5e38, 0), (3e38, HALF), (-3e38, HALF), (1e38, 65535),
                                              (float("inf"), 0), (float("nan"), 0), (float("inf"), 65536)])
def test_scales_that_are_infinite_in_fp32_are_refused(scale, threshold):
    """The factor scale * 65536 / (65536 - T) is used in fp32; infinite, it would turn zeros into NaN."""
    from hds_b200 import native

    lib = native.lib
    for call in (lambda: lib.hds_embedding_forward(4, 4, 8, F32, 256, I64, 256, 0, 0, scale, threshold, 0, 0, None, F32,
                                                   256, None),
                 lambda: lib.hds_embedding_backward(100_000, 4, 8, F32, 256, I64, 256, 0, 0, scale, threshold, 0, 0, None,
                                                    F32, 256, 0, 256, 1 << 30, None)):
        assert call() == 1
        assert "finite" in lib.hds_last_error().decode()


@pytest.mark.parametrize("scale, threshold", [(3.4e38, 0), (-3.4e38, 0), (1.7e38, HALF), (1e39, 65536), (0.0, 0)])
def test_scales_that_fit_fp32_are_taken(scale, threshold):
    """The largest factors that fit (with nothing to look up), and any finite scale of nothing kept."""
    from hds_b200 import native

    lib = native.lib
    assert lib.hds_embedding_forward(0, 4, 8, F32, None, I64, None, 0, 0, scale, threshold, 0, 0, None, F32, None, None) == 0
    assert lib.hds_embedding_backward(0, 0, 8, F32, None, I64, None, 0, 0, scale, threshold, 0, 0, None, F32, None, 0, None,
                                      0, None) == 0
