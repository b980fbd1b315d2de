"""CPU checks of the host side of the codebook operators: which device, stream and tensors a call hands to
the library, with a fake in the library's place, and what it does not hand over."""
import contextlib
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")


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


@pytest.mark.parametrize("scale, threshold", [(1e39, 0), (-1e39, 0), (3.5e38, 0), (3e38, HALF), (-3e38, HALF),
                                              (1e38, 65535), (float("inf"), 0), (float("nan"), 0),
                                              (float("inf"), 65536)])
def test_scales_that_are_infinite_in_fp32_are_refused(scale, threshold):
    """The factor scale * 65536 / (65536 - T) is used in fp32; infinite, it would turn zeros into NaN."""
    from hds_b200 import native

    lib = native.lib
    for call in (lambda: lib.hds_embedding_forward(4, 4, 8, F32, 256, I64, 256, 0, 0, scale, threshold, 0, 0, None, F32,
                                                   256, None),
                 lambda: lib.hds_embedding_backward(100_000, 4, 8, F32, 256, I64, 256, 0, 0, scale, threshold, 0, 0,
                                                    None, F32, 256, 0, 256, 1 << 30, None)):
        assert call() == 1
        assert "finite" in lib.hds_last_error().decode()


@pytest.mark.parametrize("scale, threshold", [(3.4e38, 0), (-3.4e38, 0), (1.7e38, HALF), (1e39, 65536), (0.0, 0)])
def test_scales_that_fit_fp32_are_taken(scale, threshold):
    """The largest factors that fit (with nothing to look up), and any finite scale of nothing kept."""
    from hds_b200 import native

    lib = native.lib
    assert lib.hds_embedding_forward(0, 4, 8, F32, None, I64, None, 0, 0, scale, threshold, 0, 0, None, F32, None,
                                     None) == 0
    assert lib.hds_embedding_backward(0, 0, 8, F32, None, I64, None, 0, 0, scale, threshold, 0, 0, None, F32, None, 0,
                                      None, 0, None) == 0


class CpuKernels:
    """The extension module's two operators and the gradient on CPU tensors, written through the
    tensors' addresses as the kernels do: torch does not see what they compute.  Dropout keeps all."""

    def __init__(self, monkeypatch):
        from hds_b200 import gaussian_rasterizer as ext

        monkeypatch.setattr(ext, "_check", lambda t, name: None)
        monkeypatch.setattr(ext, "on_device", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(ext, "stream_of", lambda device: 0)
        monkeypatch.setattr(ext, "lib", self)
        self.calls = []

    @staticmethod
    def at(address, count, kind=ctypes.c_float):
        return np.ctypeslib.as_array((kind * count).from_address(address))

    def hds_embedding_forward(self, n, vocab, c, table_type, table, ids_type, ids, has_padding, padding_id, scale,
                              threshold, seed, offset, draw, out_type, out, stream):
        self.calls.append(("forward", draw and list(self.at(draw, 2, ctypes.c_int64))))
        rows = self.at(table, vocab * c).reshape(vocab, c)[self.at(ids, n, ctypes.c_int64)]
        self.at(out, n * c)[:] = np.float32(scale) * rows.reshape(-1)
        return 0

    def hds_embedding_backward_scratch_bytes(self, n, vocab, c):
        return 0

    def hds_embedding_backward(self, n, vocab, c, grad_type, grad, ids_type, ids, has_padding, padding_id, scale,
                               threshold, seed, offset, draw, table_type, grad_table, accumulate, scratch,
                               scratch_bytes, stream):
        self.calls.append(("backward", draw and list(self.at(draw, 2, ctypes.c_int64))))
        out = self.at(grad_table, vocab * c).reshape(vocab, c)
        if not accumulate:
            out[:] = 0
        np.add.at(out, self.at(ids, n, ctypes.c_int64), np.float32(scale) * self.at(grad, n * c).reshape(n, c))
        return 0

    def hds_dropout(self, rows, c, type_, x, threshold, whole_rows, seed, offset, draw, y, stream):
        self.calls.append(("dropout", draw and list(self.at(draw, 2, ctypes.c_int64))))
        self.at(y, rows * c)[:] = self.at(x, rows * c)
        return 0


def small_lookup(**more):
    table = torch.arange(12.0).reshape(4, 3)
    return table, torch.tensor([2, 0, 2]), dict(scale=2.0, seed=1, offset=2, **more)


def test_forward_mode_is_refused_and_not_lost(monkeypatch):
    """A tangent has requires_grad == False.  The operators have no forward mode; a call that goes past the
    autograd node would return a constant."""
    import hds_b200
    from torch.autograd import forward_ad

    kernels = CpuKernels(monkeypatch)
    table, ids, how = small_lookup()
    assert torch.equal(hds_b200.embedding(table, ids, **how), 2 * table[ids])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        for call in (lambda: hds_b200.embedding(dual, ids, **how), lambda: hds_b200.dropout(dual, 0.5, seed=1)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call()
        # The backward passes are maps of their own; so is a tangent of what goes into them.
        leaf = table.clone().requires_grad_(True)
        grad = forward_ad.make_dual(torch.ones(3, 3), torch.ones(3, 3))
        out = hds_b200.embedding(leaf, ids, **how)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(out, leaf, grad)
        out = hds_b200.dropout(leaf, 0.5, seed=1)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones(4, 3), torch.ones(4, 3)))
        # Inside a level, tensors without a tangent go through as ever.
        assert torch.equal(hds_b200.embedding(table, ids, **how), 2 * table[ids])
    assert [c[0] for c in kernels.calls].count("backward") == 0


def test_traced_calls_run_the_kernels(monkeypatch):
    """torch.jit.trace records torch's operators; the kernels' writes are none, so the node is recorded."""
    import hds_b200

    CpuKernels(monkeypatch)
    table, ids, how = small_lookup()

    def lookup(t):
        return hds_b200.embedding(t, ids, **how)

    def drop(t):
        return hds_b200.dropout(t, 0.5, seed=1)

    for f, want in ((lookup, lambda t: 2 * t[ids]), (drop, lambda t: t)):
        traced = torch.jit.trace(f, (table,), check_trace=False)
        for t in (table, table + 1, -table):
            assert torch.equal(traced(t), want(t))


def test_the_backward_takes_the_draw_that_was_saved(monkeypatch):
    """Under hooks that save copies (save_on_cpu, say) the draw may move on before the backward, which then
    has to draw the forward's mask: from the saved copy, not from where the draw was."""
    import hds_b200

    kernels = CpuKernels(monkeypatch)
    table, ids, _ = small_lookup()
    table.requires_grad_(True)
    draw = torch.tensor([7, 1])
    with torch.autograd.graph.saved_tensors_hooks(torch.clone, lambda t: t):
        out = hds_b200.embedding(table, ids, dropout_p=0.5, draw=draw)
        out = hds_b200.dropout(out, 0.5, draw=draw)
    draw += 1
    out.sum().backward()
    assert kernels.calls == [("forward", [7, 1]), ("dropout", [7, 1]), ("dropout", [7, 1]), ("backward", [7, 1])]
    # A draw whose memory was replaced is read where it is now: the old memory may be another tensor's.
    out = hds_b200.embedding(table, ids, dropout_p=0.5, draw=draw)
    draw.data = torch.tensor([9, 9])
    out.sum().backward()
    assert kernels.calls[-1] == ("backward", [9, 9])
    # Without dropout the draw is not looked at: it may be anything and change.
    draw = torch.zeros(3)
    out = hds_b200.embedding(table, ids, draw=draw)
    draw += 1
    out.sum().backward()
    assert kernels.calls[-1] == ("backward", None)


@pytest.mark.parametrize("unpack, text", [
    (lambda t: t.to(torch.int16), "int32 or int64"),
    (lambda t: t[:-1], "in the forward"),
    (lambda t: t.repeat(2), "in the forward"),
    (lambda t: t.reshape(1, -1), "in the forward"),
    (lambda t: t.repeat_interleave(2)[::2], "contiguous"),
    (lambda t: t.to("meta"), "device"),
])
def test_the_backward_checks_the_ids_that_hooks_hand_it(monkeypatch, unpack, text):
    """A kernel would read beyond them, or through an address of another kind."""
    import hds_b200

    kernels = CpuKernels(monkeypatch)
    table, ids, how = small_lookup()
    table.requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = hds_b200.embedding(table, ids, **how)
    with pytest.raises(RuntimeError, match=text):
        out.sum().backward()
    assert [c[0] for c in kernels.calls] == ["forward"]


@pytest.mark.parametrize("unpack", [lambda t: t.int(), lambda t: t[:1], lambda t: t.to("meta"),
                                    lambda t: t.repeat_interleave(2)[::2]])
def test_the_backward_checks_the_draw_that_hooks_hand_it(monkeypatch, unpack):
    import hds_b200

    kernels = CpuKernels(monkeypatch)
    table, ids, _ = small_lookup()
    table.requires_grad_(True)
    draw = torch.tensor([7, 1])

    def changed(t):
        return unpack(t) if t.shape == (2,) else t

    for call in (lambda: hds_b200.embedding(table, ids, dropout_p=0.5, draw=draw),
                 lambda: hds_b200.dropout(table, 0.5, draw=draw)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, changed):
            out = call()
        with pytest.raises(RuntimeError, match="draw must be"):
            out.sum().backward()
    assert [c[0] for c in kernels.calls] == ["forward", "dropout"]


def test_a_mask_that_depends_on_nothing_given_warns(monkeypatch):
    """Without seed, offset or draw every call and layer would drop the same elements."""
    import warnings

    import hds_b200

    CpuKernels(monkeypatch)
    table, ids, _ = small_lookup()
    with pytest.warns(UserWarning, match="same at every call"):
        hds_b200.dropout(table, 0.5)
    with pytest.warns(UserWarning, match="same at every call") as seen:
        hds_b200.embedding(table, ids, dropout_p=0.5)
    assert seen[0].filename == __file__
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for how in (dict(seed=0), dict(offset=0), dict(seed=3, offset=4), dict(draw=torch.tensor([1, 2]))):
            hds_b200.dropout(table, 0.5, **how)
            hds_b200.embedding(table, ids, dropout_p=0.5, **how)
            leaf = table.clone().requires_grad_(True)
            hds_b200.dropout(hds_b200.embedding(leaf, ids, dropout_p=0.5, **how), 0.5, **how).sum().backward()
        for p in (0.0, 1.0):  # nothing is drawn, or nothing depends on it
            hds_b200.dropout(table, p)
            hds_b200.embedding(table, ids, dropout_p=p)
