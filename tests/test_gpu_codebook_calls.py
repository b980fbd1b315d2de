"""The codebook operators on the GPU, called in ways that are allowed and rare."""
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_the_status_may_be_the_first_call_of_a_program():
    code = ("import sys; sys.path.insert(0, 'high-dimensional-splatting_b200'); from hds_b200 import native; "
            "print(native.device_status({}), native.device_status())")
    for device in ("", "'cuda:0'", "0"):
        done = subprocess.run([sys.executable, "-c", code.format(device)], capture_output=True, text=True, timeout=240,
                              cwd=Path(__file__).resolve().parent.parent)
        assert done.returncode == 0 and done.stdout.split() == ["0", "0"], done.stderr


def test_on_a_device_that_is_not_the_current_one():
    """Values, gradient, dropout and the status word of the tensors' own device."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    import hds_b200
    from hds_b200 import native

    torch.cuda.set_device(0)
    gen = torch.Generator().manual_seed(1)
    table = torch.randn(40, 24, generator=gen)
    grad = torch.randn(6000, 24, generator=gen)
    for ids in (torch.arange(6000) % 40, torch.arange(6000) % 41):
        got = []
        for device in ("cuda:0", "cuda:1"):
            leaf = table.to(device).requires_grad_(True)
            out = hds_b200.dropout(hds_b200.embedding(leaf, ids.to(device), dropout_p=0.2, seed=1), 0.3, seed=2)
            got.append((out.detach().cpu(), torch.autograd.grad(out, leaf, grad.to(device))[0].cpu()))
            torch.cuda.synchronize(device)
            other = "cuda:0" if device == "cuda:1" else "cuda:1"
            assert native.device_status(other) == 0
            assert native.device_status(device) == int(ids.max() == 40)
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("n", [100, 6000])  # one launch, and the sorted form
@pytest.mark.parametrize("c", [24, 13])
@pytest.mark.parametrize("scale", [-2.0, 3e38])
def test_rows_of_absent_codewords_are_plain_zeros(n, c, scale):
    from hds_b200 import gaussian_rasterizer as ext

    ids = torch.arange(n, device="cuda") % 20
    got = ext.embedding_backward(torch.randn(n, c, device="cuda"), ids, 50, scale=scale)
    absent = got[20:].cpu()
    assert torch.equal(absent, torch.zeros(30, c)) and not torch.signbit(absent).any()
    assert got[:20].any()


def test_forward_mode_is_refused_and_traces_run_the_kernels():
    import hds_b200
    from torch.autograd import forward_ad

    table, ids = torch.randn(9, 16, device="cuda"), torch.arange(40, device="cuda") % 9
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        with pytest.raises(NotImplementedError, match="jvp"):
            hds_b200.embedding(dual, ids)
        with pytest.raises(NotImplementedError, match="jvp"):
            hds_b200.dropout(dual, 0.5, seed=1)
    traced = torch.jit.trace(lambda t: hds_b200.embedding(t, ids), (table,), check_trace=False)
    assert torch.equal(traced(table + 1), (table + 1)[ids])
    traced = torch.jit.trace(lambda t: hds_b200.dropout(t, 0.5, seed=1), (table,), check_trace=False)
    assert torch.equal(traced(table + 1), hds_b200.dropout(table + 1, 0.5, seed=1))


def test_saved_on_the_host_between_the_directions():
    """save_on_cpu moves the ids and the draw to the host and back; the draw advances in between."""
    import hds_b200

    table = torch.randn(30, 16, device="cuda", requires_grad=True)
    ids, draw = torch.arange(500, device="cuda") % 30, torch.tensor([3, 4], device="cuda")
    grad = torch.randn(500, 16, device="cuda")

    def step(**how):
        out = hds_b200.embedding(table, ids, dropout_p=0.3, **how)
        return hds_b200.dropout(out, 0.2, rows=True, **how)

    want, = torch.autograd.grad(step(seed=3, offset=4), table, grad)
    with torch.autograd.graph.save_on_cpu():
        out = step(draw=draw)
    draw += 1
    got, = torch.autograd.grad(out, table, grad)
    assert torch.equal(got, want)


@pytest.mark.parametrize("c, dtype", [(40_000, torch.float32), (40_000, torch.bfloat16), (48, torch.bfloat16),
                                      (48, torch.float16), (50, torch.int32)])
def test_rows_of_shards_wider_than_the_kernels_take_and_of_fewer_bits(c, dtype):
    """What the kernels do not take is indexed, and 16-bit gradients are promoted, as before them."""
    from hds_b200.band_split import add_rows, gather_rows

    table, target = torch.randn(30, c, device="cuda"), torch.randn(30, c, device="cuda")
    ids = torch.tensor([0, 3, 4, 17, 29], device="cuda")
    rows = (10 * torch.randn(5, c, device="cuda")).to(dtype)
    want = target.clone()
    want[ids] = want[ids] + rows
    add_rows(target, ids, rows)
    assert torch.equal(target, want)
    assert torch.equal(gather_rows(table, ids), table[ids])


@pytest.mark.parametrize("n", [100, 6000, 100_000])  # one launch; the sort in one digit and some tiles; in many
@pytest.mark.parametrize("c", [24, 13])
@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("padding_id, vocab", [(-1, 40), (7, 40), (2999, 3000)])  # outside and inside the table
def test_nothing_but_padding(n, c, p, padding_id, vocab):
    """No row to look up or to sum, at the sizes of every form: values and gradient are zeros whatever the
    table and the incoming gradient hold, and a buffer that is added to keeps its bits."""
    import hds_b200
    from hds_b200 import gaussian_rasterizer as ext
    from hds_b200 import native

    table = torch.full((vocab, c), float("nan"), device="cuda", requires_grad=True)
    ids = torch.full((n,), padding_id, device="cuda")
    how = dict(padding_id=padding_id, dropout_p=p, seed=1, offset=2)
    out = hds_b200.embedding(table, ids, **how)
    assert torch.equal(out.detach(), torch.zeros(n, c, device="cuda"))
    grad = torch.full_like(out, float("inf"))
    got, = torch.autograd.grad(out, table, grad)
    assert torch.equal(got, torch.zeros(vocab, c, device="cuda"))
    before = torch.randn(vocab, c, device="cuda")
    before[0, 0], before[-1, -1] = float("nan"), -0.0
    buffer = before.clone()
    ext.embedding_backward_into(buffer, grad.detach(), ids, **how)
    assert torch.equal(buffer.view(torch.int32), before.view(torch.int32))
    assert native.device_status() == 0


@pytest.mark.parametrize("n", [100, 6000, 100_000])
@pytest.mark.parametrize("c", [24, 13])
def test_one_row_among_padding(n, c):
    """All rows but the last are padding, at the sizes of every form."""
    from hds_b200 import gaussian_rasterizer as ext

    ids = torch.full((n,), -1, device="cuda")
    ids[-1] = 39
    grad = torch.full((n, c), float("nan"), device="cuda")
    grad[-1] = torch.randn(c, device="cuda")
    got = ext.embedding_backward(grad, ids, 40, padding_id=-1)
    want = torch.zeros(40, c, device="cuda")
    want[39] = grad[-1]
    assert torch.equal(got, want)
    table = torch.full((40, c), float("nan"), device="cuda")
    table[39] = torch.randn(c, device="cuda")
    values = torch.zeros(n, c, device="cuda")
    values[-1] = table[39]
    assert torch.equal(ext.embedding(table, ids, padding_id=-1), values)


@pytest.mark.parametrize("n, c", [(500, 24), (20_000, 24), (20_000, 13)])
def test_adding_into_the_leaf_on_a_side_stream_is_done_when_the_backward_returns(n, c):
    """The add is all that the backward leaves behind (autograd gets no gradient): the caller's stream has to
    wait for it all the same, and for what went before it on the side stream (here a pause)."""
    import hds_b200

    table = torch.randn(50, c, device="cuda", requires_grad=True)
    ids, grad = torch.arange(n, device="cuda") % 50, torch.randn(n, c, device="cuda")
    table.grad = torch.zeros_like(table)
    want, = torch.autograd.grad(hds_b200.embedding(table, ids), table, grad)
    side = torch.cuda.Stream()
    for k in range(1, 4):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), hds_b200.accumulate_leaf_grads():
            torch.cuda._sleep(20_000_000)
            out = hds_b200.embedding(table, ids)
            out.record_stream(torch.cuda.current_stream())
        out.backward(grad)
        seen = table.grad.clone()
        assert torch.allclose(seen, k * want, rtol=1e-5, atol=1e-5 * float(want.abs().max()))
