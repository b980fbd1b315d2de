"""The codebook lookup, its gradient and dropout on the GPU against the plain 64-bit implementation
(codebook_plain.py).

Values: the kernel multiplies the fp32 value by the fp32 factor and rounds once to the output type, so
they are compared bit for bit with that arithmetic on the CPU.  Gradients: fp32 sums within the bound
that table_gradient derives, plus half a step of the output type.  Masks: exactly."""
import numpy as np
import pytest

import codebook_plain as plain

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(autouse=True)
def _status_is_clear():
    from hds_b200 import native

    native.device_status(torch.device("cuda"))
    yield
    assert native.device_status(torch.device("cuda")) == 0


def make_ids(rng, n, vocab, spread=1, padding=None, dtype=torch.int64):
    """spread 1: uniform; larger: some ids much more popular; 0: one id only."""
    ids = np.minimum((rng.random(n) ** spread * vocab).astype(np.int64), vocab - 1) if spread else np.full(n, vocab // 2)
    if padding is not None:
        ids[rng.random(n) < 0.2] = padding
    return torch.from_numpy(ids).to(dtype).cuda()


def make_values(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype).cuda()


def as64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def expected_values(table, ids, dtype, scale=1.0, padding_id=None, p=0.0, seed=0, offset=0):
    """The lookup in the kernel's own arithmetic: one fp32 product, one rounding to the output type."""
    factor = np.float32(scale * plain.keep_share_factor(p))
    t = table.detach().float().cpu().numpy()
    flat = ids.reshape(-1).cpu().numpy()
    kept = plain.kept_elements(flat, t.shape[0], t.shape[1], padding_id, p, seed, offset)
    rows = t[np.clip(flat, 0, t.shape[0] - 1)] * factor
    return torch.from_numpy(np.where(kept, rows, np.float32(0))).to(dtype).reshape(*ids.shape, t.shape[1])


def assert_gradient(got, grad, ids, vocab, scale=1.0, padding_id=None, p=0.0, seed=0, offset=0, before=None):
    want, bound = plain.table_gradient(as64(grad), ids.cpu().numpy(), vocab, scale, padding_id, p, seed, offset)
    if before is not None:  # the add rounds once more
        want = want + as64(before)
        bound = bound + plain.U * 1.01 * (np.abs(want) + bound)
    # The store's rounding; below the smallest normal number steps stay that number's.
    info = torch.finfo(got.dtype)
    bound = bound + np.maximum(np.abs(want) + bound, info.tiny) * info.eps / 2
    error = np.abs(as64(got) - want)
    worst = np.unravel_index((error - bound).argmax(), error.shape) if error.size else None
    assert (error <= bound).all(), f"off by {error[worst]:.3e} at {worst}, bound {bound[worst]:.3e}"


SHAPES = [  # n, vocab, channels, spread
    (1, 1, 1, 1), (1, 5, 32, 1), (2, 1, 3, 1), (31, 300, 8, 1), (33, 2, 33, 1), (257, 40, 31, 2), (300, 5000, 100, 1),
    (1000, 3, 64, 1), (1025, 255, 16, 4), (2048, 256, 40, 1), (4097, 257, 7, 2), (4096, 2048, 128, 1),
    (5000, 2047, 256, 3), (6000, 1, 264, 1), (3001, 70_000, 512, 1), (10_007, 65_535, 32, 1), (9000, 65_536, 24, 2),
    (20_011, 11, 5, 1), (12_345, 4_200_000, 2, 1), (40_000, 900, 72, 0), (900, 17, 1000, 1), (700, 50, 521, 1),
    (100_000, 6, 32, 1), (131_072, 4096, 8, 4), (1_000_003, 3000, 8, 2), (990_000, 1500, 5, 0), (9, 4, 32_768, 1),
    (11, 4, 20_001, 1), (6000, 3, 3000, 1), (4096, 32_768, 9, 1), (4097, 32_769, 16, 1),
]


@pytest.mark.parametrize("n, vocab, c, spread", SHAPES)
def test_lookup_and_gradient(n, vocab, c, spread):
    import hds_b200

    rng = np.random.default_rng(n + vocab + c)
    table = make_values(rng, (vocab, c), torch.float32).requires_grad_(True)
    ids = make_ids(rng, n, vocab, spread)
    out = hds_b200.embedding(table, ids, scale=1.5)
    assert torch.equal(out.detach().cpu(), expected_values(table, ids, torch.float32, 1.5))
    grad = make_values(rng, (n, c), torch.float32)
    got, = torch.autograd.grad(out, table, grad)
    assert got.dtype == torch.float32 and got.shape == table.shape
    assert_gradient(got, grad, ids, vocab, 1.5)


@pytest.mark.parametrize("n, vocab, c, spread", [s for s in SHAPES if s[0] * s[2] <= 4_000_000])
def test_lookup_and_gradient_with_dropout_and_padding(n, vocab, c, spread):
    import hds_b200

    rng = np.random.default_rng(n + vocab + c + 1)
    table = make_values(rng, (vocab, c), torch.float32).requires_grad_(True)
    ids = make_ids(rng, n, vocab, spread, padding=-1)
    how = dict(scale=0.7, padding_id=-1, seed=2**63 + 5, offset=2**40 + n)
    out = hds_b200.embedding(table, ids, dropout_p=0.3, **how)
    assert torch.equal(out.detach().cpu(), expected_values(table, ids, torch.float32, p=0.3, **how))
    grad = make_values(rng, (n, c), torch.float32)
    got, = torch.autograd.grad(out, table, grad)
    assert_gradient(got, grad, ids, vocab, p=0.3, **how)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("c", [32, 75, 520])
@pytest.mark.parametrize("table_type, out_type", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                                  ("f16", "f32")])
@pytest.mark.parametrize("p", [0.0, 0.4])
def test_types(table_type, out_type, c, ids_dtype, p):
    import hds_b200

    rng = np.random.default_rng(c)
    n, vocab = 3000, 700
    table = make_values(rng, (vocab, c), TYPES[table_type]).requires_grad_(True)
    ids = make_ids(rng, n, vocab, 2, padding=3, dtype=ids_dtype).reshape(3, -1)
    how = dict(scale=2.25, padding_id=3, p=p, seed=9, offset=4)
    out = hds_b200.embedding(table, ids, dtype=TYPES[out_type], scale=2.25, padding_id=3, dropout_p=p, seed=9, offset=4)
    assert out.shape == (3, n // 3, c) and out.dtype == TYPES[out_type]
    assert torch.equal(out.detach().cpu(), expected_values(table, ids, TYPES[out_type], **how))
    grad = make_values(rng, (*ids.shape, c), TYPES[out_type])
    got, = torch.autograd.grad(out, table, grad)
    assert got.dtype == TYPES[table_type]
    assert_gradient(got, grad, ids, vocab, **how)


@pytest.mark.parametrize("c", [16, 50])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_ids_outside_the_table_give_zeros_and_set_the_status(c, p):
    import hds_b200
    from hds_b200 import native

    rng = np.random.default_rng(c)
    table = make_values(rng, (10, c), torch.float32).requires_grad_(True)
    ids = torch.tensor([0, -1, 10, 9, 2**40, -2**63, 5, 2**31, -2**31], device="cuda")
    out = hds_b200.embedding(table, ids, dropout_p=p)
    assert native.device_status(torch.device("cuda")) == 1
    assert native.device_status(torch.device("cuda")) == 0  # read and cleared
    assert torch.equal(out.detach().cpu(), expected_values(table, ids, torch.float32, p=p))
    assert not out.detach()[[1, 2, 4, 5, 7, 8]].any()
    grad = make_values(rng, (9, c), torch.float32)
    grad[1] = float("nan")
    got, = torch.autograd.grad(out, table, grad)
    assert native.device_status(torch.device("cuda")) == 1
    assert_gradient(got, torch.nan_to_num(grad), ids, 10, p=p)
    # The padding id is no error, wherever it lies.
    hds_b200.embedding(table.detach(), torch.tensor([-7, 3], device="cuda"), padding_id=-7)
    assert native.device_status(torch.device("cuda")) == 0


def test_every_row_masked():
    import hds_b200

    table = torch.full((4, 24), float("nan"), device="cuda", requires_grad=True)
    ids = torch.full((100,), -1, device="cuda")
    out = hds_b200.embedding(table, ids, padding_id=-1)
    assert not out.detach().any()
    got, = torch.autograd.grad(out, table, torch.full_like(out, float("inf")))
    assert not got.any()


@pytest.mark.parametrize("n, c", [(100, 24), (6000, 24), (100, 13), (6000, 13)])
def test_everything_dropped(n, c):
    import hds_b200

    table = torch.full((40, c), float("nan"), device="cuda", requires_grad=True)
    out = hds_b200.embedding(table, torch.arange(n, device="cuda") % 40, dropout_p=1.0, seed=1)
    assert not out.detach().any()
    got, = torch.autograd.grad(out, table, torch.full_like(out, float("nan")))
    assert not got.any()


@pytest.mark.parametrize("c", [8, 13])
def test_nothing_to_look_up(c):
    import hds_b200

    table = torch.randn(5, c, device="cuda", requires_grad=True)
    ids = torch.empty(0, 3, dtype=torch.int64, device="cuda")
    out = hds_b200.embedding(table, ids)
    assert out.shape == (0, 3, c)
    got, = torch.autograd.grad(out, table, torch.empty_like(out))
    assert got.shape == table.shape and not got.any()
    empty = torch.empty(0, c, device="cuda", requires_grad=True)
    ids = torch.full((6,), -1, device="cuda")
    out = hds_b200.embedding(empty, ids, padding_id=-1)
    assert not out.detach().any()
    got, = torch.autograd.grad(out, empty, out.detach())
    assert got.shape == (0, c)


@pytest.mark.parametrize("c", [32, 40, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_unaligned_and_strided_inputs(c, dtype, p):
    import hds_b200
    from hds_b200 import gaussian_rasterizer as ext

    rng = np.random.default_rng(c)
    n, vocab = 777, 90
    table = make_values(rng, (vocab * c + 1,), dtype)[1:].view(vocab, c)  # one element past an aligned base
    ids = make_ids(rng, n + 1, vocab, dtype=torch.int32)[1:]
    grad = make_values(rng, (n * c + 3,), dtype)[3:].view(n, c)
    how = dict(scale=3.0, seed=1, offset=2)
    out = hds_b200.embedding(table, ids, dropout_p=p, **how)
    assert torch.equal(out.cpu(), expected_values(table, ids, dtype, p=p, **how))
    assert_gradient(ext.embedding_backward(grad, ids, vocab, dropout_p=p, **how), grad, ids, vocab, p=p, **how)
    # Strided: columns of a wider table, every second id, a transposed gradient, a broadcast one.
    wide = make_values(rng, (vocab, 2 * c), dtype).requires_grad_(True)
    every = make_ids(rng, 2 * n, vocab)[::2]
    out = hds_b200.embedding(wide[:, c:], every, dropout_p=p, **how)
    assert torch.equal(out.detach().cpu(), expected_values(wide[:, c:], every, dtype, p=p, **how))
    grad = make_values(rng, (c, n), dtype).T
    got, = torch.autograd.grad(out, wide, grad, retain_graph=True)
    assert not got[:, :c].any()
    assert_gradient(got[:, c:], grad, every, vocab, p=p, **how)
    one = make_values(rng, (c,), dtype)
    got, = torch.autograd.grad(out, wide, one.expand(n, c))
    assert_gradient(got[:, c:], one.expand(n, c), every, vocab, p=p, **how)


@pytest.mark.parametrize("c, vocab", [(32, 500), (45, 500), (256, 20_000), (8, 3)])
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("n, skip", [(2500, 0), (2500, 3), (7000, 0), (7000, 6)])
def test_adding_into_a_buffer(c, vocab, p, n, skip):
    """skip: where the table's gradient begins in a flat buffer of all parameters' gradients."""
    from hds_b200 import gaussian_rasterizer as ext

    rng = np.random.default_rng(vocab + c)
    ids = make_ids(rng, n, vocab, 3, padding=-1)
    grad = make_values(rng, (n, c), torch.float32)
    before = make_values(rng, (vocab, c), torch.float32)
    flat = torch.zeros(vocab * c + 2 * skip, device="cuda")
    buffer = flat[skip:skip + vocab * c].view(vocab, c)
    buffer.copy_(before)
    how = dict(scale=0.5, padding_id=-1, seed=3, offset=8)
    ext.embedding_backward_into(buffer, grad, ids, dropout_p=p, **how)
    assert_gradient(buffer, grad, ids, vocab, p=p, before=before, **how)
    absent = torch.ones(vocab, dtype=torch.bool, device="cuda")
    absent[ids[ids >= 0]] = False
    assert torch.equal(buffer[absent], before[absent])
    assert not flat[:skip].any() and not flat[skip + vocab * c:].any()


def test_several_backward_passes_of_one_graph_and_second_derivatives():
    import hds_b200

    rng = np.random.default_rng(10)
    table = make_values(rng, (50, 32), torch.float32).requires_grad_(True)
    ids = make_ids(rng, 400, 50)
    out = hds_b200.dropout(hds_b200.embedding(table, ids), 0.5, seed=3)
    grads = [make_values(rng, (400, 32), torch.float32) for _ in range(3)]
    got = [torch.autograd.grad(out, table, g, retain_graph=True)[0] for g in grads]
    kept = torch.from_numpy(plain.keep_mask(0, 400 * 32, 0.5, 3, 0).reshape(400, 32))
    for g, w in zip(got, grads):
        assert_gradient(g, torch.where(kept, 2 * w.cpu(), torch.zeros(())), ids, 50)
    # A second derivative of dropout is dropout again; that of the lookup's gradient is refused.
    x = make_values(rng, (64, 8), torch.float32).requires_grad_(True)
    y = hds_b200.dropout(x, 0.5, seed=4)
    w = make_values(rng, (64, 8), torch.float32).requires_grad_(True)
    first, = torch.autograd.grad(y, x, w, create_graph=True)
    second, = torch.autograd.grad(first.sum(), w)
    assert torch.equal(second.cpu(), expected_dropout(torch.ones(64, 8), 0.5, 4, 0, False))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(out, table, grads[0].clone().requires_grad_(True), create_graph=True)


def test_gradient_is_added_into_the_leaf():
    import hds_b200

    rng = np.random.default_rng(0)
    table = make_values(rng, (50, 32), torch.float32).requires_grad_(True)
    before = make_values(rng, (50, 32), torch.float32)
    table.grad = before.clone()
    buffer = table.grad
    ids = make_ids(rng, 400, 50)
    with hds_b200.accumulate_leaf_grads():
        out = hds_b200.embedding(table, ids)
    grad = make_values(rng, (400, 32), torch.float32)
    out.backward(grad)
    assert table.grad is buffer
    assert_gradient(buffer, grad, ids, 50, before=before)


def test_the_same_call_gives_the_same_bits():
    from hds_b200 import gaussian_rasterizer as ext

    rng = np.random.default_rng(1)
    for n, vocab, c, spread in ((50_000, 12, 64, 1), (50_000, 3000, 37, 6), (200_000, 1, 8, 1)):
        ids, grad = make_ids(rng, n, vocab, spread), make_values(rng, (n, c), torch.float32)
        first = ext.embedding_backward(grad, ids, vocab)
        for _ in range(3):
            assert torch.equal(ext.embedding_backward(grad, ids, vocab), first)


def test_gradient_is_the_adjoint_of_the_lookup():
    """The lookup is linear in the table: its differences out(t + d) - out(t) = out(d), and the gradient is
    the adjoint of that map, <out(d), g> = <d, grad(g)>, mask included."""
    import hds_b200

    rng = np.random.default_rng(2)
    n, vocab, c = 3000, 200, 48
    ids = make_ids(rng, n, vocab, 2, padding=-1)
    how = dict(scale=1.25, padding_id=-1, dropout_p=0.35, seed=11, offset=12)
    table = make_values(rng, (vocab, c), torch.float32).requires_grad_(True)
    d, g = make_values(rng, (vocab, c), torch.float32), make_values(rng, (n, c), torch.float32)
    base = hds_b200.embedding(table, ids, **how)
    grad, = torch.autograd.grad(base, table, g)
    moved = hds_b200.embedding((table.detach() + d), ids, **how)
    size = float((base.detach().abs().double() * g.abs().double()).sum())
    difference = float(((moved - base.detach()).double() * g.double()).sum())
    assert abs(difference - float((d.double() * grad.double()).sum())) <= 8 * plain.U * 4 * size
    assert abs(float((hds_b200.embedding(d, ids, **how).double() * g.double()).sum())
               - float((d.double() * grad.double()).sum())) <= 8 * plain.U * 4 * size


def test_offsets_beyond_32_bits():
    """n * C past 2^31 elements: sampled rows of the values, and the gradient of a few codewords."""
    import hds_b200

    n, vocab, c = 4_300_000, 1000, 520
    gen = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
    table = torch.randn(vocab, c, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_(True)
    out = hds_b200.embedding(table, ids, dropout_p=0.5, seed=5, offset=6)
    factor = np.float32(2.0)
    t = table.detach().float().cpu().numpy()
    for row in (0, 4_129_776, 4_129_777, 4_200_001, n - 1):  # 2^31 / 520 = 4129776.2
        kept = plain.keep_mask(row * c, c, 0.5, 5, 6)
        want = torch.from_numpy(np.where(kept, t[int(ids[row])] * factor, np.float32(0))).to(torch.bfloat16)
        assert torch.equal(out[row].detach().cpu(), want)
    # A gradient that is one in the kept elements of the last rows only: sums are small whole numbers.
    grad = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    tail = 5000
    grad[-tail:] = 1
    got, = torch.autograd.grad(out, table, grad)
    kept = plain.keep_mask((n - tail) * c, tail * c, 0.5, 5, 6).reshape(tail, c)
    want = np.zeros((vocab, c))
    np.add.at(want, ids[-tail:].long().cpu().numpy(), kept * 2.0)
    assert torch.equal(got.float().cpu(), torch.from_numpy(want).float())


# ---------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------
def expected_dropout(x, p, seed, offset, rows):
    c = x.shape[-1] if rows else 1
    kept = plain.keep_mask(0, x.numel() // c if c else 0, p, seed, offset)
    kept = torch.from_numpy(np.repeat(kept, c)).reshape(x.shape)
    y = (x.detach().float().cpu() * float(np.float32(plain.keep_share_factor(p)))).to(x.dtype)
    return torch.where(kept, y, torch.zeros((), dtype=x.dtype))


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (256, 32), (255, 33), (1000, 75), (17, 4096), (4097, 2),
                                   (5, 6, 9), (100_003, 1), (1, 70_001), (2, 3, 16), (5, 40_000), (7, 33_003)])
@pytest.mark.parametrize("rows", [False, True], ids=["elements", "rows"])
@pytest.mark.parametrize("p", [0.1, 0.75])
def test_dropout_and_its_gradient(shape, dtype, rows, p):
    import hds_b200

    rng = np.random.default_rng(len(shape) * 1000 + shape[0])
    x = make_values(rng, shape, dtype).requires_grad_(True)
    y = hds_b200.dropout(x, p, seed=77, offset=2**33 + 1, rows=rows)
    assert torch.equal(y.detach().cpu(), expected_dropout(x, p, 77, 2**33 + 1, rows))
    g = make_values(rng, shape, dtype)
    got, = torch.autograd.grad(y, x, g)
    assert torch.equal(got.cpu(), expected_dropout(g, p, 77, 2**33 + 1, rows))


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("c", [64, 37])
def test_dropout_ends(rows, c):
    import hds_b200

    x = torch.randn(501, c, device="cuda")
    assert hds_b200.dropout(x, 0.0, rows=rows) is x
    assert not hds_b200.dropout(x, 1.0, rows=rows).any()
    one = hds_b200.dropout(x, 1 / 65536, seed=3, rows=rows)
    assert torch.equal(one.cpu(), expected_dropout(x, 1 / 65536, 3, 0, rows))
    assert hds_b200.dropout(x[:0], 0.5, rows=rows).shape == (0, c)
    assert hds_b200.dropout(x[:, :0], 0.5, rows=rows).shape == (501, 0)


def test_dropped_elements_are_zero_whatever_they_held():
    import hds_b200

    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e38], device="cuda").repeat(64).reshape(16, 16)
    for rows in (False, True):
        got = hds_b200.dropout(x, 0.5, seed=4, rows=rows).cpu()
        kept = plain.keep_mask(0, 16 if rows else 256, 0.5, 4, 0)
        kept = torch.from_numpy(np.repeat(kept, 16 if rows else 1)).reshape(16, 16)
        assert torch.equal(got[~kept], torch.zeros(int((~kept).sum())))
        assert torch.equal(torch.nan_to_num(got[kept]), torch.nan_to_num(x.cpu()[kept] * 2))


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows", [False, True])
def test_dropout_of_unaligned_and_strided_tensors(dtype, rows):
    import hds_b200

    rng = np.random.default_rng(3)
    flat = make_values(rng, (40 * 24 + 5,), dtype)
    for x in (flat[1:1 + 960].view(40, 24), flat[3:3 + 945].view(35, 27), flat[:960].view(24, 40).T):
        got = hds_b200.dropout(x, 0.5, seed=8, rows=rows)
        assert torch.equal(got.cpu(), expected_dropout(x, 0.5, 8, 0, rows))


def test_dropout_beyond_32_bits():
    import hds_b200

    n = 2**31 + 2**20 + 5
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = hds_b200.dropout(x, 0.5, seed=1, offset=1)
    for first in (0, 2**31 - 50_000, n - 50_000):
        kept = plain.keep_mask(first, 50_000, 0.5, 1, 1)
        assert torch.equal(y[first:first + 50_000].float().cpu(), torch.from_numpy(kept * 2.0).float())


# ---------------------------------------------------------------------------------------------
# streams, graphs, the path
# ---------------------------------------------------------------------------------------------
def test_on_another_stream():
    import hds_b200

    rng = np.random.default_rng(4)
    table = make_values(rng, (300, 64), torch.float32).requires_grad_(True)
    ids, grad = make_ids(rng, 20_000, 300), make_values(rng, (20_000, 64), torch.float32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = hds_b200.dropout(hds_b200.embedding(table, ids), 0.5, seed=1)
        got, = torch.autograd.grad(out, table, grad)
    side.synchronize()
    g = torch.from_numpy(np.where(plain.keep_mask(0, grad.numel(), 0.5, 1, 0).reshape(grad.shape),
                                  2 * grad.cpu().numpy(), np.float32(0)))
    assert_gradient(got, g, ids, 300)


def test_captured_graphs_take_the_draw_of_each_replay():
    """Two graphs captured one after another (a lookup with dropout and its gradient each), replayed in
    turn with the draw advanced on the device: every replay equals the eager call with those numbers."""
    import hds_b200

    rng = np.random.default_rng(5)
    n, vocab, c = 5000, 400, 40
    table = make_values(rng, (vocab, c), torch.float32).requires_grad_(True)
    ids = [make_ids(rng, n, vocab, s) for s in (1, 5)]
    grad = make_values(rng, (n, c), torch.float32)
    draw = torch.tensor([21, 0], device="cuda")

    def step(i, draw=None, offset=0):
        out = hds_b200.embedding(table, ids[i], dropout_p=0.4, seed=21, offset=offset, draw=draw)
        out = hds_b200.dropout(out, 0.2, seed=21, offset=offset, draw=draw, rows=True)
        return out.detach(), torch.autograd.grad(out, table, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0, draw)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(i, draw)
        graphs.append((g, outs))
    for offset in (0, 1, 2**35):
        draw[1] = offset
        for g, _ in graphs:
            g.replay()
        for i, (_, outs) in enumerate(graphs):
            want = step(i, offset=offset)
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_large_gradient_captured_beside_eager_calls():
    """The sort's blocks of more shared memory than the default, in a capture; eager gradients of the same
    table before it and between the replays, and the kernels without autograd captured while an eager graph
    of the table is alive."""
    import hds_b200
    from hds_b200 import gaussian_rasterizer as ext

    rng = np.random.default_rng(9)
    n, vocab, c = 1_100_000, 1500, 8
    table = make_values(rng, (vocab, c), torch.float32).requires_grad_(True)
    ids, grad = make_ids(rng, n, vocab, 2), make_values(rng, (n, c), torch.float32)

    def step():
        return torch.autograd.grad(hds_b200.embedding(table, ids), table, grad)[0]

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want) and torch.equal(step(), want)
    eager = hds_b200.embedding(table, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ext.embedding_backward(grad, ids, vocab)
    graph.replay()
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(eager, table, grad)[0], want)


def test_a_draw_that_moved_between_the_directions_is_refused():
    import hds_b200

    draw = torch.tensor([1, 2], device="cuda")
    x = torch.randn(64, 8, device="cuda", requires_grad=True)
    y = hds_b200.dropout(x, 0.5, draw=draw)
    draw += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="draw must be"):
        hds_b200.dropout(x, 0.5, draw=torch.tensor([1, 2]))
    with pytest.raises(RuntimeError, match="draw must be"):
        hds_b200.dropout(x, 0.5, draw=torch.tensor([1, 2, 3], device="cuda"))


def test_refusals_on_the_device():
    import hds_b200
    from hds_b200 import gaussian_rasterizer as ext

    table, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="int32 or int64"):
        hds_b200.embedding(table, ids.float())
    with pytest.raises(RuntimeError, match="table's device"):
        hds_b200.embedding(table, ids.cpu())
    with pytest.raises(RuntimeError, match="must be float32, bfloat16 or float16"):
        hds_b200.embedding(table.double(), ids)
    with pytest.raises(RuntimeError, match="of that type or float32"):
        hds_b200.embedding(table, ids, dtype=torch.float16)
    with pytest.raises(RuntimeError, match=r"\[V, C\]"):
        hds_b200.embedding(table[0], ids)
    with pytest.raises(RuntimeError, match="finite"):
        hds_b200.embedding(table, ids, scale=float("inf"))
    with pytest.raises(RuntimeError, match="grad must be"):
        ext.embedding_backward(torch.zeros(4, 8, device="cuda"), ids, 4)
    with pytest.raises(RuntimeError, match="float32 CUDA tensor"):
        ext.embedding_backward_into(table.half(), torch.zeros(3, 8, device="cuda"), ids)
    with pytest.raises(RuntimeError, match="x must be float32"):
        hds_b200.dropout(ids, 0.5)


def test_codebook_features_through_the_rasterizer():
    """A codebook model rendered and differentiated: features looked up (with dropout), whole gaussians
    dropped by their opacity, the blend, and the gradients back to the codebook -- against the same
    render of the explicit [N, C] features, whose gradient is then summed by codeword in 64 bits."""
    import hds_b200
    from hds_b200 import scenes
    from hds_b200.projection import project_gaussians

    dev = torch.device("cuda")
    s = scenes.config0(0, channels=32).to(dev)
    cam = s.cameras[0]
    n = s.means.shape[0]
    rng = np.random.default_rng(6)
    vocab = 128
    ids = make_ids(rng, n, vocab, 2, padding=-1)
    codebook = make_values(rng, (vocab, 32), torch.float32).requires_grad_(True)
    how = dict(scale=0.5, padding_id=-1, seed=31, offset=2)
    opacities = s.opacities.reshape(n, 1)
    means2D, depths, radii, conics = project_gaussians(s.means, s.scales, s.quats, opacities, cam.world_to_camera,
                                                       cam.fx, cam.fy, cam.cx, cam.cy, cam.width, cam.height)
    colors = torch.rand(n, 3, device=dev)
    kept_opacities = hds_b200.dropout(opacities, 0.2, seed=31, offset=3, rows=True).clamp(max=0.999)

    def render(features):
        return hds_b200.rasterize(means2D, depths, radii, conics, colors, kept_opacities, cam.width, cam.height,
                                  features=features)

    features = hds_b200.embedding(codebook, ids, dropout_p=0.1, **how)
    image, feature_image = render(features)
    dense = features.detach().clone().requires_grad_(True)
    dense_image, dense_feature_image = render(dense)
    assert torch.equal(feature_image, dense_feature_image) and torch.equal(image, dense_image)
    target = torch.rand_like(feature_image)
    loss = (feature_image - target).square().sum()
    got, = torch.autograd.grad(loss, codebook)
    dense_grad, = torch.autograd.grad((dense_feature_image - target).square().sum(), dense)
    assert float(got.abs().max()) > 0
    # The blend adds its gradients with atomics: two backward passes differ by rounding, which the sums
    # carry over (1e-4 of the largest entry is the suite's bound for the blend's gradients).
    want, bound = plain.table_gradient(as64(dense_grad), ids.cpu().numpy(), vocab, p=0.1, **how)
    assert np.abs(as64(got) - want).max() <= bound.max() + 1e-4 * np.abs(want).max()


@pytest.mark.parametrize("c", [64, 50])
def test_feature_shards_rows(c):
    """The rows of a feature shard leave and arrive through the lookup and its gradient: bit for bit what
    indexing gives."""
    from hds_b200.band_split import FeatureShards, add_rows, gather_rows

    rng = np.random.default_rng(8)
    table = make_values(rng, (5000, c), torch.float32)
    ids = torch.from_numpy(np.sort(rng.choice(5000, 1700, replace=False))).cuda()
    assert torch.equal(gather_rows(table, ids), table[ids])
    target, rows = make_values(rng, (5000, c), torch.float32), make_values(rng, (1700, c), torch.float32)
    want = target.clone()
    want[ids] = want[ids] + rows
    add_rows(target, ids, rows)
    assert torch.equal(target, want)
    for owner in (None, torch.zeros(5000, dtype=torch.int64)):
        shards = FeatureShards(5000, c, 0, 1, "cuda", init=lambda *a: table, owner=owner)
        assert torch.equal(shards.dispatch(ids), table[ids])
        shards.combine(ids, rows)
        shards.combine(ids, rows)
        want = torch.zeros_like(table)
        want[ids] = rows + rows
        assert torch.equal(shards.rows.grad, want)
        assert shards.dispatch(ids[:0]).shape == (0, c)
