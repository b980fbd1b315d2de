"""CPU checks of the codebook lookup and dropout: the plain implementation they are tested against, and
the refusals that happen before any device work."""
import numpy as np
import pytest

import codebook_plain as plain

torch = pytest.importorskip("torch")

F32, BF16, F16, I32, I64 = range(5)


def test_philox_known_answers():
    """The known-answer vectors published with the generator."""
    ones = 0xFFFFFFFF
    got = [int(w) for w in plain.philox4x32_10((0, 0, 0, 0), (0, 0))]
    assert got == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    got = [int(w) for w in plain.philox4x32_10((ones,) * 4, (ones,) * 2)]
    assert got == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("p", [0.0, 1 / 65536, 0.1, 0.5, 0.97, 1.0])
def test_mask_drops_the_share_it_scales_for(p):
    n = 400_000
    kept = plain.keep_mask(0, n, p, 1234, 7)
    share = 1 - plain.threshold(p) / 65536
    # Six standard deviations of a binomial share.
    assert abs(kept.mean() - share) <= 6 * np.sqrt(share * (1 - share) / n) + 1e-12
    if share:
        assert share * plain.keep_share_factor(p) == pytest.approx(1.0, abs=1e-15)


def test_mask_depends_on_seed_and_offset_and_not_on_the_window():
    a = plain.keep_mask(0, 4096, 0.5, 1, 0)
    assert np.array_equal(plain.keep_mask(1000, 77, 0.5, 1, 0), a[1000:1077])
    for seed, offset in ((2, 0), (1, 1), (1, 2**32), (1 + 2**32, 0)):
        b = plain.keep_mask(0, 4096, 0.5, seed, offset)
        assert 0.4 < (a == b).mean() < 0.6
    # Beyond 2^32 groups the counter's second word moves.
    assert not np.array_equal(plain.keep_mask(8 * 2**32, 4096, 0.5, 1, 0), a)


def forward(lib, n=4, vocab=4, channels=8, table_type=F32, table=256, ids_type=I64, ids=256, scale=1.0, drop=0,
            draw=None, out_type=F32, out=256):
    return lib.hds_embedding_forward(n, vocab, channels, table_type, table, ids_type, ids, 0, 0, scale, drop, 0, 0,
                                     draw, out_type, out, None)


def backward(lib, n=100_000, vocab=4, channels=8, grad_type=F32, grad=256, ids_type=I64, ids=256, scale=1.0, drop=0,
             table_type=F32, table=256, accumulate=0, scratch=256, scratch_bytes=1 << 30):
    return lib.hds_embedding_backward(n, vocab, channels, grad_type, grad, ids_type, ids, 0, 0, scale, drop, 0, 0,
                                      None, table_type, table, accumulate, scratch, scratch_bytes, None)


def drop(lib, rows=4, channels=8, type_=F32, x=256, threshold=100, draw=None, y=256):
    return lib.hds_dropout(rows, channels, type_, x, threshold, 0, 0, 0, draw, y, None)


INVALID, UNSUPPORTED, SCRATCH, TOO_LARGE = 1, 2, 4, 5


@pytest.mark.parametrize("call, kwargs, code, text", [
    (forward, dict(n=-1), INVALID, "negative"),
    (forward, dict(vocab=-1), INVALID, "negative"),
    (forward, dict(channels=-1), INVALID, "negative"),
    (forward, dict(n=2**31), TOO_LARGE, "too large"),
    (forward, dict(vocab=2**31), TOO_LARGE, "too large"),
    (forward, dict(channels=32769), TOO_LARGE, "too large"),
    (forward, dict(channels=2**32 + 8), TOO_LARGE, "too large"),
    (forward, dict(n=2**31 - 2**21, channels=32768, drop=1), TOO_LARGE, "dropout of"),
    (backward, dict(n=2**31 - 2**21, channels=32768, drop=1), TOO_LARGE, "dropout of"),
    (forward, dict(table_type=I32), UNSUPPORTED, "table's type"),
    (forward, dict(table_type=BF16, out_type=F16), UNSUPPORTED, "table's type"),
    (forward, dict(table_type=F32, out_type=BF16), UNSUPPORTED, "table's type"),
    (forward, dict(ids_type=F32), UNSUPPORTED, "int32 or int64"),
    (forward, dict(scale=float("nan")), INVALID, "finite"),
    (forward, dict(scale=float("inf")), INVALID, "finite"),
    (forward, dict(drop=-1), INVALID, "threshold"),
    (forward, dict(drop=65537), INVALID, "threshold"),
    (forward, dict(table=None), INVALID, "null"),
    (forward, dict(ids=None), INVALID, "null"),
    (forward, dict(out=None), INVALID, "null"),
    (forward, dict(table=257), INVALID, "misaligned"),
    (forward, dict(ids=260), INVALID, "misaligned"),
    (forward, dict(out=258), INVALID, "misaligned"),
    (forward, dict(draw=260), INVALID, "misaligned"),
    (backward, dict(n=-1), INVALID, "negative"),
    (backward, dict(n=2**31 - 1), TOO_LARGE, "too large"),
    (backward, dict(grad_type=F16, table_type=BF16), UNSUPPORTED, "table's type"),
    (backward, dict(grad_type=BF16, table_type=BF16, accumulate=1), UNSUPPORTED, "fp32"),
    (backward, dict(ids_type=BF16), UNSUPPORTED, "int32 or int64"),
    (backward, dict(grad=None), INVALID, "null"),
    (backward, dict(ids=None), INVALID, "null"),
    (backward, dict(table=None), INVALID, "null"),
    (backward, dict(grad=258), INVALID, "misaligned"),
    (backward, dict(scratch=None), SCRATCH, "scratch"),
    (backward, dict(scratch=128), SCRATCH, "scratch"),
    (backward, dict(scratch_bytes=64), SCRATCH, "scratch"),
    (drop, dict(rows=-1), INVALID, "negative"),
    (drop, dict(rows=2**40, channels=2**40), TOO_LARGE, "too large"),
    (drop, dict(type_=I64), UNSUPPORTED, "element type"),
    (drop, dict(threshold=65537), INVALID, "threshold"),
    (drop, dict(x=None), INVALID, "null"),
    (drop, dict(y=None), INVALID, "null"),
    (drop, dict(x=258), INVALID, "misaligned"),
    (drop, dict(draw=4), INVALID, "misaligned"),
])
def test_bad_calls_are_refused_on_the_host(call, kwargs, code, text):
    from hds_b200 import native

    assert call(native.lib, **kwargs) == code
    assert text in native.lib.hds_last_error().decode()


def test_empty_calls_do_nothing():
    from hds_b200 import native

    lib = native.lib
    assert forward(lib, n=0, table=None, ids=None, out=None) == 0
    assert forward(lib, channels=0, out=None) == 0
    assert backward(lib, vocab=0, table=None) == 0
    assert backward(lib, channels=0) == 0
    assert drop(lib, rows=0, x=None, y=None) == 0


def test_scratch_grows_with_the_rows():
    from hds_b200 import native

    size = native.lib.hds_embedding_backward_scratch_bytes
    assert size(1, 1, 1) == 0 < size(100_000, 1000, 32) < size(1_000_000, 1000, 512)
    # Sorted keys and rows in two buffers each.
    assert size(1_000_000, 1000, 32) >= 16 * 1_000_000


def test_python_refusals():
    import hds_b200

    table, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="table must be a CUDA tensor"):
        hds_b200.embedding(table, ids)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        hds_b200.dropout(table, 0.5)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match=r"in \[0, 1\]"):
            hds_b200.dropout(table, p)
    assert hds_b200.dropout(table, 0.0) is table  # nothing to drop
