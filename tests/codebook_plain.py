"""Plain 64-bit implementation of the codebook lookup, its gradient and dropout (numpy), written from
their definitions: the yardstick of test_codebook.py and test_gpu_codebook.py."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative


def philox4x32_10(counter, key):
    """counter: four uint64 arrays (or numbers) below 2^32; key: two numbers below 2^32.  The four words."""
    x = [np.asarray(c, np.uint64) for c in counter]
    k = [int(v) for v in key]
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> shift) ^ x[1] ^ np.uint64(k[0]), p1 & low, (p0 >> shift) ^ x[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return x


def threshold(p: float) -> int:
    return round(p * 65536)


def keep_share_factor(p: float) -> float:
    t = threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def keep_mask(first: int, count: int, p: float, seed: int, offset: int) -> np.ndarray:
    """Whether elements first .. first + count - 1 of the draw (seed, offset) are kept."""
    seed, offset = seed % 2**64, offset % 2**64
    e = np.arange(first, first + count, dtype=np.uint64)
    q = e // np.uint64(8)
    words = philox4x32_10((q & np.uint64(0xFFFFFFFF), q >> np.uint64(32),
                           np.full_like(q, offset % 2**32), np.full_like(q, offset // 2**32)),
                          (seed % 2**32, seed // 2**32))
    half = (e % np.uint64(8)).astype(np.int64)
    word = np.stack(words)[half // 2, np.arange(count)]
    bits = np.where(half % 2 == 1, word >> np.uint64(16), word & np.uint64(0xFFFF))
    return bits >= np.uint64(threshold(p))


def lookup(table, ids, scale=1.0, padding_id=None, p=0.0, seed=0, offset=0):
    """(values [n, C] in 64 bits, kept [n, C]): table as float64, ids as int64 (flat)."""
    table, ids = np.asarray(table, np.float64), np.asarray(ids, np.int64).reshape(-1)
    kept = kept_elements(ids, table.shape[0], table.shape[1], padding_id, p, seed, offset)
    rows = table[np.clip(ids, 0, max(table.shape[0] - 1, 0))] if table.shape[0] else np.zeros((ids.size, table.shape[1]))
    return np.where(kept, rows * (scale * keep_share_factor(p)), 0.0), kept


def kept_elements(ids, vocab, channels, padding_id=None, p=0.0, seed=0, offset=0):
    ids = np.asarray(ids, np.int64).reshape(-1)
    there = (ids >= 0) & (ids < vocab)
    if padding_id is not None:
        there &= ids != padding_id
    kept = np.repeat(there[:, None], channels, 1)
    if threshold(p) > 0 and kept.size:
        kept &= keep_mask(0, kept.size, p, seed, offset).reshape(kept.shape)
    return kept


def table_gradient(grad, ids, vocab, scale=1.0, padding_id=None, p=0.0, seed=0, offset=0):
    """(dtable [V, C], bound [V, C]) in 64 bits.  bound: how far an fp32 sum in the library's order may be.

    A sum along which at most P additions follow one another is off by at most P u sum |g| (u = 2^-24).
    The library adds at most L rows one after another, L = 8 to 256, then the m / L + 2 parts of m rows: up
    to 65 of them one after another, more in 64 interleaved runs and a tree of 6 steps.  So
    P <= L + max(65, m / (64 L) + 8) <= 328 + m / 512, and never more than m.  The factor and the product
    round once each, adding 2 u; 1.01 covers the terms of order u^2."""
    grad, ids = np.asarray(grad, np.float64), np.asarray(ids, np.int64).reshape(-1)
    c = grad.shape[-1]
    grad = grad.reshape(-1, c)
    kept = kept_elements(ids, vocab, c, padding_id, p, seed, offset)
    g = np.where(kept, grad, 0.0)
    there = (ids >= 0) & (ids < vocab)
    if padding_id is not None:
        there &= ids != padding_id
    sums, size = np.zeros((vocab, c)), np.zeros((vocab, c))
    rows = np.bincount(ids[there], minlength=vocab)[:vocab] if vocab else np.zeros(0)
    np.add.at(sums, ids[there], g[there])
    np.add.at(size, ids[there], np.abs(g[there]))
    f = scale * keep_share_factor(p)
    path = np.minimum(rows, 328 + rows / 512)[:, None] + 2
    return sums * f, 1.01 * path * U * size * abs(f)
