"""Attention over the 8-bit cache at shapes that between them take every form of the
kernel of few rows: one to many tiles of 16 or 32 pairs, one range of keys or several, one,
two or four groups of waves; on the GPU against 64 bits. All KV heads hold the same rows."""
import numpy as np
import pytest

import esdecode as E
import kv8
from helpers import bf16, f32, rng

pytestmark = pytest.mark.gpu

DIM = 256
SHAPES = [(5, 5, 1, 0), (8, 1, 3, 0), (64, 1, 1, 0), (5, 5, 1, 839), (8, 1, 3, 781), (8, 1, 5, 815), (5, 5, 1, 64), (8, 1, 3, 67),
          (5, 5, 20, 1602), (8, 1, 6, 62), (8, 2, 9, 2590), (5, 5, 1, 207), (8, 1, 3, 200), (5, 5, 21, 30482), (8, 1, 5, 206),
          (5, 5, 33, 3085), (256, 256, 17, 0), (128, 128, 33, 0), (32, 8, 129, 0), (256, 256, 18, 177), (128, 128, 18, 2635),
          (128, 128, 36, 157), (32, 8, 13, 26579), (32, 8, 7, 39047), (32, 8, 131, 64), (5, 5, 150, 13566)]


@pytest.mark.parametrize("hq,hk,rows,position", SHAPES)
@pytest.mark.parametrize("gate", [False, True])
def test_every_form_of_few_rows(hq, hk, rows, position, gate):
    r = rng(hq + 1000 * rows + position)
    n = position + rows
    k, v = (E.DeviceBuffer.from_numpy(kv8.keys(r, n, 1)) for _ in "kv")
    cache, one = kv8.new_cache(hk, n + 3, 0xff), kv8.new_cache(1, n, 0xff)
    for c in (cache, one):
        E.check(E.lib().es_kv8_write(c.struct, k.ptr, v.ptr, DIM, 0, 0, n, None))
    E.synchronize()
    q = kv8.keys(r, rows, hq)
    g = bf16(r.normal(0, 2, (rows, hq, 2 * DIM))) if gate else None
    got = kv8.attend(cache, q, position, g)
    assert np.isfinite(f32(got)).all()
    k, v = (f32(x).astype(np.float64) for x in kv8.read(one, 0, n))
    group = hq // hk
    for i in sorted({0, rows // 3, rows - 1}):
        for h in sorted({0, hk // 2, hk - 1}):
            of = slice(h * group, h * group + group)
            kv8.check_attention(got[i:i + 1, of], q[i:i + 1, of], k[:position + i + 1], v[:position + i + 1], position + i,
                                None if g is None else g[i:i + 1, of])


@pytest.mark.parametrize("hq,hk,rows,position", SHAPES)
def test_every_form_gives_every_row_and_head_its_own(hq, hk, rows, position):
    """Queries of zeros weigh all keys alike, and V says how many there are: every output is known."""
    n = position + rows
    v = np.zeros((n, 1, DIM), np.float32)
    v[:, 0, 0], v[0, 0, 1:] = 1.0, 1.0
    k = E.DeviceBuffer.from_numpy(kv8.keys(rng(3), n, 1))
    v = E.DeviceBuffer.from_numpy(bf16(v))
    cache = kv8.new_cache(hk, n, 0xff)
    E.check(E.lib().es_kv8_write(cache.struct, k.ptr, v.ptr, DIM, 0, 0, n, None))
    E.synchronize()
    got = f32(kv8.attend(cache, np.zeros((rows, hq, DIM), np.uint16), position)).astype(np.float64)
    share = 1 / (position + 1 + np.arange(rows))[:, None, None]
    # probabilities of eight bits, all alike and so all off the same way, sums of n in 32 bits, the output's rounding
    assert (np.abs(got[..., :1] - 1) <= 2.0 ** -8 * 2 + n * 2.0 ** -24).all()
    assert (np.abs(got[..., 1:] - share) <= (2.0 ** -8 * 2 + n * 2.0 ** -24) * share).all()


@pytest.mark.parametrize("hq,hk,rows,position", [(8, 2, 1, 500), (8, 2, 1, 3000), (8, 2, 40, 5000), (32, 8, 131, 64), (8, 2, 9, 30000),
                                                 (32, 8, 700, 300), (8, 2, 2048, 6000)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [8, 11, 14, 16])
def test_large_scores_pick_the_largest(hq, hk, rows, position, sign, size):
    """Scores of 2^size to 2^(size + 10), all of one sign and 32 nats apart at least: every query gets the values of its
    largest key (or keys: those of one score have the same)."""
    n = position + rows
    r = rng(70 + n + size)
    heights = (np.arange(8, 16) / 8 * 2.0 ** np.arange(10)[:, None]).ravel()[:79]  # e4m3 numbers, 1 to 896
    which = r.integers(0, 79, n)
    of_height = kv8.round_e4m3(r.normal(0, 1, (79, DIM)))  # at powers of two of 2^-7 and less what the cache holds
    k = bf16(np.broadcast_to(heights[which][:, None, None], (n, 1, DIM)))
    v = bf16(of_height[which][:, None])
    cache = kv8.new_cache(hk, n, 0xff)
    dk, dv = E.DeviceBuffer.from_numpy(k), E.DeviceBuffer.from_numpy(v)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, DIM, 0, 0, n, None))
    E.synchronize()
    q = bf16(np.full((rows, hq, DIM), sign * 2.0 ** (size - 4)))  # score: q height 256 / 16
    got = f32(kv8.attend(cache, q, position)).astype(np.float64)
    best = (np.maximum if sign > 0 else np.minimum).accumulate(which)[position:]
    want = of_height[best][:, None]
    # a probability's eight bits and the output's rounding
    assert (np.abs(got - want) <= 2.0 ** -7 * np.abs(want) + 1e-12).all()
