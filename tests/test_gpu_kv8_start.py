"""An 8-bit cache whose first rows start inside a block, as after a part of the context was
dropped, on the GPU: such a block has no rows, which its scale bytes say (255)."""
import numpy as np
import pytest

import esdecode as E
import kv8
from helpers import rng
from test_gpu_kv8 import f64, prepare, projections

pytestmark = pytest.mark.gpu

DIM = 256


def used_memory(heads, capacity):
    """Memory of a cache's sizes, filled and given back, for the next allocations to find."""
    cache = kv8.new_cache(heads, capacity, 0xa5)
    E.synchronize()
    for b in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        b.close()


@pytest.mark.parametrize("heads,capacity", [(1, 1), (2, 200), (8, 5000), (3, 64)])
def test_a_new_cache_has_no_rows(heads, capacity):
    used_memory(heads, capacity)
    cache = E.DeviceKV8(heads, capacity)
    for b in (cache.k_scale, cache.v_scale):
        got = b.numpy(np.uint8)
        assert got.size == heads * -(-capacity // 64) and (got == 255).all()


def expected(x, position):
    """x [rows, heads, 256] as it reads back where its first block has no rows before it."""
    out = np.empty_like(x)
    rows = x.shape[0]
    for lo in range(position // 64 * 64, position + rows, 64):
        of = slice(max(lo - position, 0), min(lo + 64 - position, rows))
        for h in range(x.shape[1]):
            e = kv8.exponent(np.abs(x[of, h]).max())
            out[of, h] = kv8.round_e4m3(x[of, h] * 2.0 ** -e) * 2.0 ** e
    return out


@pytest.mark.parametrize("position,rows", [(30, 1), (63, 1), (30, 2), (5, 59), (5, 60), (1, 150), (127, 100)])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_rows_from_the_middle_of_a_new_cache(position, rows, scale):
    used_memory(2, position + rows)
    cache = E.DeviceKV8(2, position + rows)
    r = rng(60 + position + rows)
    k, v = kv8.keys(r, rows, 2, scale), kv8.keys(r, rows, 2, scale)
    kv8.write(cache, k, v, position)
    for got, x in zip(kv8.read(cache, position, rows), (k, v)):
        assert np.array_equal(f64(got), expected(f64(x), position))


@pytest.mark.parametrize("hq,hk", [(8, 2), (5, 5), (40, 1), (70, 10)])
@pytest.mark.parametrize("position", [0, 30])
def test_prepared_one_by_one_and_at_once(hq, hk, position):
    """The same queries and powers of two, bit for bit, and the same K and V but for what becomes subnormal."""
    r = rng(31 + position)
    a = projections(r, 70, hq, hk)
    whole, single = E.DeviceKV8(hk, 100), E.DeviceKV8(hk, 100)
    want = prepare(whole, *a, position)
    got = [prepare(single, *(x[i:i + 1] for x in a[:3]), *a[3:], position + i) for i in range(70)]
    assert np.array_equal(np.concatenate(got), want)
    for w in ("k_scale", "v_scale"):
        assert np.array_equal(getattr(whole, w).numpy(np.uint8), getattr(single, w).numpy(np.uint8))
    for x, y, scale in zip(kv8.read(whole, position, 70), kv8.read(single, position, 70), (whole.k_scale, whole.v_scale)):
        x, y = f64(x), f64(y)
        e = scale.numpy(np.uint8).reshape(hk, -1).astype(float) - 127
        power = np.exp2(e.repeat(64, 1)[:, position:position + 70].T)[:, :, None]
        # A power of two changes no rounding but a subnormal one. There: half a step (2^-10 of the power) for the rows at once;
        # for single ones half a step at each lower power, 2^-10 (1 + 1/2 + ..), and 2^-4 of what is below 2^-6. A value
        # below 2^-6 reads as that itself from 15/16 of it on in one rounding, and from 14.5/16 in two (15/16 at half the
        # power, then a tie), but never as more: what reads as more than 2^-6 is no subnormal at any of the powers.
        normal = np.maximum(np.abs(x), np.abs(y)) > 2.0 ** -6 * power
        assert np.array_equal(x[normal], y[normal])
        assert (np.abs(x - y) <= 4 * 2.0 ** -10 * power).all()
        assert normal.mean() > 0.9
