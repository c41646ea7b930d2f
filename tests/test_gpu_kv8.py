"""The 8-bit key/value cache on the GPU against its plain 64-bit model: bytes
in memory after writes, values read back, attention of one token and of many."""
import numpy as np
import pytest
import torch

import esdecode as E
import kv8
from helpers import bf16, f32, rng

pytestmark = pytest.mark.gpu

DIM = 256


def f64(bits):
    return f32(bits).astype(np.float64)


def same_memory(cache, plain):
    for w, buf, scale in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
        assert np.array_equal(scale.numpy(np.uint8).reshape(plain.e[w].shape), plain.e[w] + 127), f"{w} powers"
        got = buf.numpy(np.uint8).reshape(plain.memory(w).shape)
        bad = np.argwhere(got != plain.memory(w))
        assert not len(bad), f"{w}: {len(bad)} codes differ, first at {bad[0]}"


def same_values(cache, plain, position, rows):
    for got, want in zip(kv8.read(cache, position, rows), plain.read(position, rows)):
        g = f64(got)
        assert np.array_equal(np.isnan(g), np.isnan(want))
        assert np.array_equal(g[~np.isnan(g)], f64(bf16(want.astype(np.float32)))[~np.isnan(g)])


# ---------------------------------------------------------------- writing
@pytest.mark.parametrize("heads,position,rows", [(2, 0, 1), (2, 0, 64), (1, 0, 63), (3, 0, 65), (2, 5, 1), (2, 63, 1),
                                                 (2, 63, 2), (2, 64, 64), (1, 100, 200), (5, 37, 27), (2, 1, 190)])
def test_write_and_read(heads, position, rows):
    r = rng(1000 * position + rows)
    capacity = position + rows + 70
    cache, plain = kv8.new_cache(heads, capacity), kv8.Plain(heads, capacity)
    if position:  # rows that stay, smaller and larger than the new ones
        k, v = kv8.keys(r, position, heads, 0.3), kv8.keys(r, position, heads, 2.0)
        kv8.write(cache, k, v, 0)
        plain.write(f64(k), f64(v), 0)
        same_memory(cache, plain)
    k, v = kv8.keys(r, rows, heads), kv8.keys(r, rows, heads)
    kv8.write(cache, k, v, position)
    plain.write(f64(k), f64(v), position)
    same_memory(cache, plain)
    same_values(cache, plain, 0, position + rows)
    same_values(cache, plain, position, rows)
    same_values(cache, plain, position + rows - 1, 1)


def test_tokens_one_by_one_with_growing_rows():
    r = rng(5)
    cache, plain, once = kv8.new_cache(2, 80), kv8.Plain(2, 80), kv8.Plain(2, 80)
    scale = np.exp2(r.integers(-12, 6, 70))
    k = np.stack([kv8.keys(r, 1, 2, s)[0] for s in scale])
    v = np.stack([kv8.keys(r, 1, 2, s)[0] for s in scale[::-1]])
    for t in range(70):
        kv8.write(cache, k[t:t + 1], v[t:t + 1], t)
        plain.write(f64(k[t:t + 1]), f64(v[t:t + 1]), t)
    same_memory(cache, plain)
    once.write(f64(k), f64(v), 0)
    for w in "kv":
        assert np.array_equal(plain.e[w], once.e[w])


def test_rows_written_again_keep_the_blocks_power():
    r = rng(6)
    cache, plain = kv8.new_cache(2, 128), kv8.Plain(2, 128)
    for position, rows, scale in ((0, 100, 8.0), (40, 3, 0.01), (64, 10, 0.5), (0, 2, 1.0), (1, 127, 100.0)):
        k, v = kv8.keys(r, rows, 2, scale), kv8.keys(r, rows, 2, scale)
        kv8.write(cache, k, v, position)
        plain.write(f64(k), f64(v), position)
        same_memory(cache, plain)


@pytest.mark.parametrize("scale", [0.0, 1e-40, 1e-36, 1e30, 3e38])
def test_magnitudes_at_the_ends_of_bf16(scale):
    r = rng(7)
    x = (np.clip(r.normal(0, 0.3, (66, 2, DIM)), -1, 1) * scale).astype(np.float32)
    x[3, 0, 7] = scale
    k, v = bf16(x), bf16(x[::-1])
    cache, plain = kv8.new_cache(2, 66), kv8.Plain(2, 66)
    kv8.write(cache, k, v, 0)
    plain.write(f64(k), f64(v), 0)
    same_memory(cache, plain)
    same_values(cache, plain, 0, 66)


def test_every_bf16_value():
    """Each finite bf16 as the only value of its row, beside the largest of its block."""
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    bits = bits[np.isfinite(f32(bits))]
    bits = bits[np.argsort(np.abs(f32(bits)), kind="stable")]  # blocks of like magnitude
    rows = -(-bits.size // DIM)
    k = np.zeros((rows, 1, DIM), dtype=np.uint16)
    k.reshape(-1)[:bits.size] = bits
    cache, plain = kv8.new_cache(1, rows), kv8.Plain(1, rows)
    kv8.write(cache, k, k[::-1].copy(), 0)
    plain.write(f64(k), f64(k[::-1]), 0)
    same_memory(cache, plain)
    same_values(cache, plain, 0, rows)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_row_with_a_nan_or_infinity_reads_back_as_nan(bad):
    r = rng(8)
    x, y = r.normal(0, 1, (70, 2, DIM)), r.normal(0, 1, (70, 2, DIM))
    x[5, 0, 3] = x[69, 1, 255] = y[40, 1, 200] = bad
    k, v = bf16(x), bf16(y)
    cache, plain = kv8.new_cache(2, 128), kv8.Plain(2, 128)
    kv8.write(cache, k, v, 0)
    plain.write(f64(k), f64(v), 0)
    same_memory(cache, plain)
    same_values(cache, plain, 0, 70)
    got = f32(kv8.read(cache, 0, 70)[1])
    assert np.isnan(got).all(2).sum() == np.isnan(got).any(2).sum() == 3
    k, v = kv8.keys(r, 20, 2, 50.0), kv8.keys(r, 20, 2, 50.0)  # the NaN stays when the block is rescaled
    kv8.write(cache, k, v, 70)
    plain.write(f64(k), f64(v), 70)
    same_memory(cache, plain)


@pytest.mark.parametrize("bad", [None, np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("scale", [0.0, 1e-40, 1e-36, 1.0, 1e30, 3e38])
def test_rows_one_by_one(scale, bad):
    """Single rows, each larger or smaller than those before it, over two blocks."""
    r = rng(30)
    x = (np.clip(r.normal(0, 0.2, (80, 3, DIM)), -1, 1) * np.exp2(r.integers(-20, 1, (80, 3, 1))) * scale).astype(np.float32)
    y = np.roll(x[::-1], 7, 2)
    if bad is not None:
        x[5, 0, 3] = x[63, 1, 255] = y[40, 1, 200] = y[64, 2, 0] = bad
    k, v = bf16(x), bf16(y)
    cache, plain = kv8.new_cache(3, 128), kv8.Plain(3, 128)
    for i in range(80):
        kv8.write(cache, k[i:i + 1], v[i:i + 1], i)
        plain.write(f64(k[i:i + 1]), f64(v[i:i + 1]), i)
    same_memory(cache, plain)
    same_values(cache, plain, 0, 80)


@pytest.mark.parametrize("row_stride,head_stride", [(1024, 256), (512 + 8, 256), (256, 80 * 256), (264, 8 * 2680), (2000, 768)])
def test_strides(row_stride, head_stride):
    r = rng(9)
    rows, heads = 75, 2
    n = (rows - 1) * row_stride + (heads - 1) * head_stride + DIM
    ks, vs = bf16(r.normal(0, 1, n)), bf16(r.normal(0, 1, n))
    at = (np.arange(rows)[:, None, None] * row_stride + np.arange(heads)[:, None] * head_stride + np.arange(DIM))
    cache, plain = kv8.new_cache(heads, 200), kv8.Plain(heads, 200)
    dk, dv = E.DeviceBuffer.from_numpy(ks), E.DeviceBuffer.from_numpy(vs)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, row_stride, head_stride, 0, rows, None))
    plain.write(f64(ks[at]), f64(vs[at]), 0)
    same_memory(cache, plain)
    ok, ov = E.DeviceBuffer(n * 2), E.DeviceBuffer(n * 2)
    ok.fill(0xa5)
    ov.fill(0xa5)
    E.check(E.lib().es_kv8_read(cache.struct, 0, rows, ok.ptr, ov.ptr, row_stride, head_stride, None))
    for buf, want in zip((ok, ov), plain.read(0, rows)):
        got = buf.numpy(np.uint16)
        assert np.array_equal(f64(got[at]), want)
        rest = np.ones(n, bool)
        rest[at.ravel()] = False
        assert (got[rest] == 0xa5a5).all(), "wrote between the rows"


def test_one_row_for_all_heads():
    """A stride of zero reads the same rows for every head."""
    r = rng(10)
    k, v = kv8.keys(r, 10, 1), kv8.keys(r, 10, 1)
    cache, plain = kv8.new_cache(3, 64), kv8.Plain(3, 64)
    dk, dv = E.DeviceBuffer.from_numpy(k), E.DeviceBuffer.from_numpy(v)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, DIM, 0, 0, 10, None))
    E.synchronize()
    plain.write(f64(k).repeat(3, 1), f64(v).repeat(3, 1), 0)
    same_memory(cache, plain)


# ---------------------------------------------------------------- prepare
def rotated(x, gain, position, inv_freq):
    x = f64(x)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * f64(gain)
    a = (position + np.arange(x.shape[0]))[:, None, None] * inv_freq.astype(np.float64)
    lo, hi = x[..., :32], x[..., 32:64]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a), x[..., 64:]], -1)


def prepare(cache, q_proj, k_proj, v_proj, q_gain, k_gain, position, stream=None):
    rows, hq, _ = q_proj.shape
    d = [E.DeviceBuffer.from_numpy(x) for x in (q_proj, k_proj, v_proj, q_gain, k_gain, E.rope_inv_freq())]
    query = E.DeviceBuffer(rows * hq * DIM * 2 + 64)
    query.fill(0xa5)
    E.synchronize()  # a stream of its own does not wait for the fill
    E.check(E.lib().es_attn_prepare_rows_kv8(*(b.ptr for b in d), position, rows, hq, query.ptr, cache.struct, stream))
    E.synchronize()
    got = query.numpy(np.uint16)
    assert (got[rows * hq * DIM:] == 0xa5a5).all()
    return got[:rows * hq * DIM].reshape(rows, hq, DIM)


def projections(r, rows, hq, hk):
    return (bf16(r.normal(0, 1.5, (rows, hq, 2 * DIM))), bf16(r.normal(0, 0.7, (rows, hk, DIM))),
            bf16(r.normal(0, 1, (rows, hk, DIM))), bf16(r.normal(1, 0.1, DIM)), bf16(r.normal(1, 0.1, DIM)))


@pytest.mark.parametrize("hq,hk,position,rows", [(8, 2, 0, 1), (8, 2, 131071, 1), (8, 2, 61, 9), (8, 2, 4000000, 65),
                                                 (5, 5, 0, 3), (12, 3, 100, 130), (40, 1, 63, 2)])
def test_prepare(hq, hk, position, rows):
    r = rng(position + rows)
    base = position // 64 * 64
    capacity = position + rows
    a = projections(r, rows, hq, hk)
    cache = kv8.new_cache(hk, capacity)
    held = kv8.keys(r, position - base, hk) if position > base else None
    if held is not None:
        kv8.write(cache, held, held, base)
    before = kv8.read(cache, base, position - base) if held is not None else None
    q = f64(prepare(cache, *a, position))
    freq = E.rope_inv_freq()
    want = rotated(a[0][..., :DIM], a[3], position, freq)
    # the output's rounding, and 32-bit arithmetic: sums of 256 squares, a dozen roundings, an angle's series
    size = np.sqrt((want ** 2).mean(-1, keepdims=True)) * 8
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 64 * 2.0 ** -24 * size).all()
    got_k, got_v = (f64(x) for x in kv8.read(cache, position, rows))
    exact_k = rotated(a[1], a[4], position, freq)
    blocks = slice(position // 64, (position + rows - 1) // 64 + 1)
    for w, got, exact in (("k", got_k, exact_k), ("v", got_v, f64(a[2]))):
        e = (cache.k_scale if w == "k" else cache.v_scale).numpy(np.uint8).reshape(hk, -1)[:, blocks].astype(int) - 127
        power = np.exp2(e.repeat(64, 1)[:, position - base:position - base + rows].T.astype(float))[:, :, None]
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(exact / power), 2.0 ** -6))) - 3) * power
        slack = 64 * 2.0 ** -24 * np.sqrt((exact ** 2).mean(-1, keepdims=True)) * 8
        assert (np.abs(got - exact) <= step / 2 + slack).all(), w
        assert np.abs(exact / power).max() <= 448 * (1 + 2.0 ** -18), w
        if held is None and rows >= 64:
            assert (np.abs(exact / power).reshape(-1, hk, DIM)[:64].max((0, 2)) > 223.9).all(), w
    if held is not None:
        for x, y in zip(kv8.read(cache, base, position - base), before):
            assert (np.abs(f64(x) - f64(y)) <= 2.0 ** -4 * np.abs(f64(y)) + 2.0 ** -10 * np.abs(f64(y)).max() / 224).all()


@pytest.mark.parametrize("hq,hk", [(8, 2), (5, 5), (40, 1), (70, 10)])
def test_prepare_one_by_one(hq, hk):
    """The same queries, bit for bit; K and V within what later powers of two round again."""
    r = rng(31)
    q, k, v, qg, kg = projections(r, 70, hq, hk)
    whole, single = kv8.new_cache(hk, 100), kv8.new_cache(hk, 100)
    want = prepare(whole, q, k, v, qg, kg, 30)
    got = [prepare(single, q[i:i + 1], k[i:i + 1], v[i:i + 1], qg, kg, 30 + i) for i in range(70)]
    assert np.array_equal(np.concatenate(got), want)
    assert np.array_equal(whole.k_scale.numpy(np.uint8), single.k_scale.numpy(np.uint8))
    assert np.array_equal(whole.v_scale.numpy(np.uint8), single.v_scale.numpy(np.uint8))
    power = whole.k_scale.numpy(np.uint8).max(), whole.v_scale.numpy(np.uint8).max()
    for a, b, e in zip(kv8.read(whole, 30, 70), kv8.read(single, 30, 70), power):
        a, b = f64(a), f64(b)
        # half a step each: of the value, or of the subnormals (2^-9) at the power of two; the single ones
        # twice where theirs has risen in between, more than once only below half a step
        assert (np.abs(a - b) <= 4 * (2.0 ** -4 * np.abs(a) + 2.0 ** -10 * 2.0 ** (int(e) - 127))).all()
        assert (a != b).mean() < 0.25


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e15, 1e30])
def test_prepare_of_large_and_small_keys(rows, scale):
    """K's norm in 64 bits: of any magnitude the same keys but for the epsilon."""
    r = rng(34)
    q, k, v, qg, kg = projections(r, rows, 8, 2)
    k = bf16(f32(k) * np.float32(scale))
    cache = kv8.new_cache(2, rows)
    prepare(cache, q, k, v, qg, kg, 0)
    got = f64(kv8.read(cache, 0, rows)[0])
    want = rotated(k, kg, 0, E.rope_inv_freq())
    power = np.exp2(cache.k_scale.numpy(np.uint8).reshape(2, -1).astype(float) - 127).repeat(64, 1)[:, :rows].T[:, :, None]
    # half a step of the code, or of the subnormals' at the block's power of two
    assert (np.abs(got - want) <= 2.0 ** -4 * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -10 * power).all()


def test_prepare_of_a_row_with_nan():
    r = rng(4)
    q, k, v, qg, kg = projections(r, 5, 8, 2)
    k[2, 1, 100] = 0x7fc0
    v[3, 0, 1] = 0x7f80
    q[1, 4, 30] = 0xff80
    cache = kv8.new_cache(2, 64)
    got = f32(prepare(cache, q, k, v, qg, kg, 0))
    assert np.isnan(got[1, 4]).any() and np.isnan(got).any(2).sum() == 1
    for x in kv8.read(cache, 0, 5):
        nan = np.isnan(f32(x))
        assert np.array_equal(nan.any(2), nan.all(2))
        assert sorted(map(tuple, np.argwhere(nan.any(2)))) == [(2, 1), (3, 0)]


# -------------------------------------------------------------- attention
def filled(r, heads, keys, capacity=None, scale=1.0):
    """A cache of NaN codes and powers with `keys` rows written, and their values."""
    cache = kv8.new_cache(heads, capacity or keys, 0xff)
    kv8.write(cache, kv8.keys(r, keys, heads, scale), kv8.keys(r, keys, heads), 0)
    plain = [f64(x) for x in kv8.read(cache, 0, keys)]
    return cache, plain


ATTENTION = [(8, 2, 1, 0), (8, 2, 1, 1), (8, 2, 1, 62), (8, 2, 1, 63), (8, 2, 1, 64), (8, 2, 1, 1000), (8, 2, 1, 4095),
             (8, 2, 2, 0), (8, 2, 5, 700), (8, 2, 17, 47), (8, 2, 64, 0), (8, 2, 130, 0), (8, 2, 131, 190), (5, 5, 1, 300),
             (5, 5, 33, 31), (12, 3, 3, 500), (8, 1, 1, 129), (8, 1, 9, 64), (28, 4, 1, 2000), (28, 4, 11, 100),
             (32, 1, 1, 257), (40, 1, 2, 60), (1, 1, 1, 0), (1, 1, 100, 0), (1, 1, 1, 3000), (2, 2, 200, 77)]


@pytest.mark.parametrize("hq,hk,rows,position", ATTENTION)
@pytest.mark.parametrize("gate", [False, True])
def test_attention(hq, hk, rows, position, gate):
    r = rng(hq * 100000 + rows * 1000 + position)
    cache, (k, v) = filled(r, hk, position + rows, position + rows + 5)
    q = kv8.keys(r, rows, hq)
    g = bf16(r.normal(0, 2, (rows, hq, 2 * DIM))) if gate else None
    kv8.check_attention(kv8.attend(cache, q, position, g), q, k, v, position, g)


@pytest.mark.parametrize("rows,position", [(1, 20000), (40, 5000), (300, 900)])
def test_attention_of_rows_in_the_middle(rows, position):
    """Later rows of the cache, some of them NaN, are not seen."""
    r = rng(11)
    keys = position + rows + 100
    cache = kv8.new_cache(2, keys, 0xff)
    k, v = kv8.keys(r, keys, 2), kv8.keys(r, keys, 2)
    k[position + rows + 1, :, 5] = v[position + rows + 3, :, 7] = 0x7fc0
    kv8.write(cache, k, v, 0)
    k, v = (f64(x) for x in kv8.read(cache, 0, position + rows))
    q = kv8.keys(r, rows, 8)
    kv8.check_attention(kv8.attend(cache, q, position), q, k, v, position)


@pytest.mark.parametrize("rows,position", [(1, 500), (5, 60), (90, 10), (300, 0)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_nan_reaches_the_queries_that_attend_to_it_only(rows, position, which):
    r = rng(12)
    n = position + rows
    at = n - rows // 2 - 1  # queries before it stay clean
    k, v = kv8.keys(r, n, 2), kv8.keys(r, n, 2)
    (k if which == "k" else v)[at, 1, 17] = 0x7f80
    cache = kv8.new_cache(2, n, 0xff)
    kv8.write(cache, k, v, 0)
    q = kv8.keys(r, rows, 8)
    got = f32(kv8.attend(cache, q, position))
    nan = np.isnan(got)
    want = np.zeros((rows, 8), bool)
    want[max(0, at - position):, 4:] = True
    assert np.array_equal(nan.all(2), want) and np.array_equal(nan.any(2), want)
    k, v = (f64(x) for x in kv8.read(cache, 0, n))
    kv8.check_attention(bf16(got), q, k, v, position)


def test_a_nan_or_infinity_in_a_query_stays_its_own():
    r = rng(13)
    cache, (k, v) = filled(r, 2, 200)
    q = kv8.keys(r, 40, 8)
    q[3, 2, 9], q[30, 7, 0] = 0x7fc0, 0x7f80
    got = np.isnan(f32(kv8.attend(cache, q, 160)))
    assert sorted(map(tuple, np.argwhere(got.any(2)))) == sorted(map(tuple, np.argwhere(got.all(2)))) == [(3, 2), (30, 7)]


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("scale", [0.0, 1e-3, 5.0, 20.0])
def test_flat_and_peaked_scores(rows, scale):
    r = rng(14)
    cache, (k, v) = filled(r, 2, 800)
    q = kv8.keys(r, rows, 8, scale)
    kv8.check_attention(kv8.attend(cache, q, 800 - rows), q, k, v, 800 - rows, spread=scale < 2)


@pytest.mark.parametrize("rows", [1, 70])
def test_blocks_of_unequal_powers(rows):
    """V blocks of 2^-60 .. 2^60 and K blocks whose largest channels differ by 2^6:
    each block's power of two is its own."""
    r = rng(15)
    n = 64 * 9 + 20
    k, v = r.normal(0, 1, (n, 2, DIM)), r.normal(0, 1, (n, 2, DIM))
    v *= np.exp2(np.repeat(r.integers(-60, 61, -(-n // 64)), 64)[:n, None, None])
    k *= np.exp2(np.repeat(r.integers(-5, 2, -(-n // 64)), 64)[:n, None, None])
    cache = kv8.new_cache(2, n, 0xff)
    kv8.write(cache, bf16(k), bf16(v), 0)
    k, v = (f64(x) for x in kv8.read(cache, 0, n))
    q = kv8.keys(r, rows, 8)
    kv8.check_attention(kv8.attend(cache, q, n - rows), q, k, v, n - rows, spread=False)


@pytest.mark.parametrize("rows", [1, 40])
def test_queries_of_unequal_size(rows):
    r = rng(16)
    cache, (k, v) = filled(r, 2, 500)
    q = r.normal(0, 1, (rows, 8, DIM)) * np.exp2(r.integers(-40, 3, (rows, 8, 1)))
    q[0, 0] = 0.0
    q = bf16(q)
    kv8.check_attention(kv8.attend(cache, q, 500 - rows), q, k, v, 500 - rows)


@pytest.mark.parametrize("rows", [1, 33])
def test_growing_scores_move_the_maximum_in_every_block(rows):
    r = rng(17)
    n = 1000
    k, v = r.normal(0, 0.05, (n, 2, DIM)), r.normal(0, 1, (n, 2, DIM))
    k += np.linspace(-4, 4, n)[:, None, None]
    cache = kv8.new_cache(2, n, 0xff)
    kv8.write(cache, bf16(k), bf16(v), 0)
    k, v = (f64(x) for x in kv8.read(cache, 0, n))
    q = bf16(np.abs(r.normal(0, 0.5, (rows, 8, DIM))) * np.sign(r.normal(0, 1, (rows, 8, 1))))
    kv8.check_attention(kv8.attend(cache, q, n - rows), q, k, v, n - rows, spread=False)


def same_as_in_parts(got, cache, q, position, g=None):
    """Many rows and the same ones some at a time, which other kernels compute:
    NaN in the same places, and each output's error of 2^-8 at most (root mean square) on
    either side, so one vector of another row would be seen among 20000."""
    rows = max(1, 64 * cache.heads // q.shape[1])
    parts = [kv8.attend(cache, q[i:i + rows], position + i, None if g is None else g[i:i + rows])
             for i in range(0, len(q), rows)]
    a, b = f64(got), f64(np.concatenate(parts))
    assert np.array_equal(np.isnan(a), np.isnan(b))
    ok = ~np.isnan(a)
    assert np.linalg.norm((a - b)[ok]) <= 2 * 2.0 ** -8 * np.linalg.norm(b[ok])


def check_some_rows(got, q, k, v, position, group, g=None, heads=(0, -1)):
    n, hk = len(q), k.shape[1]
    for h in sorted({h % hk for h in heads}):
        of = slice(h * group, h * group + group)
        for i in sorted({0, 1, 31 % n, 32 % n, 63 % n, 64 % n, n // 2, n - 2, n - 1}):
            kv8.check_attention(got[i:i + 1, of], q[i:i + 1, of], k[:position + i + 1, h:h + 1], v[:position + i + 1, h:h + 1],
                                position + i, None if g is None else g[i:i + 1, of])


MANY = [(32, 8, 640, 0), (32, 8, 651, 64), (8, 2, 2570, 100), (28, 4, 740, 37), (256, 256, 80, 0), (256, 256, 81, 64),
        (200, 200, 129, 5), (8, 1, 2600, 191), (16, 4, 1300, 700),
        # ranges of keys as well
        (8, 2, 33, 30000), (8, 2, 300, 20000), (1, 1, 97, 60001), (28, 4, 250, 9000), (5, 5, 700, 12345), (16, 4, 1000, 6000),
        (8, 2, 100, 4000), (12, 3, 1500, 5050)]


@pytest.mark.parametrize("hq,hk,rows,position", MANY)
@pytest.mark.parametrize("gate", [False, True])
def test_attention_of_many_rows(hq, hk, rows, position, gate):
    r = rng(hq * 100000 + rows * 1000 + position)
    cache, (k, v) = filled(r, hk, position + rows, position + rows + 5)
    q = kv8.keys(r, rows, hq)
    g = bf16(r.normal(0, 2, (rows, hq, 2 * DIM))) if gate else None
    got = kv8.attend(cache, q, position, g)
    assert np.array_equal(got, kv8.attend(cache, q, position, g))
    same_as_in_parts(got, cache, q, position, g)
    check_some_rows(got, q, k, v, position, hq // hk, g)


@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_a_nan_in_many_rows(which):
    r = rng(23)
    rows, position = 650, 40
    k, v, q = kv8.keys(r, position + rows, 8), kv8.keys(r, position + rows, 8), kv8.keys(r, rows, 32)
    want = np.zeros((rows, 32), bool)
    if which == "q":
        q[400, 9, 3] = 0x7fc0
        want[400, 9] = True
    else:
        (k if which == "k" else v)[position + 333, 5, 77] = 0xff80
        want[333:, 20:24] = True
    cache = kv8.new_cache(8, position + rows + 64, 0xff)
    kv8.write(cache, k, v, 0)
    got = kv8.attend(cache, q, position)
    nan = np.isnan(f32(got))
    assert np.array_equal(nan.all(2), want) and np.array_equal(nan.any(2), want)
    same_as_in_parts(got, cache, q, position)


@pytest.mark.parametrize("kind", ["growing", "peaked", "powers", "queries", "zero"])
def test_scores_of_many_rows(kind):
    r = rng(24)
    rows, position, heads = 660, 130, 8
    n = position + rows
    k, v, q = f32(kv8.keys(r, n, heads)), f32(kv8.keys(r, n, heads)), f32(kv8.keys(r, rows, 32))
    if kind == "growing":  # each block's scores larger than the last's
        k = np.abs(k) * (1 + np.arange(n) // 32)[:, None, None] / 8
        q = np.abs(q)
    elif kind == "peaked":
        q *= 20
    elif kind == "powers":
        k *= np.exp2(r.integers(-10, 3, n // 64 + 1))[np.arange(n) // 64][:, None, None]
        v *= np.exp2(r.integers(-10, 3, n // 64 + 1))[np.arange(n) // 64][:, None, None]
    elif kind == "queries":
        q *= np.exp2(r.integers(-30, 2, (rows, 32)))[..., None]
    else:
        k[:], q[::2] = 0, 0
    cache = kv8.new_cache(heads, n, 0xff)
    kv8.write(cache, bf16(k), bf16(v), 0)
    q = bf16(q)
    got = kv8.attend(cache, q, position)
    same_as_in_parts(got, cache, q, position)
    k, v = (f64(x) for x in kv8.read(cache, 0, n))
    check_some_rows(got, q, k, v, position, 4)


def test_far_behind_in_a_long_cache():
    """Codes of a head beyond 2^31 bytes from the first: capacity 2^22, three heads."""
    cache = kv8.new_cache(3, 1 << 22, 0xff)
    r = rng(18)
    n = 150
    k, v = kv8.keys(r, n, 3), kv8.keys(r, n, 3)
    kv8.write(cache, k, v, (1 << 22) - n)
    kv8.write(cache, k, v, 0)
    for position in ((1 << 22) - n, 0):
        for got, want in zip(kv8.read(cache, position, n), (k, v)):
            g, w = f64(got), f64(want)
            assert (np.abs(g - w) <= 2.0 ** -4 * np.abs(w) + 2.0 ** -10 * np.abs(w).max() / 224).all()
    q = kv8.keys(r, 1, 6)
    kv8.check_attention(kv8.attend(cache, q, n - 1), q, *(f64(x) for x in kv8.read(cache, 0, n)), n - 1)


@pytest.mark.parametrize("rows,hq", [(1, 6), (7, 15), (200, 6)])
def test_all_keys_of_a_long_cache(rows, hq):
    """2^22 keys of three heads, in blocks beyond 2^31 bytes. Keys of zeros weigh all
    values alike: one row everywhere but for the last ones, which are of their own."""
    cache = kv8.new_cache(3, 1 << 22, 0xff)
    r = rng(32)
    n = 1 << 22
    k, v = np.zeros((1, 3, DIM), np.uint16), kv8.keys(r, 1, 3)
    dk, dv = E.DeviceBuffer.from_numpy(k), E.DeviceBuffer.from_numpy(v)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, 0, DIM, 0, n, None))
    E.synchronize()
    last = bf16(f32(kv8.keys(r, 300, 3)) * 2.0 ** 14)
    kv8.write(cache, np.zeros((300, 3, DIM), np.uint16), last, n - 300)
    first, last = (f64(kv8.read(cache, at, m)[1]) for at, m in ((0, 1), (n - 300, 300)))
    got = f64(kv8.attend(cache, kv8.keys(r, rows, hq), n - rows))
    # the block of rows before the last 300 has their power of two, and reads back smaller values
    edge = f64(kv8.read(cache, n - 320, 20)[1])
    total = first[0] * (n - 320) + edge.sum(0)
    for i in range(rows):
        seen = 300 - rows + 1 + i
        want = (total + last[:seen].sum(0)) / (n - 300 + seen)
        size = (np.abs(first[0]) * (n - 320) + np.abs(edge).sum(0) + np.abs(last[:seen]).sum(0)) / n
        # 2^16 blocks added up in 32 bits at most, addends aligned to 2^-12 of the largest, bf16
        off = (2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -12) * size).repeat(hq // 3, 0)
        assert (np.abs(got[i] - want.repeat(hq // 3, 0)) <= off).all(), i


def test_outputs_to_the_last_of_two_gigabytes():
    """rows * q_heads = 2^22: every head has the same keys, so a few rows of a few heads say it all."""
    torch.manual_seed(4)
    heads, rows = 256, 16384
    cache = E.DeviceKV8(heads, rows)
    r = rng(33)
    k, v = kv8.keys(r, rows, 1), kv8.keys(r, rows, 1)
    dk, dv = E.DeviceBuffer.from_numpy(k), E.DeviceBuffer.from_numpy(v)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, DIM, 0, 0, rows, None))
    q = torch.randn(rows, heads, DIM, device="cuda", dtype=torch.bfloat16)
    out = torch.full((rows + 1, heads, DIM), 7.0, device="cuda", dtype=torch.bfloat16)
    need = int(E.lib().es_attn_kv8_scratch_bytes(heads, heads, rows))
    scratch = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    E.check(E.lib().es_attn_kv8(q.data_ptr(), heads, cache.struct, 0, rows, None, scratch.data_ptr(), need, out.data_ptr(),
                                None))
    torch.cuda.synchronize()
    assert (out[rows] == 7.0).all()
    assert bool(torch.isfinite(out).all())
    k, v = (f64(x)[:, :1] for x in kv8.read(cache, 0, rows))
    for i in (0, 63, 8191, rows - 1):
        for h in (0, 101, 255):
            a, b = (x[i:i + 1, h:h + 1].contiguous().view(torch.int16).cpu().numpy().view(np.uint16) for x in (out, q))
            kv8.check_attention(a, b, k[:i + 1], v[:i + 1], i)


# --------------------------------------------------------------- together
def test_a_prompt_and_tokens_after_it():
    """Prompt chunks and single tokens, prepared and attended in order on a stream
    of their own, as a decode loop runs them."""
    r = rng(19)
    hq, hk, chunks = 8, 2, (100, 77, 1, 1, 3, 1)
    total = sum(chunks)
    cache, plain_k, plain_v = kv8.new_cache(hk, total + 3, 0xff), [], []
    stream = E.c_void_p()
    E.check(E.lib().es_stream_create(E.ctypes.byref(stream)))
    position = 0
    for rows in chunks:
        a = projections(r, rows, hq, hk)
        q = prepare(cache, *a, position, stream=stream)
        out = kv8.attend(cache, q, position, a[0], stream=stream)
        k, v = (f64(x) for x in kv8.read(cache, 0, position + rows))
        kv8.check_attention(out, q, k, v, position, a[0])
        plain_k.append(rotated(a[1], a[4], position, E.rope_inv_freq()))
        plain_v.append(f64(a[2]))
        position += rows
    for got, want in zip((k, v), (np.concatenate(plain_k), np.concatenate(plain_v))):
        # a half step of the codes, and once more where a later row raised its block
        assert np.linalg.norm(got - want) <= 2.0 ** -4 * np.linalg.norm(want)
    E.check(E.lib().es_stream_destroy(stream))


def test_captured_and_replayed():
    """Prepare and attention in a captured graph, replayed on new inputs between
    eager calls that use other scratch: every replay equals the eager result."""
    torch.manual_seed(3)
    hq, hk, n = 8, 2, 900
    lib = E.lib()

    def bf(*shape):
        return torch.randn(*shape, device="cuda").to(torch.bfloat16)

    mem = [torch.zeros(hk * 15 * 16384, dtype=torch.uint8, device="cuda") for _ in range(2)]
    mem += [torch.zeros(hk * 15, dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = E.KV8(*(m.data_ptr() for m in mem), hk, 960)
    k, v, gains, freq = bf(n, hk, 256), bf(n, hk, 256), bf(2, 256), torch.from_numpy(E.rope_inv_freq()).cuda()
    E.check(lib.es_kv8_write(cache, k.data_ptr(), v.data_ptr(), 512, 256, 0, n, None))
    size = int(lib.es_attn_kv8_scratch_bytes(hq, hk, 2))
    scratch, other = (torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    qp, kp, vp, query, out = bf(2, hq, 512), bf(2, hk, 256), bf(2, hk, 256), bf(2, hq, 256), bf(2, hq, 256)

    def step(work, to, stream):
        E.check(lib.es_attn_prepare_rows_kv8(qp.data_ptr(), kp.data_ptr(), vp.data_ptr(), gains[0].data_ptr(),
                                             gains[1].data_ptr(), freq.data_ptr(), n, 2, hq, query.data_ptr(), cache,
                                             stream))
        E.check(lib.es_attn_kv8(query.data_ptr(), hq, cache, n, 2, qp.data_ptr(), work.data_ptr(), size, to.data_ptr(),
                                stream))

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(scratch, out, torch.cuda.current_stream().cuda_stream)
    eager = torch.empty_like(out)
    for _ in range(4):
        for t in (qp, kp, vp):
            t.copy_(torch.randn_like(t, dtype=torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step(other, eager, None)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


@pytest.mark.parametrize("hq,hk,rows,n", [(32, 8, 660, 0), (8, 2, 300, 20000), (8, 2, 9, 30000), (8, 2, 1, 5000)])
def test_attention_captured_and_replayed(hq, hk, rows, n):
    """Each form of the kernels, ranges and their joining: replays on new queries, among
    eager calls that use another scratch, equal the eager results."""
    torch.manual_seed(5)
    lib = E.lib()

    def bf(*shape):
        return torch.randn(*shape, device="cuda").to(torch.bfloat16)

    cache = E.DeviceKV8(hk, n + rows)
    k, v = bf(n + rows, hk, 256), bf(n + rows, hk, 256)
    torch.cuda.synchronize()
    E.check(lib.es_kv8_write(cache.struct, k.data_ptr(), v.data_ptr(), hk * 256, 256, 0, n + rows, None))
    E.synchronize()
    size = int(lib.es_attn_kv8_scratch_bytes(hq, hk, rows))
    scratch, other = (torch.empty(max(size, 16), dtype=torch.uint8, device="cuda") for _ in range(2))
    q, out, eager = bf(rows, hq, 256), bf(rows, hq, 256), bf(rows, hq, 256)

    def attend(work, to, stream):
        E.check(lib.es_attn_kv8(q.data_ptr(), hq, cache.struct, n, rows, None, work.data_ptr(), size, to.data_ptr(), stream))

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(scratch, out, torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        q.copy_(torch.randn_like(q, dtype=torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        attend(other, eager, None)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
