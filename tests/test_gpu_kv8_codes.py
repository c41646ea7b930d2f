"""Prepared keys to the byte, on the GPU: codes and powers of two of the 8-bit cache are those
of the normed and rotated value in 64 bits, over enough values that some lie within a 32-bit
rounding of a boundary between two codes."""
import numpy as np
import pytest

import esdecode as E
import kv8
from helpers import bf16, f32, rng

pytestmark = pytest.mark.gpu

DIM, HEADS, ROWS = 256, 2, 32768


def prepared(k, gain, position, bits=np.float64):
    """[rows, heads, 256]: norm, gain, rotation (angles in 64 bits)."""
    x = f32(k).astype(bits)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + bits(1e-6)) * f32(gain).astype(bits)
    a = (position + np.arange(x.shape[0]))[:, None, None] * E.rope_inv_freq().astype(np.float64)
    lo, hi = x[..., :32].copy(), x[..., 32:64].copy()
    x[..., :32], x[..., 32:64] = lo * np.cos(a).astype(bits) - hi * np.sin(a).astype(bits), \
        lo * np.sin(a).astype(bits) + hi * np.cos(a).astype(bits)
    return x.astype(np.float64)


@pytest.mark.parametrize("position", [0, 98304, (1 << 22) - ROWS])
def test_prepared_keys_to_the_byte(position):
    r = np.random.default_rng(position + 1)
    k = bf16(r.standard_normal((ROWS, HEADS, DIM), dtype=np.float32) * np.exp(r.standard_normal(DIM, dtype=np.float32) * 0.4))
    gain = bf16(r.normal(1, 0.1, DIM))
    d = [E.DeviceBuffer.from_numpy(x) for x in (np.zeros((ROWS, HEADS, 2 * DIM), np.uint16), k, k, gain, gain, E.rope_inv_freq())]
    query = E.DeviceBuffer(ROWS * HEADS * DIM * 2)
    cache = E.DeviceKV8(HEADS, position + ROWS)
    E.check(E.lib().es_attn_prepare_rows_kv8(*(b.ptr for b in d), position, ROWS, HEADS, query.ptr, cache.struct, None))
    E.synchronize()
    blocks, first = ROWS // 64, position // 64
    per_head = -(-(position + ROWS) // 64)
    x, in32 = (prepared(k, gain, position, bits).transpose(1, 0, 2).reshape(HEADS, blocks, 64, DIM)
               for bits in (np.float64, np.float32))
    top = np.abs(x).max((2, 3))
    e = np.vectorize(kv8.exponent)(top)
    near = np.abs(top / 2.0 ** e / 448 - 1) < 2.0 ** -40
    assert not near.any(), "a block's largest on the border of two powers: take another seed"
    for h in range(HEADS):
        got = cache.k_scale.numpy(np.uint8, blocks, h * per_head + first)
        assert np.array_equal(got, e[h] + 127), "powers of two"
        y = x[h] / np.exp2(e[h].astype(float))[:, None, None]
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        # 64-bit arithmetic is off by some 2^-50 of the head's largest dims (at most 16 of its norm)
        off = np.abs(np.abs(y / step - np.floor(y / step) - 0.5) * step)
        sure = off > 2.0 ** -40 * np.abs(y).max(2, keepdims=True)
        codes = kv8.codes_of(kv8.round_e4m3(y))
        got = cache.k.numpy(np.uint8, blocks * 64 * DIM, (h * per_head + first) * 64 * DIM)
        # memory: [token / 32][d / 64][(d / 16) & 1][(d / 32) & 1][token % 32][d % 16]
        got = got.reshape(blocks, 2, 4, 2, 2, 32, 16).transpose(0, 1, 5, 2, 4, 3, 6).reshape(blocks, 64, DIM)
        bad = (got != codes) & sure
        assert not bad.any(), f"head {h}: {bad.sum()} codes differ, first at {np.argwhere(bad)[0]}"
        assert (~sure).sum() < 10
        # the check is one: arithmetic in 32 bits would not pass it
        narrow = kv8.codes_of(kv8.round_e4m3(in32[h] / np.exp2(e[h].astype(float))[:, None, None])) != codes
        assert (narrow & sure).any()
