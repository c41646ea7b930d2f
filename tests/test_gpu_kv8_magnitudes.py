"""es_attn_prepare_rows_kv8 on projections of any finite bf16 magnitude, on the GPU
against 64 bits: the norm takes it out, whether squares or products with the gain pass
32 bits' range or not."""
import numpy as np
import pytest

import esdecode as E
import kv8
from helpers import bf16, f32, rng
from test_gpu_kv8 import f64, prepare, projections, rotated

pytestmark = pytest.mark.gpu

DIM = 256
LARGEST = 3.3895313892515355e38  # of bf16


def large(r, rows, heads, dims, kind):
    """Rows whose largest magnitude is that of bf16, or 2^60 .. 2^70 where sums of squares pass 2^128, or 1e20."""
    x = r.normal(0, 1, (rows, heads, dims))
    if kind == "one":  # a single dim of each row
        x[:] = 0
        x[np.arange(rows)[:, None], np.arange(heads), r.integers(0, DIM, (rows, heads))] = LARGEST
    elif kind == "largest":
        x = np.clip(x, -2, 2) / 2 * LARGEST
    elif kind == "border":
        x *= np.exp2(r.integers(56, 70, (rows, heads, 1)))
    elif kind == "mixed":  # beside ordinary heads
        x[r.random((rows, heads)) < 0.5] *= 1e30
    else:
        x *= 1e20
    return bf16(x)


KINDS = ["one", "largest", "border", "mixed", "1e20"]


@pytest.mark.parametrize("rows", [1, 2, 70])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gain", [1.0, 3.0])
def test_keys_of_any_magnitude(rows, kind, gain):
    r = rng(40 + rows)
    q, _, v, qg, kg = projections(r, rows, 8, 2)
    kg = bf16(f32(kg) * np.float32(gain))
    k = large(r, rows, 2, DIM, kind)
    cache = kv8.new_cache(2, rows)
    prepare(cache, q, k, v, qg, kg, 0)
    got = f64(kv8.read(cache, 0, rows)[0])
    want = rotated(k, kg, 0, E.rope_inv_freq())
    power = np.exp2(cache.k_scale.numpy(np.uint8).reshape(2, -1).astype(float) - 127).repeat(64, 1)[:, :rows].T[:, :, None]
    # half a step of the code, or of the subnormals' at the block's power of two
    assert (np.abs(got - want) <= 2.0 ** -4 * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -10 * power).all()


@pytest.mark.parametrize("rows", [1, 2, 70])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gain", [1.0, 3.0])
def test_queries_of_any_magnitude(rows, kind, gain):
    r = rng(50 + rows)
    _, k, v, qg, kg = projections(r, rows, 8, 2)
    qg = bf16(f32(qg) * np.float32(gain))
    q = large(r, rows, 8, 2 * DIM, kind)
    got = f64(prepare(kv8.new_cache(2, rows), q, k, v, qg, kg, 0))
    want = rotated(q[..., :DIM], qg, 0, E.rope_inv_freq())
    # the output's rounding, and 32-bit arithmetic: sums of 256 squares, a dozen roundings, an angle's series
    size = np.sqrt((want ** 2).mean(-1, keepdims=True)) * 8
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 64 * 2.0 ** -24 * size).all()
