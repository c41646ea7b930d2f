"""Attention over the 8-bit cache where one key outweighs each of many others by
10 to 18 nats, on the GPU against 64 bits. Each other key alone is too small to
matter and all of them together are not: their share is what a format of the
probabilities with a smallest number, or one that rounds the same way every time,
loses. All KV heads hold the same rows, and every query is the same."""
import numpy as np
import pytest

import esdecode as E
import kv8
from helpers import bf16, f32, rng

pytestmark = pytest.mark.gpu

DIM = 256


class Keys:
    """n keys of which the one at `at` scores `nats` above the rest, whose scores are
    normal with deviation `spread`; values around one, the sink's `sink` times one."""

    def __init__(self, n, nats, spread, sink, at=0):
        r = np.random.default_rng(n + int(8 * nats))
        k = r.standard_normal((n, 1, DIM), dtype=np.float32) * np.float32(spread)
        v = r.standard_normal((n, 1, DIM), dtype=np.float32) * np.float32(0.3) + np.float32(1.0)
        k[at] = nats / 16  # against a query of ones: nats
        v[at] = sink * np.abs(v[at])
        self.n, self.k, self.v = n, E.DeviceBuffer.from_numpy(bf16(k)), E.DeviceBuffer.from_numpy(bf16(v))
        one = self.cache(1)
        self.plain = [f32(x)[:, 0].astype(np.float64) for x in kv8.read(one, 0, n)]

    def cache(self, heads):
        cache = kv8.new_cache(heads, self.n, 0xff)
        E.check(E.lib().es_kv8_write(cache.struct, self.k.ptr, self.v.ptr, DIM, 0, 0, self.n, None))
        E.synchronize()
        return cache

    def want(self, rows):
        """The last `rows` outputs in 64 bits, and how far they may be off.

        A probability has eight significant bits: off by 2^-8 of itself, or, where that is less than `lost`, by that.
        Scores: the addends of an 8-bit product are aligned to 2^-12 of the largest (eight products), and an error of
        all scores by d moves an output by 2 d times the weighted mean of |v|; so are the sums of 64 values.
        Sums of n in 32 bits. The output's rounding: 2^-8."""
        k, v = self.plain
        s = k.sum(1) / 16
        p = np.exp(s - s.max())
        total = np.cumsum(p)[-rows:, None]
        out = np.cumsum(p[:, None] * v, 0)[-rows:] / total
        mean = np.cumsum(p[:, None] * np.abs(v), 0)[-rows:] / total
        few = np.cumsum(lost(p)[:, None] * np.abs(v), 0)[-rows:] / total
        weighted = np.concatenate([p[:, None] * np.abs(v), np.zeros((-self.n % 64, DIM))])
        largest = weighted.reshape(-1, 64, DIM).max(1).sum(0) / total
        d = 8 * 2.0 ** -12 * np.abs(k).max() / 16
        off = (2.0 ** -8 + 2 * d + self.n * 2.0 ** -24) * mean + few + 2.0 ** -12 * largest
        return out, off + 2.0 ** -8 * np.abs(out)


def lost(p):
    """How far a small probability may be off. 32 keys of a block (16 j + 0 .. 7 or 16 j + 8 .. 15) share a power of
    two that brings their largest to at least 2^7, and the lower parts have steps of 2^-14: 2^-22 of the largest
    at most, and of a key that comes out as zero no more than itself. Where the largest of the 32 outweighs the other
    three of its four eights by 2^13, these have a power of two by their own largest. (The eights: of successive
    tokens, or of four and the four 16 further on, by kernel.)"""
    out = np.zeros(-(-p.size // 64) * 64)
    out[:p.size] = p
    tokens = np.arange(64)
    for b in range(out.size // 64):
        block = out[b * 64:b * 64 + 64]  # a view: replaced below
        ref = np.empty(64)
        for half in range(2):
            of = tokens[(tokens >> 3 & 1) == half]
            top = of[block[of].argmax()]
            beside = (of >> 3 == top >> 3) | ((of >> 5 == top >> 5) & (of >> 2 & 1 == top >> 2 & 1))
            rest = block[of[~beside]].max()
            ref[of] = np.where(beside | (rest >= 2.0 ** -14 * block[top]), block[top], rest)
        block[:] = np.minimum(block, 2.0 ** -22 * ref)
    return out[:p.size]


def check(keys, heads, group, rows):
    cache = keys.cache(heads)
    got = f32(kv8.attend(cache, np.full((rows, heads * group, DIM), 0x3f80, np.uint16), keys.n - rows)).astype(np.float64)
    want, off = keys.want(rows)
    bad = ~(np.abs(got - want[:, None]) <= off[:, None])
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        share = got.sum() / (want.sum() * heads * group)
        raise AssertionError(f"{bad.mean():.1%} off, first {i}: got {got[i]!r} want {want[i[0], i[2]]!r} "
                             f"+- {off[i[0], i[2]]:.3g}; sum of outputs {share:.4f} of what it should be")


NATS = [10, 12, 13, 14, 18]
# query heads a KV head, KV heads, rows, keys
MANY = [(4, 8, 700, 1024), (4, 8, 700, 16384), (4, 2, 2048, 16384), (1, 128, 130, 4096), (8, 1, 400, 16384), (4, 8, 700, 32768),
        (4, 8, 660, 660)]
SPREAD = [(10, 1.0, 0.0, 0), (13, 1.0, 0.0, 77), (12, 2.0, 0.0, 0), (12, 0.0, -1.0, 0), (9.75, 0.0, -1.0, 500),
          (14, 1.0, 0.01, 640), (30, 4.0, 0.0, 3)]


@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("group,heads,rows,n", MANY)
def test_many_rows_behind_a_sink_without_value(group, heads, rows, n, nats):
    check(Keys(n, nats, 0.0, 0.0), heads, group, rows)


@pytest.mark.parametrize("nats,spread,sink,at", SPREAD)
@pytest.mark.parametrize("group,heads,rows,n", [(4, 8, 700, 16384), (4, 2, 2048, 16384)])
def test_many_rows_with_scores_that_differ_and_sinks_with_values(group, heads, rows, n, nats, spread, sink, at):
    check(Keys(n, nats, spread, sink, at), heads, group, rows)


@pytest.mark.parametrize("nats", [22, 30, 38])
@pytest.mark.parametrize("group,heads,rows,n", [(4, 8, 700, 2048), (4, 8, 700, 16384)])
def test_many_rows_with_a_rest_far_below(group, heads, rows, n, nats):
    """The rest keeps its eight bits however far it lies below, as far as the sink has no value."""
    check(Keys(n, nats, 0.0, 0.0), heads, group, rows)


FEW = [(4, 2, 1, 700), (4, 2, 1, 1024), (8, 1, 1, 1024), (8, 1, 1, 4096), (4, 8, 1, 20011), (4, 2, 1, 131072), (1, 32, 1, 16384),
       (1, 128, 1, 131072), (4, 2, 12, 4096), (4, 2, 40, 20040), (4, 2, 128, 28800), (8, 1, 100, 16384), (1, 256, 80, 80),
       (4, 2, 30, 640)]


@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("group,heads,rows,n", FEW)
def test_few_rows_behind_a_sink_without_value(group, heads, rows, n, nats):
    check(Keys(n, nats, 0.0, 0.0), heads, group, rows)


@pytest.mark.parametrize("nats,spread,sink,at", SPREAD)
@pytest.mark.parametrize("group,heads,rows,n", [(4, 2, 1, 1024), (4, 8, 1, 20011), (4, 2, 40, 20040), (1, 128, 2, 65536),
                                                (4, 8, 20, 700)])
def test_few_rows_with_scores_that_differ_and_sinks_with_values(group, heads, rows, n, nats, spread, sink, at):
    check(Keys(n, nats, spread, sink, min(at, n - rows)), heads, group, rows)


@pytest.mark.parametrize("nats", [22, 30, 38])
@pytest.mark.parametrize("group,heads,rows,n", [(4, 2, 1, 128), (4, 2, 1, 4096), (4, 2, 130, 900)])
def test_few_rows_with_a_rest_far_below(group, heads, rows, n, nats):
    """The rest keeps its eight bits however far it lies below, as far as the sink has no value."""
    check(Keys(n, nats, 0.0, 0.0), heads, group, rows)
