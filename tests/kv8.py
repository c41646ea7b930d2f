"""Plain 64-bit model of the 8-bit key/value cache: its rounding, its layout in
memory and attention over it (numpy)."""
import numpy as np

import esdecode as E
from helpers import bf16, f32

BLOCK, DIM, TOP = 64, 256, 448.0


def exponent(largest):
    """Smallest e >= -127 with largest * 2^-e <= 448 (-127 for zero)."""
    if largest == 0.0:
        return -127
    e = int(np.floor(np.log2(largest))) - 8
    e += int(largest > TOP * 2.0 ** e)
    return max(e, -127)


def round_e4m3(y):
    """To the nearest e4m3, ties to even (|y| <= 448)."""
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.round(y / step) * step


def codes_of(values):
    """e4m3 bit patterns of values that e4m3 holds; NaN gives 0x7f."""
    nan = np.isnan(values)
    a = np.abs(np.where(nan, 0.0, values))
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6).astype(int)
    mant = np.round(a / np.exp2(e - 3.0)).astype(int)  # 0 .. 15
    bits = np.where(mant >= 8, ((e + 7) << 3) | (mant & 7), mant)
    return np.where(nan, 0x7f, bits | (np.signbit(values) << 7)).astype(np.uint8)


def values_of(codes):
    e, m = (codes >> 3) & 15, codes & 7
    v = np.where(e > 0, (8 + m) * np.exp2(e - 10.0), m * np.exp2(-9.0))
    v = np.where((codes & 0x7f) == 0x7f, np.nan, v)
    return np.where(codes >> 7, -v, v)


class Plain:
    """Values of a cache before the powers of two: y [heads, blocks*64, 256] e4m3 numbers, e [heads, blocks]."""

    def __init__(self, heads, capacity, fill=0xa5):
        self.heads, self.blocks = heads, -(-capacity // BLOCK)
        shape = (heads, self.blocks * BLOCK, DIM)
        self.y = {w: values_of(np.full(shape, fill, dtype=np.uint8)) for w in "kv"}
        self.e = {w: np.full((heads, self.blocks), fill - 127) for w in "kv"}

    def write(self, k, v, position):
        """k, v [rows, heads, 256] float64."""
        rows = k.shape[0]
        poison = ~(np.isfinite(k).all(2) & np.isfinite(v).all(2))
        for w, x in (("k", k), ("v", v)):
            x = np.where(np.isfinite(x), x, 0.0)
            for h in range(self.heads):
                for b in range(position // BLOCK, (position + rows - 1) // BLOCK + 1):
                    lo, hi = max(position, b * BLOCK), min(position + rows, (b + 1) * BLOCK)
                    new = x[lo - position:hi - position, h]
                    e = exponent(np.abs(new).max())
                    if lo > b * BLOCK:
                        old = self.e[w][h, b]
                        e = max(e, old)
                        held = self.y[w][h, b * BLOCK:lo]
                        held[:] = round_e4m3(held * 2.0 ** (old - e))
                    self.e[w][h, b] = e
                    y = round_e4m3(new * 2.0 ** -float(e))
                    if w == "k":
                        y[poison[lo - position:hi - position, h]] = np.nan
                    self.y[w][h, lo:hi] = y

    def read(self, position, rows):
        """[rows, heads, 256] values of K and V; NaN for a position that holds one."""
        out = []
        for w in "kv":
            p = np.exp2(self.e[w].astype(np.float64)).repeat(BLOCK, 1)[:, :, None]
            out.append((self.y[w] * p)[:, position:position + rows].transpose(1, 0, 2).copy())
        out[1][np.isnan(out[0]).any(2)] = np.nan
        return out

    def memory(self, which):
        """Codes as they lie in memory: [heads, blocks, 16384]."""
        c = codes_of(self.y[which]).reshape(self.heads, self.blocks, BLOCK, DIM)
        if which == "k":
            c = c.reshape(self.heads, self.blocks, 2, 32, 4, 2, 2, 16).transpose(0, 1, 2, 4, 6, 5, 3, 7)
        else:  # token = 16 s + 8 u + 4 h + b
            c = c.reshape(self.heads, self.blocks, 4, 2, 2, 4, 8, 32).transpose(0, 1, 6, 3, 4, 7, 2, 5)
        return c.reshape(self.heads, self.blocks, BLOCK * DIM)


def new_cache(heads, capacity, fill=0xa5):
    c = E.DeviceKV8(heads, capacity)
    for b in (c.k, c.v, c.k_scale, c.v_scale):
        b.fill(fill)
    return c


def write(cache, k, v, position, stream=None):
    """k, v [rows, heads, 256] bf16 bits."""
    dk, dv = E.DeviceBuffer.from_numpy(k), E.DeviceBuffer.from_numpy(v)
    E.check(E.lib().es_kv8_write(cache.struct, dk.ptr, dv.ptr, k.shape[1] * DIM, DIM, position, k.shape[0], stream))
    E.synchronize()


def read(cache, position, rows):
    n = rows * cache.heads * DIM
    dk, dv = E.DeviceBuffer(n * 2), E.DeviceBuffer(n * 2)
    E.check(E.lib().es_kv8_read(cache.struct, position, rows, dk.ptr, dv.ptr, cache.heads * DIM, DIM, None))
    return [b.numpy(np.uint16, n).reshape(rows, cache.heads, DIM) for b in (dk, dv)]


def attend(cache, query, position, gate=None, stream=None):
    """query [rows, q_heads, 256] bf16 bits, gate [rows, q_heads, 512] or None -> out bits."""
    rows, hq, _ = query.shape
    dq, out = E.DeviceBuffer.from_numpy(query), E.DeviceBuffer(query.nbytes + 64)
    out.fill(0xa5)
    dg = None if gate is None else E.DeviceBuffer.from_numpy(gate)
    need = int(E.lib().es_attn_kv8_scratch_bytes(hq, cache.heads, rows))
    scratch = E.DeviceBuffer(need + 64)
    scratch.fill(0xff)
    E.synchronize()  # a stream of its own does not wait for the fills
    E.check(E.lib().es_attn_kv8(dq.ptr, hq, cache.struct, position, rows, dg.ptr if dg else None,
                                scratch.ptr if need else None, need, out.ptr, stream))
    E.synchronize()
    got = out.numpy(np.uint16, query.size + 32)
    assert (got[query.size:] == 0xa5a5).all(), "wrote behind the output"
    assert (scratch.numpy(np.uint8)[need:] == 0xff).all(), "wrote behind the scratch"
    return got[:query.size].reshape(query.shape)


def attention(query, k, v, position, gate=None):
    """64-bit attention of bf16 queries over k, v [keys, heads, 256]; the outputs
    and, for each, how far 32-bit sums, 8-bit products and probabilities of eight
    significant bits may be off (the rounding of the output not counted).

    A probability is off by at most 2^-8 of itself (hi and lo, four significant
    bits each) or, small ones, by half the step 2^-9 of e4m3 at a largest of
    2^8 (2^-18); the addends of an 8-bit product are aligned to 2^-12 of the
    largest, in the scores (eight products of the 256 dims) and in the sums of 64 keys. An error
    d of all scores moves an output by at most 2 d times the weighted mean of |v|.
    """
    q = f32(query).astype(np.float64)
    rows, hq, _ = q.shape
    group = hq // k.shape[1]
    out, off = np.empty(q.shape), np.empty(q.shape)
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        for r in range(rows):
            n = position + r + 1
            with np.errstate(invalid="ignore", over="ignore"):
                s = kh[:n] @ q[r, h] / 16
                p = np.exp(s - np.nanmax(s)) if not np.isnan(s).any() else np.full(n, np.nan)
                total = p.sum()
                out[r, h] = p @ vh[:n] / total
                mean = p @ np.abs(vh[:n]) / total
                pv = p[:, None] * np.abs(vh[:n])
            pad = np.zeros((-n % BLOCK, DIM))
            largest = np.concatenate([pv, pad]).reshape(-1, BLOCK, DIM).max(1).sum(0) / total
            small = 2.0 ** -18 * np.abs(vh[:n]).sum(0) / total
            d = 8 * 2.0 ** -12 * np.abs(kh[:n] * q[r, h]).max() / 16
            off[r, h] = (2.0 ** -8 + 2 * d) * mean + small + 2.0 ** -12 * largest
            off[r, h] += n * 2.0 ** -24 * mean
    if gate is not None:
        g = f32(gate).astype(np.float64)[..., DIM:]
        out, off = out / (1 + np.exp(-g)), off / (1 + np.exp(-g))
    return out, off


def check_attention(got, query, k, v, position, gate=None, spread=True):
    want, off = attention(query, k, v, position, gate)
    g = f32(got).astype(np.float64)
    assert (np.isnan(g) == np.isnan(want)).all(), "NaN in other places"
    ok = ~np.isnan(want)
    bound = off + 2.0 ** -8 * np.abs(want) + 1e-38
    bad = ok & ~(np.abs(g - want) <= bound)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{bad.sum()} of {bad.size} off, first {i}: got {g[i]!r} want {want[i]!r} +- {bound[i]:.3g}")
    if spread and ok.any():  # roundings of 2^-8 at most, independent of each other: their root mean square is below that
        err = np.linalg.norm((g - want)[ok]) / np.linalg.norm(want[ok])
        assert err <= 2.0 ** -8, f"root mean square error {err:.2e} of the output's"


def keys(r, rows, heads, scale=1.0):
    return bf16(r.normal(0, scale, (rows, heads, DIM)))
