"""What the operators of the 8-bit cache refuse, on the CPU: every call ends
at its checks, before any launch (pointers are never followed)."""
import numpy as np
import pytest

import esdecode as E
import kv8

P = 4096  # any 16-byte aligned address


def cache(**change):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, heads=2, capacity=100)
    a.update(change)
    return E.KV8(*a.values())


BAD_CACHES = [({"k": None}, "null cache"), ({"v": None}, "null cache"), ({"k_scale": None}, "null cache"),
              ({"v_scale": None}, "null cache"), ({"heads": 0}, "heads"), ({"heads": 257}, "heads"),
              ({"capacity": 0}, "capacity"), ({"capacity": (1 << 22) + 1}, "capacity"), ({"k": P + 8}, "aligned"),
              ({"v": P + 1}, "aligned")]
BAD_ROWS = [(0, 0), (0, -1), (-1, 1), (100, 1), (99, 2), (0, 101), (2**31 - 1, 2**31 - 1)]


def write(c=None, k=P, v=P, rs=512, hs=256, pos=0, rows=1):
    return E.lib().es_kv8_write(c or cache(), k, v, rs, hs, pos, rows, None)


def read(c=None, k=P, v=2 * P, rs=512, hs=256, pos=0, rows=1):
    return E.lib().es_kv8_read(c or cache(), pos, rows, k, v, rs, hs, None)


def prepare(c=None, ptrs=(P,) * 6, pos=0, rows=1, q_heads=8, query=P):
    return E.lib().es_attn_prepare_rows_kv8(*ptrs, pos, rows, q_heads, query, c or cache(), None)


def attend(c=None, query=P, q_heads=8, pos=0, rows=1, gate=None, scratch=P, size=1 << 30, out=2 * P):
    return E.lib().es_attn_kv8(query, q_heads, c or cache(), pos, rows, gate, scratch, size, out, None)


def refused(rc, text):
    assert rc == E.ES_ERR_INVALID
    assert text in E.lib().es_last_error().decode()


@pytest.mark.parametrize("call", [write, read, prepare, attend])
def test_bad_caches_and_rows(call):
    for change, text in BAD_CACHES:
        refused(call(cache(**change)), text)
    for pos, rows in BAD_ROWS:
        refused(call(pos=pos, rows=rows), "position + rows <= capacity")
    assert E.lib().es_kv8_write(None, P, P, 512, 256, 0, 1, None) == E.ES_ERR_INVALID


@pytest.mark.parametrize("call", [write, read])
def test_bad_rows_of_bf16(call):
    refused(call(k=None), "null")
    refused(call(v=None), "null")
    for bad in ({"k": P + 2}, {"v": P + 8}, {"rs": 516}, {"hs": 252}, {"rs": -512}, {"hs": -256},
                {"rs": (1 << 40) + 8}):
        refused(call(**bad), "aligned")


def test_read_refuses_rows_that_overlap():
    refused(read(v=P), "k == v")
    for rs, hs in ((0, 256), (256, 256), (248, 4096), (504, 256), (512, 248), (512, 512 + 248)):
        refused(read(rs=rs, hs=hs, rows=3), "overlap")
    refused(read(rs=512, hs=0, rows=1), "overlap")


def test_prepare_arguments():
    for i in range(6):
        refused(prepare(ptrs=tuple(None if j == i else P for j in range(6))), "null")
        refused(prepare(ptrs=tuple(P + 4 if j == i else P for j in range(6))), "aligned")
    refused(prepare(query=None), "null")
    for q_heads in (0, -2, 3, 1 << 23):
        refused(prepare(q_heads=q_heads), "q_heads")


def test_attention_arguments():
    refused(attend(query=None), "null")
    refused(attend(out=None), "null")
    for q_heads in (0, -2, 3, 1 << 23):
        refused(attend(q_heads=q_heads), "q_heads")
    for bad in ({"query": P + 8}, {"out": P + 8}, {"gate": P + 2}, {"scratch": P + 4}):
        refused(attend(**bad), "aligned")
    refused(attend(out=P), "alias")
    refused(attend(gate=2 * P), "alias")
    need = E.lib().es_attn_kv8_scratch_bytes(8, 2, 1)
    assert need > 0
    refused(attend(size=need - 1), "scratch")
    refused(attend(scratch=None), "scratch")


def test_scratch_bytes_of_bad_arguments():
    f = E.lib().es_attn_kv8_scratch_bytes
    for a in ((0, 2, 1), (8, 0, 1), (8, 2, 0), (8, 3, 1), (8, 2, -1), (1 << 20, 2, 1 << 20), (512, 512, 1)):
        assert f(*a) == 0, a


def test_plain_model_rounds_as_e4m3():
    """The tests' own model: every code is its own rounding, halfway values go to
    even codes, the layout is a permutation."""
    codes = np.arange(256, dtype=np.uint8)
    codes = codes[(codes & 0x7f) != 0x7f]
    v = kv8.values_of(codes)
    assert np.array_equal(kv8.round_e4m3(v), v)
    assert np.array_equal(kv8.codes_of(v), codes)
    pos = v[:127]
    mid = kv8.round_e4m3((pos[:-1] + pos[1:]) / 2)
    assert np.array_equal(mid, np.where(np.arange(126) % 2 == 0, pos[:-1], pos[1:]))
    for top, e in ((448.0, 0), (449.0, 1), (224.0, -1), (225.0, 0), (1.75, -8), (1.7578125, -7), (0.0, -127),
                   (2.0 ** -133, -127)):
        assert kv8.exponent(top) == e, top
    c = kv8.Plain(1, 64)
    c.y["k"][0] = values = kv8.values_of((np.arange(64 * 256) % 120).astype(np.uint8)).reshape(64, 256)
    c.y["v"][0] = values
    for w in "kv":
        assert np.array_equal(np.sort(c.memory(w).ravel()), np.sort(kv8.codes_of(values).ravel()))
