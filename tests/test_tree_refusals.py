"""What the operators over trees and the scores of logits refuse, on the CPU: every
call ends at its checks, before any launch (pointers are never followed); and the
path words of a tree."""
import numpy as np
import pytest

import esdecode as E

P = 1 << 33  # any 16-byte aligned address; its multiples lie apart whatever the sizes


def refused(rc, text):
    assert rc == E.ES_ERR_INVALID
    assert text in E.lib().es_last_error().decode()


def test_paths():
    assert E.tree_paths([-1, 0, 0, 1, -1, 4]).tolist() == [1, 3, 5, 11, 16, 48]
    assert E.tree_paths([-1, -2, 1, 0, 2]).tolist() == [1, 0, 0, 9, 0]
    chain = E.tree_paths(list(range(-1, 63)))
    assert chain[63] == np.uint64(0xffffffffffffffff) and chain[31] == 0xffffffff


@pytest.mark.parametrize("bad", [[0], [-1, 1], [-1, 2, 0], [-3], [-1, -2147483648]])
def test_parents_that_are_none(bad):
    with pytest.raises(E.EsError, match="parents"):
        E.tree_paths(bad)


def test_paths_arguments():
    one = np.zeros(65, dtype=np.int32) - 1
    out = np.zeros(65, dtype=np.uint64)
    for rows in (0, -1, 65):
        refused(E.lib().es_tree_paths(one.ctypes.data, rows, out.ctypes.data), "rows")
    refused(E.lib().es_tree_paths(None, 1, out.ctypes.data), "null")
    refused(E.lib().es_tree_paths(one.ctypes.data, 1, None), "null")


ATTN = dict(q_proj=P, k_proj=2 * P, v_proj=3 * P, q_gain=P, k_gain=P, inv_freq=P, paths=P, rows=4, q_heads=8, kv_heads=2,
            kcache=P, vcache=P, capacity=100, position=50, scratch=6 * P, size=1 << 40, k_tree=4 * P, gated=5 * P)
KEEP_KV = dict(k_tree=P, v_proj=P, paths=P, node=3, rows=4, kv_heads=2, kcache=2 * P, vcache=3 * P, capacity=100, position=50)
GDN = dict(raw=P, ring=P, conv_w=P, a_proj=P, b_proj=P, a_log=P, dt_bias=P, paths=P, position=50, rows=4, state=P, y=2 * P,
           keys=3 * P, updates=4 * P, log_decay=5 * P)
KEEP_GDN = dict(raw=P, keys=P, updates=P, log_decay=P, paths=P, node=3, rows=4, position=50, ring=2 * P, state=3 * P,
                state_out=3 * P)
LOGPROB = dict(logits=P, stride=100, rows=3, vocab=100, tokens=2 * P, top=5, scratch=3 * P, size=1 << 40, logprob=4 * P,
               entropy=5 * P, lse=6 * P, top_ids=7 * P, top_logprobs=8 * P)
CALLS = {"es_attn_tree": ATTN, "es_kv_tree_keep": KEEP_KV, "es_gdn_tree": GDN, "es_gdn_tree_keep": KEEP_GDN,
         "es_logprob_rows": LOGPROB}


def call(name, **change):
    args = dict(CALLS[name])
    assert set(change) <= set(args)
    args.update(change)
    return getattr(E.lib(), name)(*args.values(), None)


NOT_POINTERS = ("rows", "q_heads", "kv_heads", "capacity", "position", "size", "node", "stride", "vocab", "top")


@pytest.mark.parametrize("name", ["es_attn_tree", "es_kv_tree_keep", "es_gdn_tree", "es_gdn_tree_keep"])
def test_null_and_unaligned_pointers(name):
    for arg in CALLS[name]:
        if arg in NOT_POINTERS:
            continue
        refused(call(name, **{arg: None}), "paths" if arg == "paths" else "scratch" if arg == "scratch" else "null")
        refused(call(name, **{arg: CALLS[name][arg] + 4}), "aligned")


@pytest.mark.parametrize("name", ["es_attn_tree", "es_kv_tree_keep", "es_gdn_tree", "es_gdn_tree_keep"])
def test_rows_and_positions(name):
    for rows in (0, -1, 65, 2 ** 31 - 1):
        refused(call(name, rows=rows), "rows")
    for position in (-1, -2 ** 31):
        refused(call(name, position=position), "position")


@pytest.mark.parametrize("name", ["es_kv_tree_keep", "es_gdn_tree_keep"])
def test_nodes(name):
    for node in (-1, 4, 2 ** 31 - 1):
        refused(call(name, node=node), "node")


def test_caches_and_heads():
    for name in ("es_attn_tree", "es_kv_tree_keep"):
        for heads in (0, -1, 257):
            refused(call(name, kv_heads=heads), "kv_heads")
        for capacity in (0, -5, (1 << 22) + 1):
            refused(call(name, capacity=capacity), "capacity")
        refused(call(name, position=101), "position")
    refused(call("es_kv_tree_keep", position=100), "position")
    for heads in (0, 7, -8, 1026):
        refused(call("es_attn_tree", q_heads=heads), "q_heads")


OUTPUTS = {  # with their bytes
    "es_attn_tree": dict(k_tree=4 * 2 * 512, gated=4 * 8 * 512, scratch=None),
    "es_kv_tree_keep": dict(kcache=2 * 100 * 512, vcache=2 * 100 * 512),
    "es_gdn_tree": dict(y=4 * 4096, keys=4 * 8192, updates=4 * 8192, log_decay=4 * 64),
    "es_gdn_tree_keep": dict(ring=4 * 12288, state_out=1 << 20),
    "es_logprob_rows": dict(logprob=12, entropy=12, lse=12, top_ids=60, top_logprobs=60, scratch=None)}


@pytest.mark.parametrize("name", OUTPUTS)
def test_aliasing(name):
    """Every output over every other tensor: at its start, and its last 16 bytes over the other's first."""
    wide = {"vocab": 248320, "stride": 248320} if name == "es_logprob_rows" else {}
    for out, size in OUTPUTS[name].items():
        if size is None:
            size = int(E.lib().es_attn_tree_scratch_bytes(8, 2, 4) if name == "es_attn_tree" else
                       E.lib().es_logprob_scratch_bytes(3, 248320, 5))
            assert size > 0
        for other, at in CALLS[name].items():
            if other in NOT_POINTERS or other == out:
                continue
            if not (out == "state_out" and other == "state"):
                refused(call(name, **{out: at}, **wide), "alias")
            refused(call(name, **{out: at - (size - 1) // 16 * 16}, **wide), "alias")


def test_scratch_sizes():
    size = E.lib().es_attn_tree_scratch_bytes
    need = size(8, 2, 4)
    assert need > 0
    refused(call("es_attn_tree", size=need - 1), "scratch")
    for bad in ((0, 2, 4), (8, 0, 4), (8, 3, 4), (8, 2, 0), (8, 2, 65), (1026, 2, 4), (257, 257, 1)):
        assert size(*bad) == 0
    size = E.lib().es_logprob_scratch_bytes
    need = size(3, 248320, 5)
    assert need > 0 and need % 8 == 0
    refused(call("es_logprob_rows", vocab=248320, stride=248320, size=need - 1), "scratch")
    refused(call("es_logprob_rows", vocab=248320, stride=248320, scratch=None), "scratch")
    refused(call("es_logprob_rows", scratch=P + 8), "scratch")
    for bad in ((0, 100, 5), (3, 0, 0), (3, 100, 33), (3, 4, 5), (3, 100, -1), ((1 << 20) + 1, 100, 1), (1, (1 << 22) + 1, 1)):
        assert size(*bad) == 0


def test_logprob_arguments():
    name = "es_logprob_rows"
    refused(call(name, logits=None), "logits")
    refused(call(name, logits=P + 1), "logits")
    for bad in ({"rows": 0}, {"rows": (1 << 20) + 1}, {"vocab": 0}, {"vocab": (1 << 22) + 1}, {"top": -1}, {"top": 33},
                {"vocab": 4}):
        refused(call(name, **bad), "rows")
    for stride in (99, 0, -100, (1 << 40) + 1):
        refused(call(name, stride=stride), "row_stride")
    refused(call(name, tokens=None), "tokens")
    refused(call(name, logprob=None), "tokens")
    refused(call(name, top_ids=None), "top_ids")
    refused(call(name, top_logprobs=None), "top_ids")
    refused(call(name, top=0), "top_ids")
    refused(call(name, tokens=None, logprob=None, entropy=None, lse=None, top=0, top_ids=None, top_logprobs=None), "output")
