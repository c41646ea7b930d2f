"""Operators over a tree of drafted tokens on the GPU against their 64-bit models."""
import numpy as np
import pytest
import torch

import esdecode as E
import tree as T

pytestmark = pytest.mark.gpu

HEADS = [(8, 2), (5, 5), (12, 3), (8, 1), (32, 8), (1, 1), (28, 4)]


# --------------------------------------------------------------- attention
@pytest.mark.parametrize("position", [0, 1, 31, 32, 33, 64, 129, 1020, 5003])
@pytest.mark.parametrize("rows,kind", [(1, "chain"), (2, "flat"), (7, "wide"), (31, "random"), (32, "chain"), (33, "holes"),
                                       (63, "wide"), (64, "random")])
def test_attention(rows, kind, position):
    heads = HEADS[(rows + position) % len(HEADS)]
    s = T.attn_case(rows, *heads, position, T.parents_of(kind, rows, position), seed=rows * 7 + position)
    T.check_attn(s, T.run_attn(s))


@pytest.mark.parametrize("heads", HEADS + [(64, 1), (16, 16), (9, 3)])
def test_attention_head_layouts(heads):
    for rows, position in ((3, 700), (64, 97)):
        s = T.attn_case(rows, *heads, position, T.parents_of("random", rows, 3), seed=rows)
        T.check_attn(s, T.run_attn(s))


def test_attention_of_the_most_heads():
    s = T.attn_case(64, 1024, 256, 40, T.parents_of("wide", 64), seed=4)
    T.check_attn(s, T.run_attn(s))


@pytest.mark.parametrize("rows", [1, 16, 64])
def test_attention_at_the_end_of_the_longest_benchmarked_context(rows):
    s = T.attn_case(rows, 8, 2, 131072, T.parents_of("random", rows, 1), seed=rows, capacity=131072)
    T.check_attn(s, T.run_attn(s))


def test_attention_past_two_gigabytes_of_cache():
    """The largest capacity: a KV head's rows take 2^31 bytes, so the second head's lie past 32-bit offsets."""
    capacity = 1 << 22
    s = T.attn_case(3, 4, 2, 200, [-1, 0, 0], seed=5)
    for name in ("k_cache", "v_cache"):
        wide = torch.empty(2, capacity, T.DIM, dtype=torch.bfloat16, device="cuda")
        wide[:, :200] = s[name][:, :200]
        wide[:, capacity - 5000:] = 0.25
        wide[:, 200:300] = torch.nan
        s[name] = wide
    s["capacity"] = capacity
    small = dict(s, k_cache=s["k_cache"][:, :300].contiguous(), v_cache=s["v_cache"][:, :300].contiguous(), capacity=300)
    want = T.run_attn(small)
    size = int(E.lib().es_attn_tree_scratch_bytes(4, 2, 3))
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    out, k_tree = torch.empty_like(want[0]), torch.empty_like(want[1])
    T.call("es_attn_tree", s["q_proj"], s["k_proj"], s["v_proj"], s["q_gain"], s["k_gain"], s["inv_freq"], s["paths"], 3, 4, 2,
           s["k_cache"], s["v_cache"], capacity, 200, scratch, size, k_tree, out)
    assert torch.equal(out, want[0]) and torch.equal(k_tree, want[1])
    # the whole of it: every key of the context but the first 200 is the same
    for name in ("k_cache", "v_cache"):
        s[name][:, 200:] = 0.25
    T.call("es_attn_tree", s["q_proj"], s["k_proj"], s["v_proj"], s["q_gain"], s["k_gain"], s["inv_freq"], s["paths"], 3, 4, 2,
           s["k_cache"], s["v_cache"], capacity, capacity, scratch, size, k_tree, out)
    T.check_attn(dict(s, position=capacity), (out, k_tree), spread=False)


def test_attention_with_one_key_far_above_the_others():
    """Scores of hundreds: the dominant key's value comes out as it is."""
    s = T.attn_case(8, 8, 2, 300, T.parents_of("chain", 8), seed=9)
    place = torch.tensor([300.0 + i for i in range(8)], device="cuda")
    q = T.rotated(s["q_proj"][..., :T.DIM], s["q_gain"], place, s["inv_freq"])
    s["k_cache"][0, 17] = T.bf(40 * q[5, 0].float())
    got = T.run_attn(s)
    T.check_attn(s, got, spread=False)
    z = torch.sigmoid(s["q_proj"][5, 0, T.DIM:].double())
    T.near(got[0][5, 0], s["v_cache"][0, 17].double() * z, T.BF * (s["v_cache"][0, 17].double() * z).abs() * 1.001, "value")


@pytest.mark.parametrize("position", [0, 50])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_keeps_a_nodes_infinities_to_its_descendants(bad, position):
    rows = 40
    parents = T.parents_of("random", rows, 2)
    s = T.attn_case(rows, 8, 2, position, parents, seed=11)
    clean = T.run_attn(s)
    s["v_proj"][5, 1, 3] = bad
    got = T.run_attn(s)
    below = torch.tensor([5 in p for p in s["nodes"]], device="cuda")
    assert 1 < int(below.sum()) < rows - 5
    assert torch.equal(got[0][~below], clean[0][~below])
    hit = got[0][below][:, 4:, 3].float()
    assert (torch.isnan(hit) if np.isnan(bad) else hit == bad).all()
    rest = got[0].clone()
    rest[:, 4:, 3] = clean[0][:, 4:, 3]
    assert torch.equal(rest, clean[0])
    for name in ("k_proj", "q_proj"):
        t = dict(s, v_proj=s["v_proj"].clone())
        t["v_proj"][5, 1, 3] = 0
        t[name] = s[name].clone()
        t[name][7, 1, 9] = bad
        got = T.run_attn(t)
        base = T.run_attn(dict(t, **{name: s[name]}))
        touched = torch.tensor([7 in p if name == "k_proj" else i == 7 for i, p in enumerate(s["nodes"])], device="cuda")
        assert torch.equal(got[0][~touched], base[0][~touched])
        assert torch.isnan(got[0][7, 4 if name == "k_proj" else 1]).all()


def test_attention_nodes_left_out():
    rows, parents = 20, T.parents_of("holes", 20, 6)
    s = T.attn_case(rows, 8, 2, 90, parents, seed=13)
    out = torch.tensor([not p for p in s["nodes"]], device="cuda")
    assert 1 < int(out.sum()) < 15
    want = T.run_attn(s)
    for name in ("q_proj", "k_proj", "v_proj"):
        s[name][out] = torch.nan
    got = T.run_attn(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (got[0][out] == 0).all() and (got[1][out] == 0).all()
    s["paths"][:] = 0  # all of them
    got = T.run_attn(s)
    assert (got[0] == 0).all() and (got[1] == 0).all()
    # bits of later nodes and of rows that are not there count for nothing
    s = T.attn_case(rows, 8, 2, 90, T.parents_of("random", 20, 6), seed=13)
    want = T.run_attn(s)
    later = torch.tensor([-1 << (i + 1) for i in range(rows)], device="cuda")
    got = T.run_attn(dict(s, paths=s["paths"] | later))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_a_nan_in_the_context_reaches_every_node():
    s = T.attn_case(5, 8, 2, 300, T.parents_of("wide", 5), seed=15)
    s["v_cache"][0, 100, 7] = torch.nan
    got = T.run_attn(s)[0]
    assert torch.isnan(got[:, :4, 7]).all() and int(torch.isnan(got).sum()) == 20


def test_attention_of_heads_whose_squares_pass_32_bits():
    s = T.attn_case(6, 8, 2, 64, T.parents_of("chain", 6), seed=17)
    for big in (1e30, 1e-30):
        t = dict(s, q_proj=s["q_proj"].clone(), k_proj=T.bf(s["k_proj"].float() * big))
        t["q_proj"][..., :T.DIM] = T.bf(s["q_proj"][..., :T.DIM].float() * big)
        T.check_attn(t, T.run_attn(t))


def test_attention_tail_of_the_cache_is_not_met():
    """A context that fills the cache to its last row, whatever the last tile holds."""
    for position in (1, 95, 96, 97):
        s = T.attn_case(9, 8, 2, position, T.parents_of("wide", 9), seed=position, capacity=position)
        T.check_attn(s, T.run_attn(s))


# --------------------------------------------------------- Gated DeltaNet
@pytest.mark.parametrize("position", [0, 1, 2, 3, 4097])
@pytest.mark.parametrize("rows,kind", [(1, "chain"), (2, "flat"), (3, "chain"), (5, "wide"), (15, "random"), (16, "chain"),
                                       (17, "holes"), (33, "random"), (48, "wide"), (49, "chain"), (64, "chain"),
                                       (64, "random"), (64, "holes")])
def test_gdn(rows, kind, position):
    s = T.gdn_case(rows, position, T.parents_of(kind, rows, position), seed=rows + 100 * position)
    T.check_gdn(s, T.run_gdn(s))


@pytest.mark.parametrize("a", [-30.0, 30.0, 1e4, 1e38])
def test_gdn_gates_at_their_ends(a):
    """Gates of almost 1, of almost 0 and of 0, with ordinary ones behind them."""
    s = T.gdn_case(30, 5, T.parents_of("random", 30, 1), seed=3)
    s["a_proj"][::2] = a
    s["b_proj"][1::3] = a
    T.check_gdn(s, T.run_gdn(s))


def test_gdn_of_equal_keys():
    """Every key along one direction and beta of almost 1: each update undoes what its path left there."""
    s = T.gdn_case(64, 9, T.parents_of("chain", 64), seed=5)
    s["raw"][:, 2048:4096] = s["raw"][:1, 2048:4096].abs()
    s["ring"][:, 2048:4096] = s["raw"][:1, 2048:4096]
    s["conv_w"] = s["conv_w"].abs()
    s["b_proj"][:] = 6.0
    s["a_proj"][:] = -8.0
    T.check_gdn(s, T.run_gdn(s))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gdn_keeps_a_nodes_nan_to_its_descendants(bad):
    rows, parents = 50, T.parents_of("random", 50, 4)
    s = T.gdn_case(rows, 77, parents, seed=7)
    clean = T.run_gdn(s)
    node = next(i for i in range(1, rows) if 3 < sum(i in p for p in s["nodes"]) < 40)
    below = torch.tensor([node in p for p in s["nodes"]], device="cuda")
    for name, at in (("raw", (node, 2048 + 130)), ("raw", (node, 4096 + 140)), ("a_proj", (node, 1)), ("b_proj", (node, 1))):
        t = dict(s, **{name: s[name].clone()})
        t[name][at] = bad if name == "raw" else float("nan")
        got = T.run_gdn(t)
        for a, b in zip(got, clean):
            assert torch.equal(a[~below], b[~below]), name
        assert torch.isnan(got[0].view(rows, 16, 128)[node, 1]).any()


def test_gdn_of_nan_in_every_block_of_nodes():
    """A block of 16 nodes with a NaN among blocks without: what is not below it stays, call after call."""
    rows, parents = 64, T.parents_of("random", 64, 6)
    s = T.gdn_case(rows, 9, parents, seed=8)
    clean = T.run_gdn(s)
    leaves = [i for i in range(rows) if sum(i in p for p in s["nodes"]) == 1]
    for blocks in ((1,), (2,), (0, 2), (1, 2), (0, 1, 2, 3)):
        bad = [next(i for i in leaves if i // 16 == b) for b in blocks]
        t = dict(s, raw=s["raw"].clone())
        t["raw"][bad] = torch.nan
        fine = torch.ones(rows, dtype=torch.bool, device="cuda")
        fine[bad] = False
        for _ in range(20):
            for a, b in zip(T.run_gdn(t), clean):
                assert torch.equal(a[fine], b[fine]), blocks
                assert a.dtype == torch.float32 and a.shape[1:] == (16,) or torch.isnan(a[bad]).all(), blocks


def test_gdn_nodes_left_out():
    rows, parents = 30, T.parents_of("holes", 30, 8)
    s = T.gdn_case(rows, 6, parents, seed=9)
    out = torch.tensor([not p for p in s["nodes"]], device="cuda")
    want = T.run_gdn(s)
    for name in ("raw", "a_proj", "b_proj"):
        s[name][out] = torch.nan
    got = T.run_gdn(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and (a[out] == 0).all()
    s["state"][3, 5, 7] = torch.inf
    assert all((a[out] == 0).all() for a in T.run_gdn(s))


def test_gdn_of_rows_whose_squares_pass_32_bits():
    s = T.gdn_case(9, 6, T.parents_of("wide", 9), seed=11)
    for big in (1e25, 1e-25):
        t = dict(s, raw=s["raw"].clone(), ring=s["ring"].clone())
        for x in (t["raw"], t["ring"]):
            x[:, :4096] = T.bf(x[:, :4096].float() * big)
        T.check_gdn(t, T.run_gdn(t))


# ------------------------------------------------------ accepted paths
def draft_of(s, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    m = s["rows"]
    keys = torch.nn.functional.normalize(torch.empty(m, 16, 128, device="cuda").normal_(generator=g), dim=-1)
    updates = torch.empty(m, 16, 128, device="cuda").normal_(0, 0.3, generator=g)
    log_decay = -torch.empty(m, 16, device="cuda").exponential_(2.0, generator=g)
    return keys, updates, log_decay


def keep_gdn(s, draft, node, out, stream=None):
    T.call("es_gdn_tree_keep", s["raw"], *draft, s["paths"], node, s["rows"], s["position"], s["ring"], s["state"], out,
           stream=stream)
    torch.cuda.synchronize()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,kind,node", [(1, "chain", 0), (7, "wide", 6), (7, "wide", 0), (20, "random", 13),
                                            (64, "chain", 63), (64, "chain", 40), (64, "random", 63), (5, "chain", 3)])
@pytest.mark.parametrize("position", [0, 1, 3, 1022])
def test_state_behind_a_path(rows, kind, node, position, in_place):
    s = T.gdn_case(rows, position, T.parents_of(kind, rows, 1), seed=rows + node)
    draft = draft_of(s, node)
    state, ring, off = T.kept_state(s, *draft, node)
    old = s["state"].clone()
    out = s["state"] if in_place else torch.full_like(old, torch.nan)
    keep_gdn(s, draft, node, out)
    T.near(out, state, off, "state")
    assert torch.equal(s["ring"], ring)
    assert in_place or torch.equal(s["state"], old)


def test_state_behind_gates_of_zero_and_nodes_off_the_path():
    s = T.gdn_case(12, 5, T.parents_of("random", 12, 3), seed=2)
    keys, updates, log_decay = draft_of(s, 3)
    node = 11
    off_path = torch.tensor([j not in s["nodes"][node] for j in range(12)], device="cuda")
    keys[off_path] = updates[off_path] = torch.nan
    log_decay[off_path] = torch.nan
    log_decay[s["nodes"][node][0], 4] = -torch.inf
    log_decay[s["nodes"][node][-1], 5] = -1e38
    state, ring, off = T.kept_state(s, keys, updates, log_decay, node)
    out = torch.empty_like(s["state"])
    keep_gdn(s, (keys, updates, log_decay), node, out)
    T.near(out, state, off, "state")
    assert torch.equal(out[5], torch.einsum("v,k->vk", updates[node, 5], keys[node, 5]))
    assert torch.equal(s["ring"], ring)


def test_a_node_left_out_keeps_nothing():
    s = T.gdn_case(4, 5, [-1, -2, 0, 0], seed=2)
    old, ring = s["state"].clone(), s["ring"].clone()
    out = torch.empty_like(old)
    keep_gdn(s, draft_of(s, 1), 1, out)
    assert torch.equal(out, old) and torch.equal(s["ring"], ring)
    a = T.attn_case(4, 8, 2, 10, [-1, -2, 0, 0], seed=2)
    kept = a["k_cache"].clone()
    T.call("es_kv_tree_keep", a["k_proj"], a["v_proj"], a["paths"], 1, 4, 2, a["k_cache"], a["v_cache"], a["capacity"], 10)
    torch.cuda.synchronize()
    assert torch.equal(kept.view(torch.int16), a["k_cache"].view(torch.int16))


@pytest.mark.parametrize("heads", [1, 2, 5, 256])
@pytest.mark.parametrize("rows,kind,node,position,capacity", [
    (1, "chain", 0, 0, 1), (7, "wide", 6, 33, 60), (64, "chain", 63, 100, 164), (64, "chain", 63, 100, 130),
    (64, "random", 60, 5, 200), (9, "chain", 8, 50, 51)])
def test_rows_of_a_path_into_the_cache(rows, kind, node, position, capacity, heads):
    s = T.attn_case(rows, heads, heads, position, T.parents_of(kind, rows, 1), seed=rows, capacity=capacity)
    for name in ("k_cache", "v_cache"):
        s[name].normal_()
    want = {name: s[name].clone() for name in ("k_cache", "v_cache")}
    for t, j in enumerate(s["nodes"][node]):
        if position + t < capacity:
            want["k_cache"][:, position + t] = s["k_proj"][j]
            want["v_cache"][:, position + t] = s["v_proj"][j]
    T.call("es_kv_tree_keep", s["k_proj"], s["v_proj"], s["paths"], node, rows, heads, s["k_cache"], s["v_cache"], capacity,
           position)
    torch.cuda.synchronize()
    for name in want:
        assert torch.equal(s[name], want[name])


# ------------------------------------------------- together, and in graphs
def test_a_draft_through_the_layers_and_the_next_step():
    """A chain of drafted tokens through a Gated DeltaNet and an attention layer,
    part of it accepted, then the next: what one pass over all of them gives, and
    what the row operators give, which round to bf16 on the way."""
    n, rows = 70, 12
    s, a = T.gdn_case(rows, n, T.parents_of("chain", rows), seed=1), T.attn_case(rows, 8, 2, n, T.parents_of("chain", rows),
                                                                               seed=2, capacity=n + rows)
    whole = T.run_gdn(s)
    whole_attn = T.run_attn(a)
    first = 5
    part = {k: (s[k][:first].contiguous() if k in ("raw", "a_proj", "b_proj", "paths") else s[k]) for k in s}
    part.update(rows=first, nodes=s["nodes"][:first], ring=s["ring"].clone(), state=s["state"].clone())
    y0, *draft = T.run_gdn(part)
    assert torch.equal(y0, whole[0][:first])
    keep_gdn(part, draft, first - 1, part["state"])
    rest = {k: (s[k][first:].contiguous() if k in ("raw", "a_proj", "b_proj") else s[k]) for k in s}
    rest.update(rows=rows - first, position=n + first, nodes=s["nodes"][:rows - first], paths=s["paths"][:rows - first],
                state=part["state"], ring=part["ring"])
    y1 = T.run_gdn(rest)[0]
    # one state in between, rounded to fp32: the same up to the roundings that check_gdn allows
    T.check_gdn(rest, T.run_gdn(rest))
    assert float((y1.double() - whole[0][first:].double()).norm() / whole[0][first:].double().norm()) < T.BF
    # the row operators on the same tokens
    q, k, v = (torch.empty(rows, 2048, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    g, beta = (torch.empty(rows, 16, device="cuda") for _ in range(2))
    y2, state, ring = torch.empty_like(q), s["state"].clone(), s["ring"].clone()
    T.call("es_gdn_prepare_rows", s["raw"], ring, s["conv_w"], s["a_proj"], s["b_proj"], s["a_log"], s["dt_bias"], n, rows, q, k,
           v, g, beta)
    T.call("es_gdn_recur_rows", q, k, v, g, beta, rows, state, y2)
    torch.cuda.synchronize()
    assert float((y2.double() - whole[0].double()).norm() / whole[0].double().norm()) < 8 * T.BF
    kept = [t.clone() for t in (s["state"], s["ring"])]
    keep_gdn(s, whole[1:], rows - 1, kept[0])
    assert float((kept[0] - state).norm() / state.norm()) < 8 * T.BF
    assert torch.equal(s["ring"], ring)
    # attention: the accepted rows into the cache, then the rest as a draft of its own
    T.call("es_kv_tree_keep", whole_attn[1], a["v_proj"], a["paths"], first - 1, rows, 2, a["k_cache"], a["v_cache"],
           a["capacity"], n)
    torch.cuda.synchronize()
    b = dict(a, rows=rows - first, position=n + first, nodes=a["nodes"][:rows - first], paths=a["paths"][:rows - first])
    for name in ("q_proj", "k_proj", "v_proj"):
        b[name] = a[name][first:].contiguous()
    got = T.run_attn(b)
    T.check_attn(b, got)
    assert torch.equal(got[1], whole_attn[1][first:])
    err = (got[0].double() - whole_attn[0][first:].double()).norm() / got[0].double().norm()
    assert float(err) < 2 * T.BF
    # the row operators over the same cache
    query, gated = torch.empty(rows, 8, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, 2048, dtype=torch.bfloat16,
                                                                                            device="cuda")
    o = torch.empty_like(gated)
    T.call("es_attn_prepare_rows", a["q_proj"], a["k_proj"], a["v_proj"], a["q_gain"], a["k_gain"], a["inv_freq"], n, rows, query,
           a["k_cache"], a["v_cache"], a["capacity"])
    T.call("es_attn_prefill", query, a["k_cache"], a["v_cache"], n, rows, a["capacity"], o)
    T.call("es_attn_gate_rows", o, a["q_proj"], rows, gated)
    torch.cuda.synchronize()
    err = (gated.double().view(rows, 8, 256) - whole_attn[0].double()).norm() / gated.double().norm()
    assert float(err) < 4 * T.BF


def test_graphs_and_other_streams():
    """Each operator captured and replayed with eager work between, and on a stream of its own, with inputs that change."""
    s, a = T.gdn_case(40, 12, T.parents_of("random", 40, 2), seed=3), T.attn_case(40, 8, 2, 2000, T.parents_of("random", 40, 2),
                                                                               seed=4)
    m = 40
    size = int(E.lib().es_attn_tree_scratch_bytes(8, 2, m))
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    bufs = dict(y=torch.empty(m, 2048, dtype=torch.bfloat16, device="cuda"), k=torch.empty(m, 16, 128, device="cuda"),
                u=torch.empty(m, 16, 128, device="cuda"), lg=torch.empty(m, 16, device="cuda"),
                state=torch.empty_like(s["state"]), gated=torch.empty(m, 8, 256, dtype=torch.bfloat16, device="cuda"),
                k_tree=torch.empty(m, 2, 256, dtype=torch.bfloat16, device="cuda"))
    cache = [torch.zeros_like(a["k_cache"]), torch.zeros_like(a["v_cache"])]

    def work():
        T.call("es_gdn_tree", s["raw"], s["ring"], s["conv_w"], s["a_proj"], s["b_proj"], s["a_log"], s["dt_bias"], s["paths"],
               12, m, s["state"], bufs["y"], bufs["k"], bufs["u"], bufs["lg"])
        T.call("es_gdn_tree_keep", s["raw"], bufs["k"], bufs["u"], bufs["lg"], s["paths"], 39, m, 12, s["ring"], s["state"],
               bufs["state"])
        T.call("es_attn_tree", a["q_proj"], a["k_proj"], a["v_proj"], a["q_gain"], a["k_gain"], a["inv_freq"], a["paths"], m, 8,
               2, a["k_cache"], a["v_cache"], a["capacity"], 2000, scratch, size, bufs["k_tree"], bufs["gated"])
        T.call("es_kv_tree_keep", bufs["k_tree"], a["v_proj"], a["paths"], 39, m, 2, *cache, a["capacity"], 2000)

    ring = s["ring"].clone()

    def answer(run):
        s["ring"].copy_(ring)
        for b in list(bufs.values()) + cache:
            b.zero_()
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        return [b.clone() for b in list(bufs.values()) + cache + [s["ring"]]]

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    want = answer(work)
    with torch.cuda.graph(graph):
        work()

    def on_side():
        with torch.cuda.stream(side):
            work()

    for change in range(3):
        for x in (s["raw"], s["a_proj"], a["q_proj"], a["k_proj"], a["v_proj"]):
            x.mul_(-1.0 if change else 1.0)
        parents = T.parents_of(["random", "wide", "chain"][change], m, change)
        s["paths"].copy_(T.words(parents))
        a["paths"].copy_(T.words(parents))
        want = answer(work)
        for run in (graph.replay, on_side, graph.replay):
            for g, w in zip(answer(run), want):
                assert torch.equal(g, w)


def test_two_drafts_at_once():
    """Two streams, each with scratch and outputs of its own, over the same cache and state."""
    rows = [(64, "random"), (9, "wide")]
    gdn = [T.gdn_case(m, 12, T.parents_of(kind, m, 1), seed=5) for m, kind in rows]
    attn = [T.attn_case(m, 8, 2, 9000, T.parents_of(kind, m, 1), seed=6) for m, kind in rows]
    attn[1].update(k_cache=attn[0]["k_cache"], v_cache=attn[0]["v_cache"], capacity=attn[0]["capacity"])
    gdn[1].update(ring=gdn[0]["ring"], state=gdn[0]["state"])
    want = [(T.run_gdn(s), T.run_attn(a)) for s, a in zip(gdn, attn)]
    streams = [torch.cuda.Stream() for _ in rows]
    sizes = [int(E.lib().es_attn_tree_scratch_bytes(8, 2, m)) for m, _ in rows]
    got = [([torch.empty_like(t) for t in w[0]], [torch.empty_like(t) for t in w[1]],
            torch.empty(size, dtype=torch.uint8, device="cuda")) for w, size in zip(want, sizes)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, a, stream, (m, _), (y, o, scratch), size in zip(gdn, attn, streams, rows, got, sizes):
            with torch.cuda.stream(stream):
                T.call("es_gdn_tree", s["raw"], s["ring"], s["conv_w"], s["a_proj"], s["b_proj"], s["a_log"], s["dt_bias"],
                       s["paths"], 12, m, s["state"], *y)
                T.call("es_attn_tree", a["q_proj"], a["k_proj"], a["v_proj"], a["q_gain"], a["k_gain"], a["inv_freq"],
                       a["paths"], m, 8, 2, a["k_cache"], a["v_cache"], a["capacity"], 9000, scratch, size, o[1], o[0])
    torch.cuda.synchronize()
    for (y, o, _), w in zip(got, want):
        for t, u in zip(y + o, list(w[0]) + list(w[1])):
            assert torch.equal(t, u)
