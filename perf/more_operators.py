"""Performance cases of the operators that check a tree of drafted tokens and
score tokens, through the C ABI of include/es_decode.h (the esdecode binding),
beside the same operators in their plain form.

A draft is a tree of up to 64 tokens behind `position` consumed ones: paths[i]
has bit i and the bits of node i's ancestors, which come before it, so a node's
own position is position + popcount(paths[i]) - 1.

  attn      one attention layer over the tree: queries and keys of each node
            RMS-normalised and rotated at its position (both held in bf16, as
            the cache and the query tensors hold them), attention to the whole
            context and to the node's path, output gate
  gdn       one Gated DeltaNet layer over the tree, the state left as it is:
            convolution along the path, delta rule along the path
  gdn_keep  the layer's state and convolution ring behind an accepted path
  kv_keep   the keys and values of an accepted path into the cache
  logprob   log probabilities of given tokens, entropy and top alternatives of
            rows of logits

Inputs are random with the distributions the model has: K rows of unit variance
with channels of unequal size, scores of unit variance, gains N(1, 0.1),
convolution weights N(0, 0.5), A_log = log U(0.5, 2), dt_bias N(-1, 0.5), logits
with a few tokens far above the rest.
"""
import math
import os
import random
import sys

import torch

own = False

DIM, ROTARY, TREE = 256, 64, 64               # attention heads, rotated dims, most nodes
GDN_HEADS, GDN_DIM, CONV = 16, 128, 6144
VOCAB, MAX_CONTEXT, MAX_ROWS = 248320, 131072, 2048
HEADS = [(8, 2), (8, 2), (8, 2), (16, 4), (32, 8), (12, 3), (8, 1), (5, 5), (28, 4)]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token behind a short context: bound by latency
        {"name": "attn_1_at_1020", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 1020, "rows": 1, "deep": 1},
        # a small draft in the middle of a long context
        {"name": "attn_7_at_33001", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 33001, "rows": 7,
         "deep": 4},
        # a middle-sized draft of a model with more heads
        {"name": "attn_21_at_20010_of_32_heads", "kind": "attn", "q_heads": 32, "kv_heads": 8, "position": 20010,
         "rows": 21, "deep": 6},
        # the largest draft at the end of the longest benchmarked context
        {"name": "attn_64_at_131008", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 131008, "rows": 64,
         "deep": 9},
        # a small draft through a Gated DeltaNet layer
        {"name": "gdn_5", "kind": "gdn", "position": 4097, "rows": 5, "deep": 3},
        # the largest draft, with a long path in it
        {"name": "gdn_64", "kind": "gdn", "position": 131008, "rows": 64, "deep": 24},
        # two accepted tokens of a small draft into the state
        {"name": "gdn_keep_2", "kind": "gdn_keep", "position": 4097, "rows": 7, "deep": 2},
        # a long chain accepted whole
        {"name": "gdn_keep_48", "kind": "gdn_keep", "position": 70000, "rows": 48, "deep": 48},
        # three accepted tokens of a small draft into the cache
        {"name": "kv_keep_3", "kind": "kv_keep", "kv_heads": 2, "position": 33001, "rows": 7, "deep": 3},
        # a long path of a large draft of a model with more heads
        {"name": "kv_keep_40_of_8_heads", "kind": "kv_keep", "kv_heads": 8, "position": 20010, "rows": 64, "deep": 40},
        # a sampled token's log probability with its alternatives: one row of the model's vocabulary
        {"name": "logprob_1", "kind": "logprob", "rows": 1, "vocab": VOCAB, "stride": VOCAB, "top": 20,
         "masked": False},
        # the log probabilities of a prompt's tokens
        {"name": "logprob_2048", "kind": "logprob", "rows": MAX_ROWS, "vocab": VOCAB, "stride": VOCAB, "top": 5,
         "masked": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "gdn", "gdn_keep", "kv_keep", "logprob", "logprob"])
    if kind == "logprob":
        vocab = rng.choice([VOCAB, _log_int(rng, 40, 300000)])
        case = {"kind": kind, "rows": _log_int(rng, 1, min(32768, MAX_ROWS * VOCAB // vocab)), "vocab": vocab}
        case["stride"] = vocab + rng.choice([0, 0, rng.randrange(64)])
        case["top"] = rng.choice([0, 1, rng.randrange(2, 33)])
        case["masked"] = rng.random() < 0.25
        if case["rows"] * case["stride"] > MAX_ROWS * VOCAB:
            case["rows"] = max(1, MAX_ROWS * VOCAB // case["stride"])
        return case
    rows = _log_int(rng, 1, TREE)
    case = {"kind": kind, "rows": rows, "deep": _log_int(rng, 1, rows)}
    q_heads, kv_heads = rng.choice(HEADS)
    span = min(MAX_CONTEXT, 8 * MAX_CONTEXT // q_heads, 2 * MAX_CONTEXT // kv_heads)  # the largest listed case costs most
    case["position"] = rng.choice([rng.randrange(span - TREE + 1), _log_int(rng, 1, span - TREE + 1) - 1])
    if kind == "attn":
        case["q_heads"] = q_heads
    if kind in ("attn", "kv_keep"):
        case["kv_heads"] = kv_heads
    return case


# ----------------------------------------------------------------- inputs
class Draws:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def floats(self, *shape, mean=0.0, std=1.0):
        return torch.empty(*shape, device="cuda").normal_(mean, std, generator=self.g)

    def normal(self, *shape, mean=0.0, std=1.0):
        return self.floats(*shape, mean=mean, std=std).to(torch.bfloat16)

    def keys(self, *shape):
        """Rows of unit variance on the whole with channels of unequal size."""
        size = self.floats(shape[-1], std=0.4).exp_()
        return self.floats(*shape).mul_(size * size.square().mean().rsqrt()).to(torch.bfloat16)

    def uniform(self, *shape, lo, hi):
        return torch.empty(*shape, device="cuda").uniform_(lo, hi, generator=self.g)


def _tree(case, seed):
    """Path words of a tree of `rows` nodes with a path of `deep` nodes, and that path's last node."""
    rng, rows = random.Random(seed), case["rows"]
    main = [0] + sorted(rng.sample(range(1, rows), case["deep"] - 1))
    paths = []
    for i in range(rows):
        up = main[main.index(i) - 1] if i in main[1:] else rng.randrange(-1, i) if i else -1
        paths.append(1 << i | (paths[up] if up >= 0 else 0))
    return paths, main[-1]


def _rope_freq():
    i = torch.arange(ROTARY // 2, device="cuda", dtype=torch.float64)
    return (10000000.0 ** (-i / (ROTARY // 2))).float()


def prepare(case, seed):
    d, kind, m = Draws(seed), case["kind"], case["rows"]
    if kind == "logprob":
        return _prepare_logprob(case, d)
    paths, node = _tree(case, seed)
    s = {"case": case, "node": node, "paths": torch.tensor([p - (p >> 63 << 64) for p in paths], device="cuda")}
    n = case["position"]
    if kind in ("attn", "kv_keep"):
        hk = case["kv_heads"]
        s["capacity"] = n + TREE
        s["v_proj"] = d.normal(m, hk, DIM)
        if kind == "kv_keep":
            s["k_tree"] = d.keys(m, hk, DIM)
            s["k_cache"], s["v_cache"] = (d.normal(hk, n + TREE, DIM) for _ in range(2))
            return s
        s["k_cache"], s["v_cache"] = d.keys(hk, n + TREE, DIM), d.normal(hk, n + TREE, DIM)
        s["q_proj"], s["k_proj"] = d.normal(m, case["q_heads"], 2 * DIM), d.keys(m, hk, DIM)
        s["q_gain"], s["k_gain"] = d.normal(DIM, mean=1.0, std=0.1), d.normal(DIM, mean=1.0, std=0.1)
        s["inv_freq"] = _rope_freq()
        return s
    s["raw"], s["ring"] = d.normal(m, CONV), d.normal(4, CONV)
    s["state"] = d.floats(GDN_HEADS, GDN_DIM, GDN_DIM, std=0.1)
    a_log = d.uniform(GDN_HEADS, lo=0.5, hi=2.0).log()
    if kind == "gdn":
        s["conv_w"], s["a_log"] = d.normal(CONV, 4, std=0.5), a_log
        s["dt_bias"] = d.normal(GDN_HEADS, mean=-1.0, std=0.5)
        s["a_proj"], s["b_proj"] = d.normal(m, GDN_HEADS), d.normal(m, GDN_HEADS)
        return s
    s["keys"] = torch.nn.functional.normalize(d.floats(m, GDN_HEADS, GDN_DIM), dim=-1)
    s["updates"] = d.floats(m, GDN_HEADS, GDN_DIM, std=0.3)
    s["log_decay"] = -a_log.exp() * torch.log1p(d.floats(m, GDN_HEADS, mean=-1.0, std=1.1).exp())
    return s


def _prepare_logprob(case, d):
    m, vocab = case["rows"], case["vocab"]
    shape = (m, case["stride"])
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, 2.0, generator=d.g)
    peaks = torch.empty(shape, dtype=torch.bool, device="cuda").bernoulli_(min(0.1, 40 / vocab), generator=d.g)
    x += peaks * torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(9.0, 3.0, generator=d.g)
    if case["masked"]:  # most of the vocabulary excluded, another part in each row
        x.masked_fill_(peaks.bernoulli_(0.9, generator=d.g), -math.inf)
    tokens = (d.uniform(m, lo=0, hi=1).double() * vocab).long().clamp_(max=vocab - 1)
    x.scatter_(1, tokens[:, None], d.normal(m, 1, mean=9.0, std=3.0))
    tokens = tokens.to(torch.int32)
    return {"case": case, "logits": x, "tokens": tokens}


# ------------------------------------------------------------- plain form
def _bits(s):
    """[rows, rows]: whether the node of the column is on the row's path."""
    return (s["paths"][:, None] >> torch.arange(s["case"]["rows"], device="cuda") & 1).bool()


def _rotated(x, gain, place, inv_freq):
    """RMS norm and rotation of x [rows, heads, DIM] in 32 bits at positions `place`, their angles in 64."""
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain.float()
    angle = place.double()[:, None, None] * inv_freq.double()
    cos, sin, half = angle.cos().float(), angle.sin().float(), ROTARY // 2
    a, b = x[..., :half], x[..., half:ROTARY]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROTARY:]], -1).to(torch.bfloat16)


def _run_attn(s):
    case, bits = s["case"], _bits(s)
    m, n, hk = case["rows"], case["position"], case["kv_heads"]
    place = n + bits.sum(1) - 1
    q = _rotated(s["q_proj"][..., :DIM], s["q_gain"], place, s["inv_freq"])
    k = _rotated(s["k_proj"], s["k_gain"], place, s["inv_freq"])
    keys = torch.cat([s["k_cache"][:, :n], k.transpose(0, 1)], 1).float()
    values = torch.cat([s["v_cache"][:, :n], s["v_proj"].transpose(0, 1)], 1).float()
    q = q.float().view(m, hk, -1, DIM).transpose(0, 1)  # [kv heads, rows, group, DIM]
    x = (q.reshape(hk, -1, DIM) @ keys.transpose(1, 2)).view(hk, m, -1, n + m) / 16
    x[..., n:].masked_fill_(~bits[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = (x.view(hk, -1, n + m) @ values).view(q.shape) / x.sum(-1, keepdim=True)
    o = o.transpose(0, 1).reshape(m, case["q_heads"], DIM) / (1 + torch.exp(-s["q_proj"][..., DIM:].float()))
    return [o.to(torch.bfloat16), k]


def _path_rows(s):
    """[rows, 4] rows of raw behind the ring's four, of each node's last four positions, oldest first."""
    bits, n = _bits(s), s["case"]["position"]
    after = bits.flip(1).cumsum(1).flip(1)  # how many of the path from the column's node on
    depth = bits.sum(1) - 1
    back = torch.arange(3, -1, -1, device="cuda")
    at = (bits[:, None] & (after[:, None] == back[:, None] + 1)).int().argmax(-1)  # the ancestor `back` steps up
    return torch.where(back <= depth[:, None], 4 + at, (n + depth[:, None] - back) & 3)


def _run_gdn(s):
    bits, m = _bits(s), s["case"]["rows"]
    rows = torch.cat([s["ring"], s["raw"]]).float()[_path_rows(s)]  # [rows, 4, CONV]
    x = (rows * s["conv_w"].float().T).sum(1)
    q, k, v = (x / (1 + torch.exp(-x))).view(m, 3, GDN_HEADS, GDN_DIM).permute(1, 2, 0, 3)
    q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + 1e-6) * GDN_DIM ** -0.5
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + 1e-6)
    gate = s["a_proj"].float() + s["dt_bias"].float()
    log_g = -s["a_log"].exp() * (gate.clamp(min=0) + torch.log1p(torch.exp(-gate.abs())))  # [rows, heads]
    beta = (1 / (1 + torch.exp(-s["b_proj"].float()))).T[..., None]
    total = (bits.double() @ log_g.double()).T  # along each path, [heads, rows]
    between = torch.exp((total[:, :, None] - total[:, None, :]).masked_fill(~bits, -math.inf)).float()
    decay, state = total.exp().float()[..., None], s["state"].transpose(1, 2)
    # (1 + L) u = b with L strictly lower triangular: its inverse is (1 - L)(1 + L^2)(1 + L^4) ...
    one = torch.eye(m, device="cuda")
    low = beta * (k @ k.transpose(1, 2)) * between * (1 - one)
    inverse, power = one - low, low
    for _ in range(5):
        power = power @ power
        inverse = inverse @ (one + power)
    u = inverse @ (beta * (v - decay * (k @ state)))
    y = decay * (q @ state) + (q @ k.transpose(1, 2) * between) @ u
    y, k, u = (t.transpose(0, 1).contiguous() for t in (y, k, u))
    return [y.reshape(m, -1).to(torch.bfloat16), k, u, log_g]


def _path_of(s):
    """The nodes on the accepted path, in order."""
    return _bits(s)[s["node"]].nonzero()[:, 0]


def _run_gdn_keep(s):
    at, n = _path_of(s), s["case"]["position"]
    log_g = s["log_decay"][at].double()
    after = log_g.flip(0).cumsum(0).flip(0)  # [path, heads], a node's own gate and those behind it
    weight = (after - log_g).exp().float()[..., None]
    state = s["state"] * after[0].exp().float()[:, None, None]
    state = state + (s["updates"][at] * weight).permute(1, 2, 0) @ s["keys"][at].transpose(0, 1)
    slot = torch.arange(n, n + at.numel(), device="cuda")[-4:] & 3
    ring = s["ring"].clone()
    ring[slot] = s["raw"][at[-4:]]
    return [state, ring]


def _run_kv_keep(s):
    at, n = _path_of(s), s["case"]["position"]
    out = []
    for cache, rows in ((s["k_cache"], s["k_tree"]), (s["v_cache"], s["v_proj"])):
        cache[:, n:n + at.numel()] = rows[at].transpose(0, 1)
        out.append(cache[:, n:n + s["case"]["deep"]])
    return out


def _run_logprob(s):
    case = s["case"]
    x = s["logits"][:, :case["vocab"]].float()
    largest = x.amax(1, keepdim=True)
    d = x - largest
    e = torch.exp(d)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = total.log()
    entropy = log_total - (e * d.clamp(min=-1e30)).sum(1, keepdim=True, dtype=torch.float64) / total
    given = d.gather(1, s["tokens"].long()[:, None]) - log_total
    out = [given[:, 0].float(), entropy[:, 0].float(), (largest + log_total)[:, 0].float()]
    if case["top"]:
        # by value, then by index: both in one whole number
        order = (x + 0).view(torch.int32)
        order = (order ^ (order >> 31 & 0x7fffffff)).long() << 32
        ids = (order - torch.arange(case["vocab"], device="cuda")).topk(case["top"], 1).indices
        out += [ids.int(), (d.gather(1, ids) - log_total).float()]
    return out


# -------------------------------------------------------- framework's form
def _esdecode():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "enginesmith-qwen35-08b-long-decode-m5max-round005_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import esdecode
    return esdecode


def _buffer(s, name, *shape, dtype=torch.float32):
    """An output or workspace that a program keeps from call to call."""
    if name not in s:
        s[name] = torch.empty(*shape, dtype=dtype, device="cuda")
    return s[name]


def _call(E, name, *args):
    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    E.check(getattr(E.lib(), name)(*args, torch.cuda.current_stream().cuda_stream))


def _own_attn(s):
    E, case = _esdecode(), s["case"]
    m, hq, hk = case["rows"], case["q_heads"], case["kv_heads"]
    size = int(E.lib().es_attn_tree_scratch_bytes(hq, hk, m))
    scratch = _buffer(s, "scratch", size, dtype=torch.uint8)
    out, k_tree = _buffer(s, "out", m, hq, DIM, dtype=torch.bfloat16), _buffer(s, "k_tree", m, hk, DIM,
                                                                              dtype=torch.bfloat16)
    _call(E, "es_attn_tree", s["q_proj"], s["k_proj"], s["v_proj"], s["q_gain"], s["k_gain"], s["inv_freq"],
          s["paths"], m, hq, hk, s["k_cache"], s["v_cache"], s["capacity"], case["position"], scratch, size, k_tree,
          out)
    return [out, k_tree]


def _own_gdn(s):
    E, m = _esdecode(), s["case"]["rows"]
    y = _buffer(s, "y", m, GDN_HEADS * GDN_DIM, dtype=torch.bfloat16)
    k, u = (_buffer(s, name, m, GDN_HEADS, GDN_DIM) for name in ("keys", "updates"))
    log_g = _buffer(s, "log_decay", m, GDN_HEADS)
    _call(E, "es_gdn_tree", s["raw"], s["ring"], s["conv_w"], s["a_proj"], s["b_proj"], s["a_log"], s["dt_bias"],
          s["paths"], s["case"]["position"], m, s["state"], y, k, u, log_g)
    return [y, k, u, log_g]


def _own_gdn_keep(s):
    E, case = _esdecode(), s["case"]
    out = _buffer(s, "state_out", *s["state"].shape)
    _call(E, "es_gdn_tree_keep", s["raw"], s["keys"], s["updates"], s["log_decay"], s["paths"], s["node"],
          case["rows"], case["position"], s["ring"], s["state"], out)
    return [out, s["ring"]]


def _own_kv_keep(s):
    E, case = _esdecode(), s["case"]
    _call(E, "es_kv_tree_keep", s["k_tree"], s["v_proj"], s["paths"], s["node"], case["rows"], case["kv_heads"],
          s["k_cache"], s["v_cache"], s["capacity"], case["position"])
    n = case["position"]
    return [s[name][:, n:n + case["deep"]] for name in ("k_cache", "v_cache")]


def _own_logprob(s):
    E, case = _esdecode(), s["case"]
    m, top = case["rows"], case["top"]
    size = int(E.lib().es_logprob_scratch_bytes(m, case["vocab"], top))
    scratch = _buffer(s, "scratch", size, dtype=torch.uint8)
    given, entropy, lse = (_buffer(s, name, m) for name in ("given", "entropy", "lse"))
    ids, alternatives = _buffer(s, "ids", m, top, dtype=torch.int32), _buffer(s, "alternatives", m, top)
    _call(E, "es_logprob_rows", s["logits"], case["stride"], m, case["vocab"], s["tokens"], top, scratch, size, given,
          entropy, lse, ids if top else None, alternatives if top else None)
    return [given, entropy, lse] + ([ids, alternatives] if top else [])


_RUN = {"attn": (_run_attn, _own_attn), "gdn": (_run_gdn, _own_gdn), "gdn_keep": (_run_gdn_keep, _own_gdn_keep),
        "kv_keep": (_run_kv_keep, _own_kv_keep), "logprob": (_run_logprob, _own_logprob)}


def run(state):
    return _RUN[state["case"]["kind"]][1 if own else 0](state)


# ------------------------------------------------------------------- work
def work(case):
    kind, m = case["kind"], case["rows"]
    if kind == "logprob":
        return {"bytes": m * (2 * case["vocab"] + 16 + 8 * case["top"]), "flops": 6 * m * case["vocab"]}
    if kind == "attn":
        n, hq, hk = case["position"], case["q_heads"], case["kv_heads"]
        return {"bytes": 4 * n * hk * DIM + m * DIM * (6 * hq + 6 * hk), "flops": 4 * hq * DIM * m * (n + case["deep"])}
    if kind == "kv_keep":
        return {"bytes": 8 * case["deep"] * case["kv_heads"] * DIM, "flops": 0}
    head = GDN_HEADS * GDN_DIM
    if kind == "gdn":
        return {"bytes": 2 * (m + 7) * CONV + 4 * head * GDN_DIM + m * head * (2 + 8) + 8 * m * GDN_HEADS,
                "flops": 8 * m * CONV + 4 * m * head * (GDN_DIM + m)}
    return {"bytes": 8 * head * GDN_DIM + 8 * case["deep"] * head + 4 * min(4, case["deep"]) * CONV,
            "flops": 2 * (case["deep"] + 1) * head * GDN_DIM}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprob":
        return _exact_logprob(case, s)
    paths, node = _tree(case, seed)
    nodes = [[j for j in range(case["rows"]) if p >> j & 1] for p in paths]
    n = case["position"]
    if case["kind"] == "kv_keep":
        return [s[name][nodes[node]].transpose(0, 1).double() for name in ("k_tree", "v_proj")]
    if case["kind"] == "attn":
        return _exact_attn(case, s, nodes)
    if case["kind"] == "gdn":
        return _exact_gdn(case, s, nodes)
    state, ring = s["state"].double(), s["ring"].double()
    for t, j in enumerate(nodes[node]):
        u, k = s["updates"][j].double(), s["keys"][j].double()
        state = torch.exp(s["log_decay"][j].double())[:, None, None] * state + u[:, :, None] * k[:, None, :]
        ring[(n + t) % 4] = s["raw"][j].double()
    return [state, ring]


def _exact_rotation(x, gain, place, inv_freq):
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / DIM + 1e-6) * gain.double()
    z = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device), place[:, None, None] * inv_freq.double())
    pair = torch.complex(y[..., :ROTARY // 2], y[..., ROTARY // 2:ROTARY]) * z
    return torch.cat([pair.real, pair.imag, y[..., ROTARY:]], -1)


def _exact_attn(case, s, nodes):
    n, m, hq = case["position"], case["rows"], case["q_heads"]
    place = torch.tensor([n + len(p) - 1.0 for p in nodes], dtype=torch.float64, device="cuda")
    q = _exact_rotation(s["q_proj"][..., :DIM].double(), s["q_gain"], place, s["inv_freq"])
    k = _exact_rotation(s["k_proj"].double(), s["k_gain"], place, s["inv_freq"])
    out = torch.empty(m, hq, DIM, dtype=torch.float64, device="cuda")
    seen = torch.full((m, m), -math.inf, dtype=torch.float64, device="cuda")
    for i, p in enumerate(nodes):
        seen[i, p] = 0
    for h in range(hq):
        g = h // (hq // case["kv_heads"])
        keys = torch.cat([s["k_cache"][g, :n].double(), k[:, g]])
        x = q[:, h] @ keys.T / math.sqrt(DIM)
        x[:, n:] += seen
        out[:, h] = torch.softmax(x, -1) @ torch.cat([s["v_cache"][g, :n], s["v_proj"][:, g]]).double()
    return [out * torch.sigmoid(s["q_proj"][..., DIM:].double()), k]


def _exact_gdn(case, s, nodes):
    n, m = case["position"], case["rows"]
    raw, ring, w = s["raw"].double(), s["ring"].double(), s["conv_w"].double()
    log_g = -s["a_log"].double().exp() * torch.nn.functional.softplus(s["a_proj"].double() + s["dt_bias"].double())
    beta = torch.sigmoid(s["b_proj"].double())
    states, outs = {}, []
    for i, p in enumerate(nodes):
        last = [ring[(n + len(p) - 1 - b) % 4] if b >= len(p) else raw[p[-1 - b]] for b in (3, 2, 1, 0)]
        x = torch.nn.functional.silu(sum(last[t] * w[:, t] for t in range(4))).view(3, GDN_HEADS, GDN_DIM)
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in x[:2])
        state = (states[p[-2]] if len(p) > 1 else s["state"].double()) * log_g[i].exp()[:, None, None]
        u = beta[i][:, None] * (x[2] - (state * k[:, None]).sum(-1))
        states[i] = state + u[:, :, None] * k[:, None]
        outs.append(((states[i] * q[:, None]).sum(-1).reshape(-1) / math.sqrt(GDN_DIM), k, u))
    return [torch.stack(t) for t in zip(*outs)] + [log_g]


def _exact_logprob(case, s):
    given, entropy, lse, top = [], [], [], []
    for x, tokens in zip(s["logits"][:, :case["vocab"]].split(64), s["tokens"].split(64)):
        x = x.double()
        log_p = torch.log_softmax(x, -1)
        p = log_p.exp()
        given.append(log_p.gather(1, tokens.long()[:, None])[:, 0])
        entropy.append(-torch.where(p > 0, p * log_p, 0.0).sum(1))
        lse.append(torch.logsumexp(x, 1))
        top.append(log_p.topk(case["top"], 1).values)
    out = [torch.cat(v) for v in (given, entropy, lse)]
    return out + [None, torch.cat(top)] if case["top"] else out
