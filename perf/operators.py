"""Performance cases of the key/value cache in 8 bits: writing and reading it,
preparing projected rows into it, and attention over it, through the C ABI of
include/es_decode.h (the esdecode binding), beside the same operators in their
plain form.

The cache holds e4m3 codes with one power of two for each block of 64 tokens of
a head, keys and values apart: the smallest that brings the block's largest
magnitude to at most 448. Rows from `position` on are written; the block that
holds `position` keeps its earlier rows and only ever raises its power of two.

Inputs are random with the distributions the model has: K rows of unit variance
(they are RMS-normalised) with channels of unequal size, V rows of unit
variance, attention scores of unit variance, gains N(1, 0.1).
"""
import math
import os
import sys

import torch

own = False

DIM, BLOCK, ROTARY, LARGEST = 256, 64, 64, 448.0
MAX_ROWS, MAX_CONTEXT = 4096, 131072
MAX_PAIRS = 8 * 4096 * 32768          # rows x query heads x context of the largest prompt chunk
HEADS = [(8, 2), (8, 2), (8, 2), (16, 4), (32, 8), (12, 3), (8, 1), (5, 5), (28, 4)]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one generated token's K and V into a context of 40001, and its block read back: the smallest call
        {"name": "write_1", "kind": "write", "kv_heads": 2, "position": 40001, "rows": 1, "token_major": True},
        # a full prompt chunk's projected K and V
        {"name": "write_4096", "kind": "write", "kv_heads": 2, "position": 8192, "rows": 4096, "token_major": True},
        # a whole bf16 cache of the longest benchmarked context converted at once
        {"name": "write_131072", "kind": "write", "kv_heads": 2, "position": 0, "rows": 131072, "token_major": False},
        # part of a context handed to a program that keeps bf16
        {"name": "read_50003", "kind": "read", "kv_heads": 2, "position": 1027, "rows": 50003},
        # one generated token at the end of the longest context: norm, rotation, append
        {"name": "prepare_1_at_131071", "kind": "prepare", "q_heads": 8, "kv_heads": 2, "position": 131071, "rows": 1},
        # the last chunk of a 32K prompt: norm, rotation, write
        {"name": "prepare_4096_at_28672", "kind": "prepare", "q_heads": 8, "kv_heads": 2, "position": 28672,
         "rows": 4096},
        # one generated token over a short context, with the output gate: bound by latency
        {"name": "attn_1_at_1020", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 1020, "rows": 1,
         "gate": True},
        # one generated token over the longest benchmarked context, with the output gate
        {"name": "attn_1_at_131071", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 131071, "rows": 1,
         "gate": True},
        # one generated token of a model with more heads
        {"name": "attn_1_at_20010_of_32_heads", "kind": "attn", "q_heads": 32, "kv_heads": 8, "position": 20010,
         "rows": 1, "gate": False},
        # several tokens checked at once at the end of a long context
        {"name": "attn_5_at_70000", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 70000, "rows": 5,
         "gate": True},
        # the first, ragged chunk of a medium prompt
        {"name": "attn_1000_at_0", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 0, "rows": 1000,
         "gate": False},
        # the last chunk of a 32K prompt
        {"name": "attn_4096_at_28672", "kind": "attn", "q_heads": 8, "kv_heads": 2, "position": 28672, "rows": 4096,
         "gate": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "prepare", "step", "step", "rows", "chunk", "chunk"])
    q_heads, kv_heads = rng.choice(HEADS)
    span = 2 * MAX_CONTEXT // kv_heads  # tokens of the largest cache with this many heads
    span = min(span, MAX_CONTEXT)
    case = {"kind": kind, "kv_heads": kv_heads}
    if kind in ("write", "read"):
        case["rows"] = _log_int(rng, 1, span // 2)
        case["position"] = rng.choice([0, rng.randrange(span - case["rows"] + 1)])
        if kind == "write":
            case["token_major"] = rng.random() < 0.5
        return case
    case["q_heads"] = q_heads
    if kind == "prepare":
        case["rows"] = _log_int(rng, 1, max(1, MAX_ROWS * 8 // max(8, q_heads)))
        case["position"] = rng.choice([0, rng.randrange(span - case["rows"] + 1)])
        return case
    case["kind"], case["gate"] = "attn", rng.random() < 0.5
    if kind == "step":
        case["rows"], case["position"] = 1, _log_int(rng, 1, span) - 1
    elif kind == "rows":
        case["rows"] = rng.randrange(2, 33)
        case["position"] = _log_int(rng, 1, span - case["rows"]) - 1
    else:
        case["rows"] = _log_int(rng, 33, MAX_ROWS * 8 // max(8, q_heads))
        most = min(span, MAX_PAIRS // (case["rows"] * q_heads)) - case["rows"]
        case["position"] = rng.choice([0, rng.randrange(most + 1)])
    return case


# ----------------------------------------------------------------- inputs
class Draws:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, mean=0.0, std=1.0):
        return torch.empty(*shape, device="cuda").normal_(mean, std, generator=self.g).to(torch.bfloat16)

    def keys(self, tokens, heads):
        """[tokens, heads, DIM] rows with channels of unequal size, unit variance on the whole."""
        size = torch.empty(DIM, device="cuda").normal_(0.0, 0.4, generator=self.g).exp_()
        x = torch.empty(tokens, heads, DIM, device="cuda").normal_(generator=self.g)
        return x.mul_(size * size.square().mean().rsqrt()).to(torch.bfloat16)


def _inputs(case, seed):
    """The bf16 tensors of a case; "held" K and V are what the cache has before the call."""
    d, kind, n = Draws(seed), case["kind"], case["position"] + case["rows"]
    m, hk = case["rows"], case["kv_heads"]
    if kind == "attn":
        hq = case["q_heads"]
        return {"held_k": d.keys(n, hk), "held_v": d.normal(n, hk, DIM), "query": d.normal(m, hq, DIM),
                "q_proj": d.normal(m, hq, 2 * DIM) if case["gate"] else None}
    if kind == "read":
        return {"held_k": d.keys(n, hk), "held_v": d.normal(n, hk, DIM)}
    first = case["position"] // BLOCK * BLOCK  # only the block of `position` holds rows that the call meets
    s = {"held_k": d.keys(case["position"] - first, hk), "held_v": d.normal(case["position"] - first, hk, DIM)}
    if kind == "write":
        k, v = d.keys(m, hk), d.normal(m, hk, DIM)
        if not case["token_major"]:
            k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
        return {**s, "k": k, "v": v}
    freq = 10000000.0 ** (-torch.arange(ROTARY // 2, device="cuda", dtype=torch.float64) / (ROTARY // 2))
    return {**s, "q_proj": d.normal(m, case["q_heads"], 2 * DIM), "k_proj": d.keys(m, hk),
            "v_proj": d.normal(m, hk, DIM), "q_gain": d.normal(DIM, mean=1.0, std=0.1),
            "k_gain": d.normal(DIM, mean=1.0, std=0.1), "inv_freq": freq.float()}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    n, hk = case["position"] + case["rows"], case["kv_heads"]
    held_k, held_v = s.pop("held_k"), s.pop("held_v")
    start = n - held_k.shape[0] if case["kind"] in ("attn", "read") else case["position"] - held_k.shape[0]
    if own:
        return _prepare_own(s, n, start, held_k, held_v)
    blocks = -(-n // BLOCK)
    for name in ("k", "v"):
        s[name + "_codes"] = torch.zeros(hk, blocks * BLOCK, DIM, device="cuda").to(torch.float8_e4m3fn)
        s[name + "_exp"] = torch.full((hk, blocks), -127, dtype=torch.int32, device="cuda")
    if held_k.shape[0]:
        _write_plain(s, held_k, held_v, start)
    return s


# ------------------------------------------------------------- plain form
def _exponent(largest):
    """Smallest e with largest * 2^-e <= LARGEST, by exact steps."""
    half, e = torch.frexp(largest)  # half in [0.5, 1)
    return torch.where(largest > 0, e - 8 - (half <= 0.875).int(), -127).clamp_(-127, 127)


def _e4m3(x, e):
    return torch.ldexp(x, -e).to(torch.float8_e4m3fn)


def _write_plain(s, k, v, position):
    first = position // BLOCK
    keep, m = position - first * BLOCK, k.shape[0]
    blocks = -(-(keep + m) // BLOCK)
    for name, rows in (("k", k), ("v", v)):
        codes, exps = s[name + "_codes"], s[name + "_exp"]
        heads = codes.shape[0]
        x = torch.zeros(heads, blocks * BLOCK, DIM, device="cuda")
        x[:, keep:keep + m] = rows.transpose(0, 1)
        e = _exponent(x.view(heads, blocks, -1).abs().amax(-1))
        if keep:
            before = exps[:, first]
            e[:, 0] = torch.maximum(e[:, 0], before)
            held = codes[:, first * BLOCK:position]
            shift = (before - e[:, 0])[:, None, None]
            held.copy_(_e4m3(held.float(), -shift))
        new = _e4m3(x, e.repeat_interleave(BLOCK, 1)[:, :, None])
        codes[:, position:position + m] = new[:, keep:keep + m]
        exps[:, first:first + blocks] = e


def _held_plain(s, name, start, end):
    """[heads, end - start, DIM] values of the cache in 32 bits."""
    exps = s[name + "_exp"].repeat_interleave(BLOCK, 1)[:, start:end, None]
    return torch.ldexp(s[name + "_codes"][:, start:end].float(), exps)


def _read_plain(s, start, end):
    return [_held_plain(s, name, start, end).transpose(0, 1).to(torch.bfloat16) for name in ("k", "v")]


def _rotated_plain(x, gain, position, inv_freq):
    """RMS norm and rotation of x [rows, heads, DIM] in 32 bits, its angles in 64."""
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain.float()
    angle = (position + torch.arange(x.shape[0], device="cuda")).double()[:, None, None] * inv_freq.double()
    cos, sin, half = angle.cos().float(), angle.sin().float(), ROTARY // 2
    a, b = x[..., :half], x[..., half:ROTARY]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROTARY:]], -1)


def _run_write(s):
    case = s["case"]
    _write_plain(s, s["k"], s["v"], case["position"])
    return _read_plain(s, case["position"] // BLOCK * BLOCK, case["position"] + case["rows"])


def _run_read(s):
    return _read_plain(s, s["case"]["position"], s["case"]["position"] + s["case"]["rows"])


def _run_prepare(s):
    case = s["case"]
    q = _rotated_plain(s["q_proj"][..., :DIM], s["q_gain"], case["position"], s["inv_freq"])
    k = _rotated_plain(s["k_proj"], s["k_gain"], case["position"], s["inv_freq"])
    _write_plain(s, k, s["v_proj"], case["position"])
    return [q.to(torch.bfloat16),
            *_read_plain(s, case["position"] // BLOCK * BLOCK, case["position"] + case["rows"])]


def _run_attn(s):
    case, query = s["case"], s["query"]
    m, hq, _ = query.shape
    n, group = case["position"] + m, hq // case["kv_heads"]
    keys, values = _held_plain(s, "k", 0, n), _held_plain(s, "v", 0, n)
    out = torch.empty(m, hq, DIM, dtype=torch.bfloat16, device="cuda")
    cols = torch.arange(n, device="cuda")
    step = max(1, (1 << 28) // (n * group))
    for r in range(0, m, step):
        last = case["position"] + torch.arange(r, min(m, r + step), device="cuda")
        for h in range(case["kv_heads"]):
            q = query[r:r + step, h * group:(h + 1) * group].float()
            x = (q.reshape(-1, DIM) @ keys[h].T / 16).view(q.shape[0], group, n)
            x.masked_fill_((cols > last[:, None])[:, None], -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            x /= x.sum(-1, keepdim=True)
            o = (x.view(-1, n) @ values[h]).view(q.shape)
            if s["q_proj"] is not None:
                gate = s["q_proj"][r:r + step, h * group:(h + 1) * group, DIM:].float()
                o = o / (1 + torch.exp(-gate))
            out[r:r + step, h * group:(h + 1) * group] = o
    return [out]


# -------------------------------------------------------- framework's form
def _esdecode():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "enginesmith-qwen35-08b-long-decode-m5max-round005_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import esdecode
    return esdecode


def _ptr(t):
    return None if t is None else t.data_ptr()


def _prepare_own(s, n, start, held_k, held_v):
    E, case = _esdecode(), s["case"]
    hk, m, blocks = case["kv_heads"], case["rows"], -(-n // BLOCK)
    first = case["position"] // BLOCK * BLOCK

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    s["memory"] = [empty(hk * blocks * BLOCK * DIM, dtype=torch.uint8) for _ in range(2)] + \
                  [empty(hk * blocks, dtype=torch.uint8) for _ in range(2)]
    s["cache"] = E.KV8(*(t.data_ptr() for t in s["memory"]), hk, n)
    if held_k.shape[0]:
        E.check(E.lib().es_kv8_write(s["cache"], _ptr(held_k), _ptr(held_v), held_k.stride(0), held_k.stride(1), start,
                                     held_k.shape[0], None))
    if case["kind"] == "attn":
        size = int(E.lib().es_attn_kv8_scratch_bytes(case["q_heads"], hk, m))
        s["scratch"], s["out"] = empty(size, dtype=torch.uint8), empty(m, case["q_heads"], DIM)
    else:
        read = m if case["kind"] == "read" else n - first
        s["k_out"], s["v_out"] = empty(read, hk, DIM), empty(read, hk, DIM)
    if case["kind"] == "prepare":
        s["query"] = empty(m, case["q_heads"], DIM)
    return s


def _own_read(E, s, start, end):
    E.check(E.lib().es_kv8_read(s["cache"], start, end - start, _ptr(s["k_out"]), _ptr(s["v_out"]),
                                s["k_out"].stride(0), s["k_out"].stride(1), None))
    return [s["k_out"], s["v_out"]]


def _own_write(s):
    E, case = _esdecode(), s["case"]
    E.check(E.lib().es_kv8_write(s["cache"], _ptr(s["k"]), _ptr(s["v"]), s["k"].stride(0), s["k"].stride(1),
                                 case["position"], case["rows"], None))
    return _own_read(E, s, case["position"] // BLOCK * BLOCK, case["position"] + case["rows"])


def _own_read_rows(s):
    return _own_read(_esdecode(), s, s["case"]["position"], s["case"]["position"] + s["case"]["rows"])


def _own_prepare(s):
    E, case, p = _esdecode(), s["case"], _ptr
    E.check(E.lib().es_attn_prepare_rows_kv8(p(s["q_proj"]), p(s["k_proj"]), p(s["v_proj"]), p(s["q_gain"]),
                                             p(s["k_gain"]), p(s["inv_freq"]), case["position"], case["rows"],
                                             case["q_heads"], p(s["query"]), s["cache"], None))
    return [s["query"], *_own_read(E, s, case["position"] // BLOCK * BLOCK, case["position"] + case["rows"])]


def _own_attn(s):
    E, case = _esdecode(), s["case"]
    E.check(E.lib().es_attn_kv8(_ptr(s["query"]), case["q_heads"], s["cache"], case["position"], case["rows"],
                                _ptr(s["q_proj"]), _ptr(s["scratch"]), s["scratch"].numel(), _ptr(s["out"]), None))
    return [s["out"]]


_RUN = {"write": (_run_write, _own_write), "read": (_run_read, _own_read_rows),
        "prepare": (_run_prepare, _own_prepare), "attn": (_run_attn, _own_attn)}


def run(state):
    return _RUN[state["case"]["kind"]][1 if own else 0](state)


# ------------------------------------------------------------------- work
def work(case):
    m, hk = case["rows"], case["kv_heads"]
    n = case["position"] + m
    row = 2 * hk * DIM  # elements of a token's K and V
    if case["kind"] == "read":
        return {"bytes": m * row * 3, "flops": m * row}
    if case["kind"] in ("write", "prepare"):
        back = n - case["position"] // BLOCK * BLOCK
        made = 0 if case["kind"] == "write" else 2 * m * case["q_heads"] * DIM
        return {"bytes": m * row * 3 + back * row * 3 + 2 * made, "flops": 2 * m * row + back * row + 8 * made}
    hq = case["q_heads"]
    pairs = m * case["position"] + m * (m + 1) // 2
    return {"bytes": n * row + m * hq * DIM * (6 if case["gate"] else 4), "flops": 4 * hq * DIM * pairs}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = _inputs(case, seed)
    pos, m = case["position"], case["rows"]
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    if case["kind"] == "read":
        return [_exact_codes(s[name], 0)[pos:pos + m] for name in ("held_k", "held_v")]
    if case["kind"] == "write":
        return [_exact_append(s["held_" + name], s[name].double()) for name in ("k", "v")]
    q = _exact_rotation(s["q_proj"].double()[:, :, :DIM], s["q_gain"], pos, s["inv_freq"])
    k = _exact_rotation(s["k_proj"].double(), s["k_gain"], pos, s["inv_freq"])
    return [q, _exact_append(s["held_k"], k), _exact_append(s["held_v"], s["v_proj"].double())]


def _exact_power(x):
    """log2 of the power of two of x [blocks, heads, rows * DIM]'s codes."""
    top = x.abs().amax(-1)
    e = torch.floor(torch.log2(top)) - 8
    e = torch.where(torch.exp2(e) * LARGEST < top, e + 1, e)
    return torch.where(top > 0, e, -127.0).clamp(-127, 127)


def _exact_round(y):
    """y to the nearest number of four significant bits, steps of at least 2^-9, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_codes(x, skip):
    """Values of x [tokens, heads, DIM] in the cache, its first token `skip` tokens into a block."""
    tokens, heads, _ = x.shape
    pad = torch.zeros(-(-(skip + tokens) // BLOCK) * BLOCK, heads, DIM, dtype=torch.float64, device=x.device)
    pad[skip:skip + tokens] = x
    y = pad.view(-1, BLOCK, heads, DIM).transpose(1, 2).reshape(-1, heads, BLOCK * DIM)
    power = torch.exp2(_exact_power(y))[:, :, None]
    y = (_exact_round(y / power) * power).view(-1, heads, BLOCK, DIM).transpose(1, 2)
    return y.reshape(-1, heads, DIM)[skip:skip + tokens]


def _exact_append(held, new):
    """The block of held rows with new ones behind them, and all blocks after it."""
    if held.shape[0] == 0:
        return _exact_codes(new, 0)
    keep = held.shape[0]
    part = new[:BLOCK - keep]
    flat = torch.cat([held.double(), part]).transpose(0, 1).reshape(1, held.shape[1], -1)
    power = torch.exp2(_exact_power(flat))[0, :, None]
    before = _exact_codes(held, 0)
    first = torch.cat([_exact_round(before / power) * power, _exact_round(part / power) * power])
    return torch.cat([first, _exact_codes(new[BLOCK - keep:], 0)]) if new.shape[0] > BLOCK - keep else first


def _exact_rotation(x, gain, position, inv_freq):
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / DIM + 1e-6) * gain.double()
    turn = torch.arange(position, position + x.shape[0], device=x.device, dtype=torch.float64)
    z = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device), turn[:, None, None] * inv_freq.double())
    pair = torch.complex(y[..., :ROTARY // 2], y[..., ROTARY // 2:ROTARY]) * z
    return torch.cat([pair.real, pair.imag, y[..., ROTARY:]], -1)


def _exact_attn(case, s):
    m, hq = case["rows"], case["q_heads"]
    k, v = _exact_codes(s["held_k"], 0), _exact_codes(s["held_v"], 0)
    n, group, out = k.shape[0], hq // case["kv_heads"], torch.empty(m, hq, DIM, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // n)
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        for r in range(0, m, step):
            x = s["query"][r:r + step, h].double() @ kh.T / math.sqrt(DIM)
            row = torch.arange(case["position"] + r, case["position"] + r + x.shape[0], device="cuda")
            x = torch.where(torch.arange(n, device="cuda") <= row[:, None], x, -math.inf)
            out[r:r + step, h] = torch.softmax(x, -1) @ vh
    if s["q_proj"] is not None:
        out = out * torch.sigmoid(s["q_proj"][..., DIM:].double())
    return [out]
