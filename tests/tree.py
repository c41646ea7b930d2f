"""Plain 64-bit models of the operators over a tree of drafted tokens, and of
the scores of logits (torch, double), with how far 32-bit arithmetic may be off."""
import random

import numpy as np
import torch

import esdecode as E

DIM, HEADS, STATE, CONV = 256, 16, 128, 6144
EPS = 2.0 ** -24  # half a step of fp32
BF = 2.0 ** -8    # half a step of bf16
BIG = 1 << 64


def parents_of(kind, rows, seed=0):
    r = random.Random(seed)
    if kind == "chain":
        return [i - 1 for i in range(rows)]
    if kind == "flat":
        return [-1] * rows
    if kind == "wide":
        return [(i - 1) // 3 if i else -1 for i in range(rows)]
    if kind == "holes":  # some nodes left out
        return [-2 if r.random() < 0.2 else r.randrange(-1, i) if i else -1 for i in range(rows)]
    return [r.randrange(max(-1, i - 5), i) if i else -1 for i in range(rows)]


def nodes_of(parents):
    """The nodes on each node's path, itself the last; none for a node left out."""
    out = []
    for i, up in enumerate(parents):
        out.append([] if up == -2 or (up >= 0 and not out[up]) else (out[up] if up >= 0 else []) + [i])
    return out


def words(parents, device="cuda"):
    return torch.from_numpy(E.tree_paths(parents).view(np.int64)).to(device)


def bf(x):
    return x.to(torch.bfloat16)


def call(name, *args, stream=None):
    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    if stream is None:
        stream = torch.cuda.current_stream().cuda_stream
    E.check(getattr(E.lib(), name)(*args, stream))


# --------------------------------------------------------------- attention
def rotated(x, gain, place, inv_freq):
    """x [rows, heads, 256] -> RoPE(RMSNorm(x) * gain) at `place`, in 64 bits."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain.double()
    angle = place.double()[:, None, None] * inv_freq.double()
    cos, sin = angle.cos(), angle.sin()
    a, b = y[..., :32], y[..., 32:64]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 64:]], -1)


def attention(s):
    """gated and k_tree of a case's inputs in 64 bits, and how far gated may be off.

    Queries and keys are bf16 values; where 32 bits round one the other way it is off
    by 2^-7 of itself, so a score by at most d = 2^-7 (the query) or 2^-6 (a node's key too)
    of the sum of its products' magnitudes, 256 roundings of 32 bits beside that. A
    probability's rounding to bf16 is 2^-8 of it, in the sum as in the products. An error d
    of all scores moves an output by at most 2 d times the weighted mean of |v|, the
    roundings by 2 2^-8 of that, sums of 32 bits by the number of keys times 2^-24."""
    n, m, hk = s["position"], s["rows"], s["kv_heads"]
    nodes = s["nodes"]
    dev = s["q_proj"].device
    place = torch.tensor([n + max(0, len(p) - 1) for p in nodes], dtype=torch.float64, device=dev)
    q = rotated(s["q_proj"][..., :DIM], s["q_gain"], place, s["inv_freq"]).to(torch.bfloat16).double()
    k = rotated(s["k_proj"], s["k_gain"], place, s["inv_freq"]).to(torch.bfloat16)
    used = torch.tensor([bool(p) for p in nodes], device=dev)
    k = torch.where(used[:, None, None], k, torch.zeros_like(k))
    out = torch.zeros(m, s["q_heads"], DIM, dtype=torch.float64, device=dev)
    off = torch.zeros_like(out)
    seen = torch.zeros(m, n + m, dtype=torch.bool, device=dev)
    seen[:, :n] = True
    for i, p in enumerate(nodes):
        seen[i, [n + j for j in p]] = True
    group = s["q_heads"] // hk
    for h in range(s["q_heads"]):
        g = h // group
        keys = torch.cat([s["k_cache"][g, :n].double(), k[:, g].double()])
        values = torch.cat([s["v_cache"][g, :n].double(), s["v_proj"][:, g].double()])
        x = (q[:, h] @ keys.T / 16).masked_fill(~seen, -torch.inf)
        size = (q[:, h].abs() @ keys.abs().T / 16).masked_fill(~seen, 0)
        p = torch.softmax(x, -1)
        for i in range(m):
            if not nodes[i]:
                continue
            at = seen[i]
            o = p[i, at] @ values[at]
            mean = p[i, at] @ values[at].abs()
            d = (2.0 ** -7 + 256 * EPS) * size[i].max() + (2.0 ** -7 * size[i, n:].max() if m else 0)
            z = torch.sigmoid(s["q_proj"][i, h, DIM:].double())
            out[i, h] = o * z
            off[i, h] = (torch.expm1(2 * d) + 2 * BF + (n + m) * EPS) * mean * z
    return out, k, off


def attn_case(rows, q_heads, kv_heads, position, parents, seed=0, scale=1.0, capacity=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(*shape, device="cuda").normal_(mean, std, generator=g).to(torch.bfloat16)

    capacity = max(1, position + 7 if capacity is None else capacity)
    s = dict(rows=rows, q_heads=q_heads, kv_heads=kv_heads, position=position, capacity=capacity, parents=parents,
             nodes=nodes_of(parents), paths=words(parents), q_proj=normal(rows, q_heads, 2 * DIM),
             k_proj=normal(rows, kv_heads, DIM), v_proj=normal(rows, kv_heads, DIM),
             q_gain=normal(DIM, mean=scale, std=0.1), k_gain=normal(DIM, mean=1.0, std=0.1),
             inv_freq=torch.from_numpy(E.rope_inv_freq()).cuda(), k_cache=normal(kv_heads, capacity, DIM),
             v_cache=normal(kv_heads, capacity, DIM))
    # what lies behind the context is nobody's business
    s["k_cache"][:, position:] = torch.nan
    s["v_cache"][:, position:] = torch.inf
    return s


def run_attn(s, stream=None, buffers=None):
    """gated, k_tree; checks that nothing else is written."""
    m, hq, hk = s["rows"], s["q_heads"], s["kv_heads"]
    need = int(E.lib().es_attn_tree_scratch_bytes(hq, hk, m))
    assert need > 0
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((m * hq * DIM + 32,), -3.0, dtype=torch.bfloat16, device="cuda")
    k_tree = torch.full((m * hk * DIM + 32,), -3.0, dtype=torch.bfloat16, device="cuda")
    kept = [s[x].clone() for x in ("k_cache", "v_cache")]
    torch.cuda.synchronize()
    call("es_attn_tree", s["q_proj"], s["k_proj"], s["v_proj"], s["q_gain"], s["k_gain"], s["inv_freq"], s["paths"], m, hq,
         hk, s["k_cache"], s["v_cache"], s["capacity"], s["position"], scratch, need, k_tree, out, stream=stream)
    torch.cuda.synchronize()
    assert (out[m * hq * DIM:] == -3).all() and (k_tree[m * hk * DIM:] == -3).all() and (scratch[need:] == 255).all()
    for a, x in zip(kept, ("k_cache", "v_cache")):
        assert torch.equal(a.view(torch.int16), s[x].view(torch.int16)), "the cache is read only"
    return out[:m * hq * DIM].view(m, hq, DIM), k_tree[:m * hk * DIM].view(m, hk, DIM)


def near(got, want, bound, what):
    most = torch.finfo(got.dtype).max  # what the output's type cannot hold is an infinity there
    got, want = got.double(), want.double()
    want = torch.where(want.abs() > most, want.sign() * torch.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.equal(inf, torch.isinf(got)), f"{what}: other infinities"
    ok = torch.isfinite(want)
    bad = ok & ~((got - want).abs() <= bound)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        b = bound if isinstance(bound, float) else torch.as_tensor(bound).expand_as(want)[i]
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first {i}: {got[i]} for {want[i]} +- {b}")
    return ok


def check_attn(s, got, spread=True):
    out, k, off = attention(s)
    near(got[1], k.double(), 2 * BF * k.double().abs() + 1e-30, "k_tree")
    ok = near(got[0], out, off + BF * out.abs() + 1e-38, "gated")
    if spread and ok.any() and out[ok].norm() > 0:
        # independent roundings of probabilities and of the output, each below 2^-8 / sqrt(3) in the root mean square
        err = float((got[0].double() - out)[ok].norm() / out[ok].norm())
        assert err <= BF, f"root mean square error {err:.2e}"


# --------------------------------------------------------- Gated DeltaNet
def gdn_case(rows, position, parents, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(*shape, device="cuda").normal_(mean, std, generator=g)

    return dict(rows=rows, position=position, parents=parents, nodes=nodes_of(parents), paths=words(parents),
                raw=bf(normal(rows, CONV)), ring=bf(normal(4, CONV)), conv_w=bf(normal(CONV, 4, std=0.5)),
                a_proj=bf(normal(rows, HEADS)), b_proj=bf(normal(rows, HEADS)), a_log=normal(HEADS, std=0.4) + 0.1,
                dt_bias=bf(normal(HEADS, mean=-1.0, std=0.5)), state=normal(HEADS, STATE, STATE, std=0.1))


def run_gdn(s, stream=None):
    m = s["rows"]
    y = torch.full((m * 2048 + 32,), -3.0, dtype=torch.bfloat16, device="cuda")
    k, u = (torch.full((m * 2048 + 32,), -3.0, device="cuda") for _ in range(2))
    lg = torch.full((m * HEADS + 32,), -3.0, device="cuda")
    kept = {x: s[x].clone() for x in ("state", "ring", "raw")}
    torch.cuda.synchronize()
    call("es_gdn_tree", s["raw"], s["ring"], s["conv_w"], s["a_proj"], s["b_proj"], s["a_log"], s["dt_bias"], s["paths"],
         s["position"], m, s["state"], y, k, u, lg, stream=stream)
    torch.cuda.synchronize()
    for t in (y, k, u, lg):
        assert (t[-32:] == -3).all()
    for x, a in kept.items():
        assert torch.equal(a.view(torch.int16), s[x].view(torch.int16)), f"{x} is read only"
    return y[:-32].view(m, 2048), k[:-32].view(m, HEADS, STATE), u[:-32].view(m, HEADS, STATE), lg[:-32].view(m, HEADS)


def gdn(s):
    """(y, k, u, log g) in 64 bits, each with how far it may be off.

    Beside every value runs the same recurrence over magnitudes (sums of absolute
    values). An expression of at most `c` roundings is off by c 2^-24 of its
    magnitude, and what an ancestor's u is off by arrives through the magnitude's own
    terms, so a node's error is at most (ancestors + 1) c 2^-24 of its magnitude. c counts
    128 + 64 additions of the sums and their products, the convolution, exponentials
    and divisions before them (24), and the angles of the gates: a sum of log gates is
    rounded to 32 bits, 2^-24 of it in the exponential."""
    n, dev = s["position"], s["raw"].device
    raw, ring, w = s["raw"].double(), s["ring"].double(), s["conv_w"].double()
    x = s["a_proj"].double() + s["dt_bias"].double()
    log_g = -s["a_log"].double().exp() * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    log_off = EPS * (12 + x.abs()) * log_g.abs() + 1e-45
    beta = torch.sigmoid(s["b_proj"].double())
    zero = torch.zeros(HEADS, STATE, dtype=torch.float64, device=dev)
    res = {name: [] for name in ("y", "k", "u", "ym", "um", "km")}
    states, total = {}, {}
    for i, p in enumerate(s["nodes"]):
        if not p:
            for name in res:
                res[name].append(zero)
            log_g[i] = 0
            log_off[i] = 0
            continue
        taps = [ring[(n + len(p) - 1 - b) % 4] if b >= len(p) else raw[p[-1 - b]] for b in (3, 2, 1, 0)]
        c = sum(taps[t] * w[:, t] for t in range(4))
        cm = 1.1 * sum((taps[t] * w[:, t]).abs() for t in range(4))
        a, am = (torch.nn.functional.silu(c).view(3, HEADS, STATE), cm.view(3, HEADS, STATE))
        root = torch.sqrt((a * a).sum(-1, keepdim=True) + 1e-6)
        q, k, v = a[0] / root[0] / STATE ** 0.5, a[1] / root[1], a[2]
        qm, km, vm = am[0] / root[0] / STATE ** 0.5, am[1] / root[1], am[2]
        up = p[-2] if len(p) > 1 else None
        S, Sm = states[up] if up is not None else (s["state"].double(), s["state"].double().abs())
        gate = log_g[i].exp()[:, None, None]
        S, Sm = gate * S, gate * Sm
        u = beta[i][:, None] * (v - (S * k[:, None]).sum(-1))
        um = beta[i][:, None] * (vm + (Sm * km[:, None]).sum(-1))
        S, Sm = S + u[:, :, None] * k[:, None], Sm + um[:, :, None] * km[:, None]
        states[i] = (S, Sm)
        total[i] = log_g[i].abs() + (total[up] if up is not None else 0)
        c = EPS * (len(p) * (216 + total[i][:, None]))
        for name, value in (("y", (S * q[:, None]).sum(-1)), ("k", k), ("u", u),
                            ("ym", c * (Sm * qm[:, None]).sum(-1)), ("um", c * um), ("km", EPS * 24 * km)):
            res[name].append(value)
    res = {name: torch.stack(v) for name, v in res.items()}
    flat = lambda t: t.reshape(t.shape[0], -1)  # noqa: E731
    return (flat(res["y"]), res["k"], res["u"], log_g), (flat(res["ym"]), res["km"], res["um"], log_off)


def check_gdn(s, got):
    want, off = gdn(s)
    for name, a, b, o in zip(("y", "keys", "updates", "log_decay"), got, want, off):
        o = o + BF * b.abs() if name == "y" else o + EPS * b.abs()
        ok = near(a, b, o + 1e-38, name)
        if name in ("keys", "updates") and b[ok].norm() > 0:
            # 32-bit roundings of random sign: far below 2^-16 together
            err = float((a.double() - b)[ok].norm() / b[ok].norm())
            assert err < 2.0 ** -16, f"{name}: root mean square error {err:.2e}"


def kept_state(s, keys, updates, log_decay, node):
    """state and ring behind a node's path in 64 bits, and how far the state may be off."""
    state, size = s["state"].double(), s["state"].double().abs()
    ring, total = s["ring"].clone(), 0
    path = s["nodes"][node]
    for t, j in enumerate(path):
        gate = log_decay[j].double().clamp(min=-1e30).exp()[:, None, None]
        term = updates[j].double()[:, :, None] * keys[j].double()[:, None, :]
        state, size = gate * state + term, gate * size + term.abs()
        ring[(s["position"] + t) % 4] = s["raw"][j]
        total = total + log_decay[j].double().abs().clamp(max=200)
    off = EPS * (len(path) + 16 + total)
    return state, ring, size * (off[:, None, None] if path else 0)
