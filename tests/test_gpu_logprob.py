"""es_logprob_rows on the GPU against its 64-bit model."""
import pytest
import torch

import esdecode as E
import tree as T

pytestmark = pytest.mark.gpu

INF = float("inf")


def run(x, vocab, tokens, top, stream=None):
    """x [rows, stride] bf16; outputs, checking that nothing behind them is written."""
    rows, stride = x.shape[0], x.stride(0)
    need = int(E.lib().es_logprob_scratch_bytes(rows, vocab, top))
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    out = [torch.full((rows + 8,), -3.0, device="cuda") for _ in range(3)]
    ids = torch.full((rows * top + 8,), -3, dtype=torch.int32, device="cuda")
    alt = torch.full((rows * top + 8,), -3.0, device="cuda")
    torch.cuda.synchronize()
    T.call("es_logprob_rows", x, stride, rows, vocab, tokens, top, scratch if need else None, need, *out, ids if top else None,
           alt if top else None, stream=stream)
    torch.cuda.synchronize()
    for t in out + [ids, alt]:
        assert (t[-8:] == -3).all()
    assert (scratch[need:] == 255).all()
    return [t[:rows] for t in out] + [ids[:-8].view(rows, top), alt[:-8].view(rows, top)]


def check(x, vocab, tokens, top, got):
    """32-bit sums of the row's exponentials without its largest: a thread adds at most
    vocab / 256 + 8 of them, each off by its exponential's argument (|x - m| log2(e) 2^-24 and
    a few 2^-24), then 64 bits; what is off counts by its share in the whole. Outputs round once."""
    for r in range(x.shape[0]):
        v = x[r, :vocab].double()
        m = v.max()
        order = torch.where(torch.isnan(v), -INF, v)
        if top:  # by value, -0 as +0, then by index; NaN below -inf
            nan = torch.isnan(v)
            rank = torch.argsort(torch.where(nan, 0, order), descending=True, stable=True)
            rank = torch.cat([rank[~nan[rank]], nan.nonzero()[:, 0]]) if nan.any() else rank
            assert torch.equal(got[3][r].long(), rank[:top]), f"row {r}: alternatives"
        t = int(tokens[r])
        xt = v[t] if 0 <= t < vocab else torch.tensor(float("nan"), dtype=torch.float64, device="cuda")
        if not torch.isfinite(m):
            assert torch.isnan(got[0][r]) and torch.isnan(got[1][r])
            assert got[2][r] == m or (torch.isnan(m) and torch.isnan(got[2][r]))
            assert torch.isnan(got[4][r]).all()
            continue
        d = v - m
        e = d.exp()
        e[int(v.argmax())] = 0
        rest, part = e.sum(), (e * d.clamp(min=-1e300)).sum()
        a = torch.log1p(rest)
        terms = vocab / 256 + 16
        rel = T.EPS * terms * rest / (1 + rest) + 1.5 * T.EPS * part.abs() / (1 + rest)
        ent = a - part / (1 + rest)
        far = part.abs() / (1 + rest)
        square = (e * d.clamp(min=-1e100) ** 2).sum() / (1 + rest)
        near = lambda g, w, b, what: T.near(g.reshape(1), w.reshape(1), float(b) + 1e-44, f"row {r}: {what}")  # noqa: E731
        near(got[0][r], xt - m - a, rel + T.EPS * (xt - m - a).abs().nan_to_num(0, 0, 0), "log probability")
        near(got[1][r], ent, rel * (1 + far) + T.EPS * (terms * far + 1.5 * square) + T.EPS * ent.abs(), "entropy")
        near(got[2][r], m + a, rel + T.EPS * (m + a).abs(), "log sum")
        if top:
            w = v[got[3][r].long()] - m - a
            T.near(got[4][r], w, rel + T.EPS * w.abs().nan_to_num(0, 0, 0), f"row {r}: alternatives")


def logits(rows, stride, seed, peaks=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty(rows, stride, device="cuda").normal_(0, 2.0, generator=g)
    if peaks:
        hot = torch.empty_like(x).uniform_(generator=g) < 0.003
        x += hot * torch.empty_like(x).normal_(9, 3, generator=g)
    tokens = (torch.empty(rows, device="cuda").uniform_(generator=g) * stride).int()
    return x.to(torch.bfloat16), tokens


@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 40, 255, 256, 2047, 2048, 2049, 4096, 8191, 8192, 8193, 16500, 248320])
def test_rows(vocab, top):
    top = min(top, vocab)
    for rows, pad in ((1, 0), (3, 5), (2, 1)):
        x, tokens = logits(rows, vocab + pad, vocab + top)
        x[:, vocab:] = torch.inf  # nobody's
        tokens %= vocab
        check(x, vocab, tokens, top, run(x, vocab, tokens, top))


@pytest.mark.parametrize("rows", [1023, 1024, 1500])
def test_many_rows(rows):
    for vocab in (40, 3001, 9000):
        x, tokens = logits(rows, vocab + 3, rows)
        tokens %= vocab
        got = run(x, vocab, tokens, 7)
        at = [0, 1, 2, 3, 700, rows - 1]
        check(x[at], vocab, tokens[at], 7, [g[at] for g in got])


def test_rows_that_start_anywhere():
    """Rows and the whole tensor off the 16-byte grid."""
    for off in range(1, 9):
        flat, tokens = logits(1, 5 * 3007 + 16, off)
        x = flat[0, off:off + 5 * 3007].view(5, 3007)
        tokens = (tokens * 0 + torch.arange(5, device="cuda", dtype=torch.int32) * 600 + off).int()
        check(x, 3000, tokens, 4, run(x, 3000, tokens, 4))


@pytest.mark.parametrize("vocab", [33, 5000, 70000])
def test_ties_go_to_the_lowest_index(vocab):
    x, tokens = logits(6, vocab, 1, peaks=False)
    x[0] = 1.5                                # all equal
    x[1] = torch.where(x[1] > 0, 3.0, -1.0)   # two values
    x[2] = 0.0
    x[2, 1::2] = -0.0                         # equal values of two kinds
    x[3] = -INF
    x[3, vocab // 2] = 0.25
    x[4] = -INF
    x[4, ::3] = x[5, ::3]
    x[5] = x[5].float().round().to(torch.bfloat16)
    tokens %= vocab
    check(x, vocab, tokens, 32, run(x, vocab, tokens, 32))


def test_rows_in_order():
    """Every element passes all before it, and the reverse."""
    for vocab in (9000, 30000):
        up = torch.linspace(-30, 30, vocab, device="cuda").to(torch.bfloat16)
        x = torch.stack([up, up.flip(0)])
        tokens = torch.tensor([3, vocab - 2], dtype=torch.int32, device="cuda")
        check(x, vocab, tokens, 32, run(x, vocab, tokens, 32))


@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_rows_with_a_nan_or_an_infinity(bad):
    for vocab in (20, 3000, 70000):
        x, tokens = logits(5, vocab, 5)
        tokens %= vocab
        x[1, vocab // 3] = bad
        x[2, :] = bad
        x[3, ::2] = bad
        x[4, vocab - 1] = -INF
        x[0, 0] = -INF
        check(x, vocab, tokens, 13, run(x, vocab, tokens, 13))


def test_values_behind_a_beginning_of_nan():
    """A list full of NaN takes every value after them, -inf too."""
    for vocab, end in ((30000, 9000), (100000, 99990), (300, 290)):
        x, tokens = logits(3, vocab, 5)
        x[0, :end] = float("nan")
        x[1, :end] = float("nan")
        x[1, end:] = -INF
        x[2, :end] = -INF
        x[2, end + 3:] = float("nan")
        tokens %= vocab
        check(x, vocab, tokens, 20, run(x, vocab, tokens, 20))


def test_rows_without_a_finite_logit():
    x, tokens = logits(2, 300, 5)
    x[1] = -INF
    tokens %= 300
    check(x, 300, tokens, 3, run(x, 300, tokens, 3))


def test_rows_of_excluded_tokens():
    """Most of the vocabulary at -inf, whole ranges of it among them."""
    x, tokens = logits(4, 100000, 6)
    x[0, :99990] = -INF
    x[1, 10:] = -INF
    x[2, 20000:90000] = -INF
    x[3][torch.empty(100000, device="cuda").uniform_() < 0.9] = -INF
    check(x, 100000, tokens, 20, run(x, 100000, tokens, 20))


def test_nearly_certain_tokens_keep_their_digits():
    x = torch.full((3, 5000), -20.0, dtype=torch.bfloat16, device="cuda")
    x[:, 1234] = torch.tensor([3.0, -2.0, 10.0], device="cuda")
    tokens = torch.full((3,), 1234, dtype=torch.int32, device="cuda")
    got = run(x, 5000, tokens, 2)
    check(x, 5000, tokens, 2, got)
    want = -4999 * torch.exp(torch.tensor([-23.0, -18.0, -30.0], dtype=torch.float64))
    assert torch.allclose(got[0].cpu().double(), want, rtol=1e-4)


def test_largest_magnitudes():
    x, tokens = logits(4, 4000, 8)
    x[0] = torch.where(x[0] > 0, 3.3e38, -3.3e38).to(torch.bfloat16)
    x[1, 77] = 3.3e38
    x[2] = -3.3e38
    x[2, 9] = -3.2e38
    x[3] *= 1e30
    check(x, 4000, tokens, 3, run(x, 4000, tokens, 3))


def test_tokens_that_are_none_and_outputs_left_out():
    x, _ = logits(3, 3000, 9)
    tokens = torch.tensor([-1, 3000, 5], dtype=torch.int32, device="cuda")
    got = run(x, 3000, tokens, 2)
    assert torch.isnan(got[0][:2]).all() and torch.isfinite(got[0][2])
    check(x, 3000, tokens, 2, got)
    need = int(E.lib().es_logprob_scratch_bytes(3, 3000, 0))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    only = torch.empty(3, device="cuda")
    T.call("es_logprob_rows", x, 3000, 3, 3000, None, 0, scratch, need, None, only, None, None, None)
    torch.cuda.synchronize()
    assert torch.equal(only, got[1])


def test_row_offsets_past_32_bits():
    """The last row starts past 2^32 elements."""
    stride = (1 << 31) + 8
    x = torch.zeros(2 * stride + 5000, dtype=torch.bfloat16, device="cuda")
    rows, tokens = logits(3, 5000, 10)
    for r in range(3):
        x[r * stride:r * stride + 5000] = rows[r]
    tokens %= 5000
    want = run(rows, 5000, tokens, 4)
    got = run(x.as_strided((3, 5000), (stride, 1)), 5000, tokens, 4)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_row_alone_and_among_others_in_graphs_and_on_a_stream():
    x, tokens = logits(8, 50000, 11)
    want = run(x, 50000, tokens, 6)
    one = [run(x[r:r + 1], 50000, tokens[r:r + 1], 6) for r in range(8)]
    for r in range(8):
        check(x[r:r + 1], 50000, tokens[r:r + 1], 6, one[r])
        assert torch.equal(one[r][3][0], want[3][r])
    need = int(E.lib().es_logprob_scratch_bytes(8, 50000, 6))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = [torch.empty(8, device="cuda") for _ in range(3)]
    ids, alt = torch.empty(8, 6, dtype=torch.int32, device="cuda"), torch.empty(8, 6, device="cuda")

    def work():
        T.call("es_logprob_rows", x, 50000, 8, 50000, tokens, 6, scratch, need, *out, ids, alt)

    work()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        work()
    for change in range(3):
        x.copy_(x.roll(change * 1717, 1))
        want = run(x, 50000, tokens, 6)

        def on_side():
            with torch.cuda.stream(side):
                work()

        for go in (graph.replay, on_side, graph.replay):
            for t in out + [ids, alt]:
                t.zero_()
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            for a, b in zip(out + [ids, alt], want):
                assert torch.equal(a, b)


def test_beside_the_greedy_token_of_each_row():
    """es_greedy_bf16 rounds its log sum, and logit less log sum, to bf16: half a step of each."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = T.bf(torch.empty(9, 5003, device="cuda").normal_(0, 3, generator=g))
    tokens = torch.zeros(9, dtype=torch.int32, device="cuda")
    need = int(E.lib().es_head_scratch_bytes(5003))
    scratch, token, lse = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(9, dtype=torch.int32, device="cuda"), \
        torch.empty(9, device="cuda")
    for r in range(9):
        T.call("es_greedy_bf16", x[r].contiguous(), 5003, scratch, need, token[r:], lse[r:])
    torch.cuda.synchronize()
    got = run(x, 5003, token, 1)
    assert torch.allclose(got[2], lse, rtol=T.BF, atol=0)
    assert torch.allclose(got[0], got[4][:, 0], rtol=2 * T.BF, atol=T.BF * float(lse.max()))
    exact = x.double().log_softmax(1)
    assert torch.allclose(got[0].double(), exact[torch.arange(9), token.long()], rtol=8 * T.EPS, atol=0)
