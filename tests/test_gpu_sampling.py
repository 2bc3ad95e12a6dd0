"""The choice of the next token (gq_sample) against float64 on the host.

Which tokens are kept and which one is drawn has to be the one that float64
gives, unless u W lies within the sums' rounding of the border between two
tokens: a term is rounded to a whole number of 2^-45 and its exponential is
within 2^-47 of it, so a sum over V tokens is off by less than
d = V * 2^-45 of the largest term.  A drawn token i has to satisfy
cum(i - 1) - d <= u W <= cum(i) + d.  The log-probability is off by the same
relative to W (at least 1), and by its rounding to float32.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_gptq_b200 import eval as E
from jax_gptq_b200 import sampling

INF = math.inf


def _kept(row, t, k, p, mp):
    """(indices in order, weights) kept of one float64 row without NaN."""
    if not (t > 0):
        return np.array([int(np.argmax(row))]), np.array([1.0])
    order = np.argsort(-row, kind="stable")
    order = order[row[order] > -INF]
    mx = row.max()
    with np.errstate(invalid="ignore"):
        d = np.where(row[order] == mx, 0.0, (row[order] - mx) / t)
    w = np.exp(d)
    if k >= 1:
        order, w = order[:int(k)], w[:int(k)]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int(np.count_nonzero(before < p * w.sum())))
        order, w = order[:n], w[:n]
    n = max(1, int(np.count_nonzero(w >= mp)))
    order, w = order[:n], w[:n]
    by = np.argsort(order)
    return order[by], w[by]


def _per_row(v, rows):
    return v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, float(v))


def _check(logits, u, **kw):
    got = sampling.sample_tokens(logits, u, **kw)
    z = logits.double().cpu().numpy()
    z = z[None] if z.ndim == 1 else z
    rows, vocab = z.shape
    t, k, p, mp = (_per_row(kw.get(n, d), rows) for n, d in
                   (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
    uu = u.double().cpu().numpy().reshape(-1)
    tok, lp = got.tokens.cpu().numpy(), got.logprobs.double().cpu().numpy()
    assert got.tokens.dtype == torch.int64 and tok.shape == (rows,) and lp.shape == (rows,)
    for b in range(rows):
        row = np.where(np.isnan(z[b]), -INF, z[b])
        if not (row > -INF).any():
            assert tok[b] == -1 and lp[b] == -INF
            continue
        idx, w = _kept(row, t[b], k[b], p[b], mp[b])
        cum = np.cumsum(w)
        d = vocab * 2.0 ** -45
        at = np.nonzero(idx == tok[b])[0]
        assert len(at) == 1, (b, tok[b], "is not kept")
        i = int(at[0])
        want = uu[b] * cum[-1]
        assert (cum[i] - w[i]) - d <= want <= cum[i] + d, (b, tok[b])
        ref = math.log(w[i] / cum[-1])
        assert abs(lp[b] - ref) <= 2 * d / cum[-1] + 2.0 ** -23 * abs(ref) + 2.0 ** -40
    again = sampling.sample_tokens(logits, u, **kw)
    assert torch.equal(got.tokens, again.tokens) and torch.equal(got.logprobs, again.logprobs)
    return got


def _logits(rows, vocab, dtype, seed, std=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn((rows, vocab), generator=gen, device="cuda") * std
    return z.to(dtype), torch.rand((rows,), generator=gen, device="cuda")


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_p=0.8),
            dict(min_p=0.1), dict(temperature=0.8, top_k=50, top_p=0.95),
            dict(temperature=1.5, top_k=300, top_p=0.7, min_p=0.001), dict(top_p=0.0),
            dict(temperature=0.0), dict(temperature=1e-6), dict(temperature=1e6, top_p=0.5),
            dict(min_p=1.0), dict(top_k=10 ** 9), dict(temperature=30.0, top_k=999, top_p=0.99)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("shape", [(5, 1000), (3, 32001), (2, 128256)])
def test_matches_float64(shape, setting, dtype):
    z, u = _logits(*shape, dtype, shape[1])
    _check(z, u, **setting)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 31, 33, 255, 4097, 8193, 65537])
def test_odd_vocabularies_and_strides(vocab):
    z, u = _logits(9, vocab + 5, torch.bfloat16, vocab)
    for off in (0, 1, 5):  # rows that begin at any alignment
        _check(z[:, off:off + vocab], u, top_k=11, top_p=0.9)
        _check(z.float()[:, off:off + vocab], u)
    _check(z.t().contiguous().t()[:, :vocab], u, top_p=0.5)
    one = sampling.sample_tokens(z[0, :vocab], u[0])
    assert one.tokens.shape == (1,)


def test_one_row_of_any_row_stride():
    """The stride of a dimension of one element says nothing."""
    z, u = _logits(1, 5000, torch.float32, 21)
    want = sampling.sample_tokens(z, u, top_k=40, top_p=0.9)
    column = z.t().contiguous()  # [vocab, 1]
    for row in (column.t(), z[0].as_strided((1, 5000), (1, 1)), z[0].as_strided((1, 5000), (0, 1)),
                z[0].as_strided((1, 5000), (77777, 1)), z[0].expand(1, 5000)):
        assert row.shape == (1, 5000)
        for uu in (u, u[0], u.as_strided((1,), (9,))):
            got = sampling.sample_tokens(row, uu, top_k=40, top_p=0.9)
            assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)
    one = sampling.sample_tokens(z[:, :1].as_strided((1, 1), (3, 5)), u)
    assert one.tokens.tolist() == [0] and one.logprobs.tolist() == [0.0]


@pytest.mark.parametrize("rows", [1, 2, 40, 75, 149, 300, 1000])
def test_many_rows(rows):
    z, u = _logits(rows, 9001, torch.float32, rows)
    _check(z, u.double(), temperature=0.9, top_k=40, top_p=0.9)


def test_equal_logits_in_order_of_index():
    """Borders inside runs of equal logits, longer than any list kept on chip."""
    for vocab in (4, 1000, 30000, 200000):
        z = torch.zeros((6, vocab), device="cuda")
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 0.25], device="cuda")
        n = vocab // 4
        got = _check(z, u)
        assert got.tokens.tolist()[:4] == [0, n, 2 * n, 3 * n]
        got = _check(z, u, top_k=3)
        assert got.tokens.tolist() == [0, 0, 1, 2, 2, 0]
        got = _check(z, u, top_p=0.5)  # the first half: before it less than half lies
        assert got.tokens.tolist()[:4] == [0, vocab // 8 if vocab > 4 else 0, n, 3 * vocab // 8]
        z[:, vocab // 2:] = 1.0
        _check(z, u, top_k=vocab // 2 + 3)
        _check(z, u, top_p=0.8)
        _check(z, u, top_k=vocab // 2 + 3, top_p=0.9, min_p=0.5)
        z[:, 1::3] = -0.0
        _check(z, u, top_k=vocab // 2 + vocab // 5)


def test_coarse_logits_with_many_ties():
    gen = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randint(-6, 7, (12, 50000), generator=gen, device="cuda").to(torch.bfloat16)
    u = torch.rand((12,), generator=gen, device="cuda")
    for setting in (dict(top_k=100), dict(top_k=20000), dict(top_p=0.3), dict(top_p=0.99),
                    dict(top_k=30000, top_p=0.999), dict(min_p=0.3), dict(temperature=3.0, top_p=0.6)):
        _check(z, u, **setting)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_empty_rows(dtype):
    z, u = _logits(12, 5000, dtype, 3)
    z[0] = -INF                       # nothing left
    z[1, 1:] = -INF                   # one token left
    z[2, :4990] = -INF
    z[3] = float("nan")
    z[4, ::2] = float("nan")
    z[5, 77] = INF                    # takes everything
    z[6, 100:103] = INF
    z[7] = torch.finfo(dtype).min     # masks of the type's lowest value, nothing else
    z[8, 10:] = torch.finfo(dtype).min
    z[9] = torch.finfo(dtype).max
    z[10, 9] = torch.finfo(dtype).max
    for setting in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.0),
                    dict(temperature=0.5, top_k=20, top_p=0.9, min_p=0.01)):
        got = _check(z, u, **setting)
        assert got.tokens[0] == -1 and got.tokens[3] == -1 and got.tokens[1] == 0
        assert got.tokens[5] == 77 and 100 <= got.tokens[6] < 103


def _runs_past_min_p(vocab, inside, past, dtype):
    """Rows, temperature and min_p for which `past` equal logits lie 1 part in
    21000 of a bin (an 11th of a power of two) behind the end of min-p's bin,
    with one logit at the top and `inside` equal ones in the bin."""
    z = torch.full((6, vocab), -8.0, device="cuda")
    at = torch.randperm(vocab, generator=torch.Generator().manual_seed(vocab))
    z[:, at[0]] = 0.0
    z[:, at[1:1 + inside]] = -0.9765625
    z[:, at[1 + inside:1 + inside + past]] = -1.0
    return z.to(dtype), 11 / math.log(2) / 21.001, 2.0 ** (-20.7 / 11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,inside,past,k", [
    (5000, 1500, 1000, 1512), (5000, 1500, 1000, 2500), (32000, 1500, 30000, 20000),
    (32000, 2000, 60, 2055), (128256, 1900, 100000, 90000), (128256, 10, 100000, 90000),
    (128256, 10, 1000, 900), (5000, 1500, 1000, 1000), (5000, 2047, 1000, 3000),
    (5000, 2048, 1000, 3000), (5000, 2100, 1000, 3000)])
def test_min_p_before_the_border_of_top_k(vocab, inside, past, k, dtype):
    """The list that min-p makes short enough grows too long by equal logits next
    to its end; the k-th token lies in a later bin."""
    z, t, mp = _runs_past_min_p(vocab, inside, past, dtype)
    u = torch.tensor([0.0, 0.2, 0.4, 0.6, 0.8, 0.999], device="cuda")
    got = _check(z, u, temperature=t, top_k=k, min_p=mp)
    _check(z, u, temperature=t, min_p=mp)
    _check(z, u, temperature=t, top_k=k)
    _check(z, u, temperature=t, top_k=k, top_p=0.97, min_p=mp)
    _check(z, u, temperature=t, top_p=0.999, min_p=mp)
    one = _check(z[2:3], u[2:3], temperature=t, top_k=k, min_p=mp)
    assert one.tokens[0] == got.tokens[2] and one.logprobs[0] == got.logprobs[2]


@pytest.mark.parametrize("k", [3, 2500, 9000, 30000])
def test_top_k_with_min_p_on_coarse_logits(k):
    gen = torch.Generator(device="cuda").manual_seed(k)
    z = torch.randint(-40, 41, (32, 40000), generator=gen, device="cuda").to(torch.bfloat16) / 8
    u = torch.rand((32,), generator=gen, device="cuda")
    # every row another temperature; min_p halfway between the terms of two logits
    t = 0.4 + 3 * torch.rand((32,), generator=gen, device="cuda").double()
    steps = torch.randint(0, 60, (32,), generator=gen, device="cuda")
    mp = torch.exp(-(steps.double() + 0.5) / 8 / t)
    _check(z, u, temperature=t, top_k=k, min_p=mp)
    _check(z.float(), u, temperature=t, top_k=k, min_p=mp)


def test_lowest_temperatures():
    """Logits that differ by subnormal numbers, at temperatures of their size: one
    below 1e-37 counts as 1e-37."""
    z = torch.zeros((4, 3000), device="cuda")
    z += torch.arange(3000, device="cuda") % 50 * -4e-39
    u = torch.tensor([0.0, 0.3, 0.6, 0.999], device="cuda")
    for setting in (dict(top_k=2), dict(top_k=200), dict(top_p=0.3), dict(min_p=0.9),
                    dict(top_k=500, top_p=0.9, min_p=0.8), dict()):
        want = _check(z, u, temperature=1e-37, **setting)
        for t in (2e-38, 1e-40, 1e-300):
            got = sampling.sample_tokens(z, u, temperature=t, **setting)
            assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)
        _check(z * 100, u, temperature=1e-36, **setting)


def test_highest_temperatures():
    """Logits further apart than the largest float32: a temperature above 1e36 counts
    as 1e36, where such a term is zero for every way of finding it."""
    z = torch.full((4, 3000), -3.2e38, device="cuda")
    z[:, ::2] = 3.3e38
    z[:, ::7] = 3.1e38
    z[:, ::11] = 3e36
    u = torch.tensor([0.0, 0.3, 0.6, 0.999], device="cuda")
    for setting in (dict(), dict(top_k=2), dict(top_k=1400), dict(top_k=2500), dict(top_p=0.99),
                    dict(min_p=1e-9), dict(top_k=2900, top_p=0.9999, min_p=1e-14)):
        want = _check(z, u, temperature=1e36, **setting)
        for t in (1e38, 1e300, INF):
            got = sampling.sample_tokens(z, u, temperature=t, **setting)
            assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)
    flat = _logits(4, 3000, torch.float32, 3)[0]
    _check(flat, u, temperature=1e36, top_p=0.5)


def test_settings_per_row():
    rows = 64
    z, u = _logits(rows, 20011, torch.float32, 5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    r = torch.rand((4, rows), generator=gen, device="cuda")
    t = torch.where(r[0] < 0.2, torch.zeros_like(r[0]), 0.3 + r[0])
    k = torch.where(r[1] < 0.3, torch.zeros_like(r[1]), 1 + 500 * r[1])
    p = torch.where(r[2] < 0.3, torch.ones_like(r[2]), r[2])
    mp = torch.where(r[3] < 0.5, torch.zeros_like(r[3]), 0.2 * r[3])
    for kd, fd in ((torch.int32, torch.float32), (torch.int64, torch.float64)):
        got = _check(z, u, temperature=t.to(fd), top_k=k.to(kd), top_p=p.to(fd), min_p=mp.to(fd))
    for i in range(0, rows, 9):  # a row does not depend on its neighbours
        one = sampling.sample_tokens(z[i:i + 1], u[i:i + 1], temperature=t[i:i + 1],
                                     top_k=k.to(torch.int32)[i:i + 1], top_p=p[i:i + 1],
                                     min_p=mp[i:i + 1])
        assert one.tokens[0] == got.tokens[i] and one.logprobs[0] == got.logprobs[i]


def test_ends_of_u():
    z, _ = _logits(4, 3000, torch.float32, 7)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0], device="cuda")
    got = sampling.sample_tokens(z, u, top_k=5)
    kept = [np.sort(np.argsort(-r, kind="stable")[:5]) for r in z.double().cpu().numpy()]
    assert got.tokens.tolist() == [int(kept[0][0]), int(kept[1][-1]), int(kept[2][-1]), int(kept[3][-1])]


def test_frequencies_follow_the_distribution():
    """A fine grid of u: each token's share of draws is its probability, to a step."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    z = torch.randn((1, 40), generator=gen, device="cuda") * 2
    n = 4000
    u = (torch.arange(n, device="cuda") + 0.5).double() / n
    got = sampling.sample_tokens(z.expand(n, 40).contiguous(), u)
    share = torch.bincount(got.tokens, minlength=40).double() / n
    assert float((share - torch.softmax(z[0].double(), 0)).abs().max()) <= 1.0 / n + 1e-12


def test_logprob_is_what_the_evaluation_scores():
    """The unfiltered log-probability against eval's masked NLL of the drawn tokens."""
    z, u = _logits(16, 32000, torch.float32, 11)
    got = sampling.sample_tokens(z, u)
    pair = torch.stack([z, z], dim=1)  # position 0 scores the label at position 1
    labels = torch.stack([got.tokens, got.tokens], dim=1)
    nll, count = E.masked_nll_from_logits(pair, labels)
    assert count == 16
    assert abs(nll + float(got.logprobs.double().sum())) <= 1e-5 * abs(nll)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9000, 40000])
def test_rows_do_not_depend_on_the_batch(vocab, dtype):
    """The split of a row over blocks follows the number of rows; whole-number
    sums make the results the same for every split."""
    z, u = _logits(300, vocab, dtype, vocab)
    settings = dict(temperature=0.5 + torch.rand(300, device="cuda"),
                    top_k=torch.where(u < 0.5, 0, 1 + (u * 3000)).int(),
                    top_p=torch.where(u < 0.2, 1.0, 0.5 + u / 2), min_p=torch.where(u > 0.7, 0.01, 0.0))
    all_at_once = sampling.sample_tokens(z, u, **settings)
    for n in (1, 20, 100):
        some = sampling.sample_tokens(z[:n], u[:n], **{k: v[:n] for k, v in settings.items()})
        assert torch.equal(some.tokens, all_at_once.tokens[:n])
        assert torch.equal(some.logprobs, all_at_once.logprobs[:n])


@pytest.mark.parametrize("rows,vocab", [(150, 110000), (2, 1 << 20)])
def test_flat_rows(rows, vocab):
    """Nearly all of a block's tokens in one cell: its sums have to have room for
    that many terms, however many tokens the block has."""
    z = (-(64 + torch.arange(rows, device="cuda")) / 256)[:, None].repeat(1, vocab)
    z[:, torch.arange(vocab, device="cuda") % 11 > 8] -= 1 / 256  # the border is among these
    z = z.bfloat16()
    z[:, 3] = 0
    u = torch.rand((rows,), generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda")
    _check(z, u, top_p=0.95)


def test_streams_and_graphs():
    z, u = _logits(8, 32000, torch.bfloat16, 13)
    kw = dict(temperature=0.8, top_k=50, top_p=0.9)
    ref = sampling.sample_tokens(z, u, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = sampling.sample_tokens(z, u, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got.tokens, ref.tokens)
    graphs, outs, bufs = [], [], [z.clone(), z.clone()]
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sampling.sample_tokens(b, u, **kw))
        graphs.append(g)
    bufs[1].copy_(z.flip(1))
    want = sampling.sample_tokens(bufs[1], u, **kw)
    graphs[0].replay()
    graphs[1].replay()
    assert torch.equal(outs[0].tokens, ref.tokens) and torch.equal(outs[1].tokens, want.tokens)


def test_refusals():
    z, u = _logits(4, 100, torch.float32, 1)
    for args, kw, text in (((z.double(), u), {}, "logits must be float32"),
                           ((z[None], u), {}, "rows, vocab"), ((z[:, :0], u), {}, "rows, vocab"),
                           ((z.cpu(), u), {}, "CUDA device"), ((z, u[:3]), {}, "u must have"),
                           ((z, u.cpu()), {}, "u must have"), ((z, u.half()), {}, "u must be"),
                           ((z, u), dict(temperature=-1.0), "temperature"),
                           ((z, u), dict(temperature=float("nan")), "temperature"),
                           ((z, u), dict(top_k=-1), "top_k"), ((z, u), dict(top_p=1.5), "top_p"),
                           ((z, u), dict(top_p=-0.1), "top_p"), ((z, u), dict(min_p=2.0), "min_p"),
                           ((z, u), dict(top_p=u.half()), "top_p must be"),
                           ((z, u), dict(top_k=torch.ones(3, dtype=torch.int32, device="cuda")), "top_k must have")):
        with pytest.raises(ValueError, match=text):
            sampling.sample_tokens(*args, **kw)
    empty = sampling.sample_tokens(z[:0], u[:0])
    assert empty.tokens.shape == (0,) and empty.logprobs.shape == (0,)
