"""Sampling one token per row from a given number (ops/sampling.sample_rows) against the definition in 64 bits, row by row
and without a histogram: every setting, ties, masks, infinities, rows without a choice, strides, refusals."""
import math

import numpy as np
import pytest
import torch

from skyrl_isoexec_b200.ops.sampling import sample_rows

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _by_definition(x, u, T, k, p, m):
    """(token, log-probability, distance of u's place from the nearest border of two tokens) of one row, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    top = x.max()
    if top == -np.inf:
        return 0, -np.inf, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    if not T > 0:
        return int(order[0]), 0.0, 1.0
    v = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(v == top, 1.0, np.exp((v - top) / T))
    n = len(w) if k <= 0 else min(k, len(w))
    if m > 0:
        n = min(n, int((w >= m).sum()))
    w = w[:max(n, 1)]
    if p < 1:
        total, run, n = math.fsum(w), 0.0, 0
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < p * total).sum()))
        w = w[:n]
    c = np.cumsum(w)
    at = min(int((c <= u * c[-1]).sum()), int((w > 0).sum()) - 1)
    return int(order[at]), math.log(w[at] / c[-1]), float(np.abs(np.concatenate([c / c[-1]]) - u).min())


def _check(logits, u, T=None, k=None, p=None, m=None):
    dev, n = logits.device, logits.shape[0]
    f = lambda t, d, dt: None if t is None else torch.as_tensor(t, dtype=dt).expand(n).contiguous().to(dev)  # noqa: E731
    u, T, p, m = (f(t, 0, torch.float32) for t in (u, T, p, m))
    k = f(k, 0, torch.int32)
    tokens, lps = sample_rows(logits, u, T, k, p, m)
    assert tokens.dtype == torch.int64 and lps.dtype == torch.float32 and tokens.shape == lps.shape == (n,)
    x = logits.float().cpu().numpy()
    num = lambda t, i, d: d if t is None else t[i].item()  # noqa: E731
    for i in range(n):
        tok, lp, far = _by_definition(x[i], num(u, i, 0.0), num(T, i, 1.0), num(k, i, 0), num(p, i, 1.0), num(m, i, 0.0))
        # both sides sum in 64 bits: on a border within 1e-11 of the weight either neighbour is right
        assert tokens[i].item() == tok or far < 1e-11, (i, tokens[i].item(), tok, far)
        if tokens[i].item() == tok:
            # one rounding of a number of at most |lp|, and the logarithm of a quotient known to 1e-11
            assert lps[i].item() == lp or abs(lps[i].item() - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (i, lps[i].item(), lp)
    again = sample_rows(logits, u, T, k, p, m)
    assert torch.equal(tokens, again[0]) and torch.equal(lps, again[1])
    return tokens, lps


def _settings(n, gen):
    pick = lambda vals: torch.tensor(vals)[torch.randint(len(vals), (n,), generator=gen)]  # noqa: E731
    return dict(T=pick([0.0, 0.2, 0.7, 1.0, 1.0, 2.5, -1.0]), k=pick([0, 0, 1, 2, 5, 50, 10 ** 6, -3]), p=pick([1.0, 0.95, 0.5, 0.1, 0.0, 2.0]),
                m=pick([0.0, 0.0, 0.01, 0.2, 1.0, -1.0]))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 9, 64, 1000, 2048, 4097, 32003])
def test_every_setting_on_ordinary_rows(dev, dtype, V):
    gen = torch.Generator().manual_seed(V)
    n = 40
    x = (torch.randn(n, V, generator=gen) * 2.5 + 6.0 * (torch.rand(n, V, generator=gen) < 5 / V)).to(dtype).to(dev)
    u = torch.rand(n, generator=gen)
    _check(x, u)
    _check(x, u, **_settings(n, gen))
    for name, value in (("T", 0.6), ("k", 20), ("p", 0.8), ("m", 0.05)):
        _check(x, u, **{name: value})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V", [(1, 151936), (3, 248320), (40, 128256), (5, 524288), (160, 70001), (300, 32000)])
def test_whole_vocabularies(dtype, n, V):
    gen = torch.Generator().manual_seed(n)
    x = (torch.randn(n, V, generator=gen) * 2.0).to(dtype).cuda()
    u = torch.rand(n, generator=gen)
    _check(x, u)
    _check(x, u, **_settings(n, gen))
    _check(x, u, p=0.9)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shapes_of_the_distribution(dev, dtype):
    """Ties, constant rows, two values, values close to zero beside large ones, wide and narrow rows, both zeros."""
    gen = torch.Generator().manual_seed(5)
    V = 3001
    z = torch.randn(16, V, generator=gen)
    rows = [torch.full((V,), 1.5), torch.zeros(V), torch.where(z[0] > 0, 2.0, -1.0), (z[1] * 4).round(), z[2] * 1e-3, z[3] * 1e-30, z[4] * 300,
            torch.where(z[5] > 2, 9.0, z[5] * 1e-6), torch.where(z[6] > 2, 1.0, z[6] * 1e-6), -z[7].abs() * 1e-5, torch.where(z[8] > 0, 0.0, -0.0),
            z[9] * 1e37, torch.linspace(-50, 0, V), torch.linspace(0, 1e-6, V).flip(0), torch.where(z[10] > 0, 1e-4, -1e-4), z[11] + 1000]
    x = torch.stack(rows).to(dtype).to(dev)
    n = len(rows)
    for trial in range(6):
        u = torch.rand(n, generator=gen)
        _check(x, u)
        _check(x, u, **_settings(n, gen))
    _check(x, torch.zeros(n))
    _check(x, torch.full((n,), 1 - 2.0 ** -24))
    for k in (1, 2, 999, V - 1, V, V + 1):
        _check(x, torch.rand(n, generator=gen), k=k)
    for p in (1e-30, 0.25, 0.5, 1 - 2.0 ** -24):
        _check(x, torch.rand(n, generator=gen), p=p)
    for T in (1e-30, 1e-3, 50.0, 1e30, float("inf")):
        _check(x, torch.rand(n, generator=gen), T=T)
    for m in (1e-30, 0.5, 1.0, 3.0):
        _check(x, torch.rand(n, generator=gen), m=m)


@pytest.mark.gpu
def test_rows_whose_beginning_says_nothing_about_the_rest():
    """Long rows in a large batch are laid out by their first tokens: all kinds of beginnings that mislead."""
    gen = torch.Generator().manual_seed(11)
    V, n = 60001, 160
    x = torch.randn(n, V, generator=gen) * 2
    x[0:10, :5000] = float("-inf")                                   # nothing there
    x[10:20, :5000] *= 1e-4                                          # much smaller than the rest
    x[20:30, :5000] *= 40                                            # and much larger
    x[30:40] = torch.where(x[30:40] > 7.9, x[30:40], x[30:40] * 1e-6)
    x[40:50, :5000] = -x[40:50, :5000].abs() - 1                     # all below zero, the rest next to it
    x[40:50, 5000:] *= 1e-7
    x[50:60, 55000] = 60.0                                           # the largest comes late
    x[60:70, :5000] = 0.0
    x[70:80, :5000] = float("nan")
    x[80:90, 59999] = float("inf")
    x[90:100] = -x[90:100].abs() * 30
    x[90:100, 50000:] = -1e-3
    x[100:110, 1:] = float("-inf")
    x[110:120, :4200] = -1e30
    x[120:130] = -1e-6 * x[120:130].abs()
    x[120:130, 5000] = 1e-3
    x = x.bfloat16().cuda()
    for trial in range(2):
        _check(x, torch.rand(n, generator=gen), **(_settings(n, gen) if trial else {}))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_infinities_and_nan(dev, dtype):
    gen = torch.Generator().manual_seed(6)
    V, inf, nan = 2500, float("inf"), float("nan")
    z = torch.randn(12, V, generator=gen) * 2
    x = z.clone()
    x[0] = -inf                                          # nothing left
    x[1] = nan
    x[2] = -inf
    x[2, 1234] = -3.0                                    # one token
    x[3] = torch.where(z[3] > 1, z[3], -inf)
    x[4] = torch.where(z[4] > 1, z[4], nan)
    x[5] = torch.where(z[5] > 1, z[5], torch.finfo(dtype).min)      # masked by the type's lowest number
    x[6] = torch.finfo(dtype).min                        # and nothing but that
    x[7, 77], x[7, 1777] = inf, inf                      # two certain tokens
    x[8, 5], x[8, 6] = inf, nan
    x[9] = torch.where(z[9] > 1, z[9], -1e9)
    x[10, 3:] = -inf
    x[11] = inf
    x = x.to(dtype).to(dev)
    for trial in range(4):
        u = torch.rand(12, generator=gen)
        _check(x, u)
        tokens, lps = _check(x, u, **_settings(12, gen))
        assert tokens[0] == 0 and lps[0] == -inf and tokens[1] == 0 and tokens[2] == 1234
        assert (tokens >= 0).all() and (tokens < V).all()
    _check(x, u, T=0.0)
    # numbers outside [0, 1) are moved to its ends
    for bad, good in ((-0.5, 0.0), (1.0, 1 - 2.0 ** -24), (7.0, 1 - 2.0 ** -24), (nan, 0.0), (inf, 1 - 2.0 ** -24), (-inf, 0.0)):
        b, g = (torch.full((12,), v, device=dev) for v in (bad, good))
        assert all(torch.equal(s, t) for s, t in zip(sample_rows(x, b), sample_rows(x, g)))
    # settings that are no numbers are off, a temperature that is none is greedy
    for name in ("p", "m"):
        assert torch.equal(_check(x, u, **{name: nan})[0], _check(x, u)[0])
    assert torch.equal(_check(x, u, T=nan)[0], _check(x, u, T=0.0)[0])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dev, dtype):
    gen = torch.Generator().manual_seed(7)
    wide = torch.full((9, 1200), float("inf")).to(dtype).to(dev)     # whoever reads beside the row draws that
    for off in (0, 1, 3, 8):
        for V in (1, 5, 1000, 1013):
            x = (torch.randn(9, V, generator=gen) * 2).to(dtype).to(dev)
            buf = wide.clone()
            buf[:, off:off + V] = x
            u = torch.rand(9, generator=gen)
            got, _ = _check(buf[:, off:off + V], u, T=0.9, p=0.95)
            assert torch.equal(got, _check(x, u, T=0.9, p=0.95)[0])
    x = torch.randn(64, 33, generator=gen).to(dtype).to(dev)
    u = torch.rand(33, generator=gen)
    assert torch.equal(_check(x.t(), u)[0], _check(x.t().contiguous(), u)[0])
    one = x.t()[:1].contiguous().expand(7, 64)
    _check(one, torch.rand(7, generator=gen), k=10)
    s = torch.rand(18, generator=gen).to(dev)[::2]
    sample_rows(wide[:, :7].contiguous(), s, s, None, s, s)          # settings with a stride
    empty = sample_rows(wide[:0], s[:0])
    assert empty[0].shape == empty[1].shape == (0,)


@pytest.mark.parametrize("dev", DEVICES)
def test_numbers_spread_evenly_give_the_distribution(dev):
    """u = (i + 0.5) / n walks through the kept weight: every token comes up as often as it weighs, give or take one."""
    gen = torch.Generator().manual_seed(8)
    V, n = 37, 4096
    x = (torch.randn(1, V, generator=gen) * 1.5).bfloat16().to(dev)
    u = ((torch.arange(n) + 0.5) / n).to(dev)
    k = torch.full((n,), 12, dtype=torch.int32, device=dev)
    tokens, lps = sample_rows(x.expand(n, V), u, None, k)
    w = torch.exp(x[0].double().cpu())
    kept = w.topk(12).indices
    prob = torch.zeros(V, dtype=torch.float64)
    prob[kept] = w[kept] / w[kept].sum()
    seen = torch.bincount(tokens.cpu(), minlength=V).double()
    assert ((seen - n * prob).abs() <= 1.0 + 1e-6).all()
    assert (lps.cpu().double() - prob[tokens.cpu()].log()).abs().max() < 1e-6


def test_refusals():
    x, u = torch.randn(4, 9), torch.rand(4)
    bad = [
        (lambda: sample_rows(x[0], u), "rows, V"),
        (lambda: sample_rows(x.double(), u), "bf16 or fp32"),
        (lambda: sample_rows(x.half(), u), "bf16 or fp32"),
        (lambda: sample_rows(x[:, :0], u), "empty vocabulary"),
        (lambda: sample_rows(x, None), "one number"),
        (lambda: sample_rows(x, u[:3]), "u is"),
        (lambda: sample_rows(x, u.double()), "u is"),
        (lambda: sample_rows(x, u, torch.ones(4, 1)), "temperature is"),
        (lambda: sample_rows(x, u, 0.7), "temperature is"),
        (lambda: sample_rows(x, u, None, torch.ones(4)), "top_k is"),
        (lambda: sample_rows(x, u, None, torch.ones(4, dtype=torch.int64)), "top_k is"),
        (lambda: sample_rows(x, u, None, None, torch.ones(5)), "top_p is"),
        (lambda: sample_rows(x, u, None, None, None, torch.ones(4).bfloat16()), "min_p is"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


@pytest.mark.gpu
def test_gpu_refusals_capture_and_streams():
    x = torch.randn(6, 3000, device="cuda").bfloat16()
    u = torch.rand(6, device="cuda")
    with pytest.raises(ValueError, match="logits' device"):
        sample_rows(x, u.cpu())
    with pytest.raises(ValueError, match="at most"):
        sample_rows(torch.zeros(1, 2 ** 19 + 1, device="cuda").bfloat16(), u[:1])
    p = torch.full((6,), 0.9, device="cuda")
    want = sample_rows(x, u, None, None, p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = sample_rows(x, u, None, None, p)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_rows(x, u, None, None, p)
    x.copy_(torch.randn(6, 3000, device="cuda").bfloat16())
    u.copy_(torch.rand(6, device="cuda"))
    graph.replay()
    now = sample_rows(x, u, None, None, p)
    assert torch.equal(want[0], other[0]) and torch.equal(got[0], now[0]) and torch.equal(got[1], now[1])
    many = torch.randn(1, 20, device="cuda").bfloat16().expand(70000, 20)      # more rows than one launch takes
    uu = torch.rand(70000, device="cuda")
    tok, _ = sample_rows(many, uu)
    part, _ = sample_rows(many[69990:], uu[69990:])
    assert torch.equal(tok[69990:], part)
