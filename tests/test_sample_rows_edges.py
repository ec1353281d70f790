"""One token per row from one given number (ops/sampling.sample_rows): a row's bits are its own, whatever batch it stands in;
weights that are small beside the largest; an infinite temperature."""
import math

import pytest
import torch
from test_sample_rows import DEVICES, _check, _settings

from skyrl_isoexec_b200.ops.sampling import sample_rows


def _rows(V, gen):
    """Rows of every kind, and some whose beginning misleads whoever lays a histogram out by it."""
    z = torch.randn(24, V, generator=gen) * 2
    x = [z[0], z[1] * 8, z[2] * 0.01, z[3].round(), torch.where(z[4] > 3, 30.0, z[4] * 1e-4), torch.zeros(V), torch.full((V,), -1e-6),
         torch.where(z[5] > 2, z[5], float("-inf")), -z[6].abs() * 30, z[7] + 500, z[8] * 1e-30, torch.where(z[9] > 0, 1e-4, -1e-4)]
    small = torch.full((V,), 1.25 * 2.0 ** -11)              # one large number, all others next to zero
    small[0] = 30.0
    x += [small, small - 15.0, torch.where(torch.arange(V) == 40000 % V, 60.0, z[10])]
    for k, factor in ((11, 1e-4), (12, 40.0), (13, 0.0), (14, 2.5), (15, 0.4), (16, 6.0)):
        row = z[k].clone()
        row[:5000] *= factor
        x.append(row)
    row = z[17].clone()
    row[:5000], row[20000:] = float("-inf"), row[20000:] * 1e-5
    x.append(row)
    for scale in (3.0, 1.0, 0.3):                            # every binade between the largest and far below it has its tokens
        x.append(torch.where(z[18] > 0, 1.0, -1.0) * scale * 2.0 ** (-24 * torch.rand(V, generator=gen)))
    return torch.stack(x)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9001, *(pytest.param(v, marks=pytest.mark.gpu) for v in (60001, 151936, 524288))])
def test_a_row_has_the_same_bits_in_every_batch(dev, dtype, V):
    if dev == "cpu" and V > 10000:
        pytest.skip("no other path there")
    gen = torch.Generator().manual_seed(V)
    x = _rows(V, gen).to(dtype).to(dev)
    n = x.shape[0]
    big = 300 if dev == "cuda" else 40
    for trial in range(4):
        s = _settings(n, gen) if trial else dict(T=torch.ones(n), k=torch.zeros(n, dtype=torch.int64), p=torch.ones(n), m=torch.zeros(n))
        s = {k: v.to(torch.int32 if k == "k" else torch.float32).to(dev) for k, v in s.items()}
        u = torch.rand(n, generator=gen).to(dev) if trial > 1 else torch.full((n,), trial * (1 - 2.0 ** -24), device=dev)
        alone = [sample_rows(x[i:i + 1], u[i:i + 1], *(s[k][i:i + 1] for k in "Tkpm")) for i in range(n)]
        tokens, lps = (torch.cat(t) for t in zip(*alone))
        at = torch.arange(big, device=dev) % n
        many = sample_rows(x[at], u[at], *(s[k][at] for k in "Tkpm"))
        some = sample_rows(x, u, *(s[k] for k in "Tkpm"))
        for got in ((many[0], many[1], at), (*some, torch.arange(n, device=dev))):
            wrong = (got[0] != tokens[got[2]]) | (got[1] != lps[got[2]])
            assert not wrong.any(), (trial, wrong.nonzero()[:, 0].tolist(), got[1][wrong].tolist(), lps[got[2]][wrong].tolist())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [4001, pytest.param(524288, marks=pytest.mark.gpu)])
def test_many_weights_that_are_small_beside_the_largest(dev, dtype, V):
    """One likely token, all others together some 1e-8 of it: each of them is below any whole number of 2^-44 of the largest."""
    if dev == "cpu" and V > 100000:
        pytest.skip("the CPU form sums in 64-bit floating point")
    rows = []
    for top, below in ((0.0, 31.21), (30.0, 31.2), (31.2, 31.2), (2.0, 30.0), (1.0, 36.0), (-3.0, 31.2)):
        row = torch.full((V,), top - below)
        row[::3] += 0.11
        row[17] = top
        rows.append(row)
    x = torch.stack(rows).to(dtype).to(dev)
    n = len(rows)
    u = torch.zeros(n)
    u[::2] = 1 - 2.0 ** -24
    _check(x, u)
    _check(x, u, p=1 - 2.0 ** -24)
    _check(x, u, T=0.5, m=1e-30)
    tokens, lps = _check(x[:, :V - 1], u)
    many = sample_rows(x[:, :V - 1].repeat(30, 1), u.repeat(30).to(dev))
    assert torch.equal(many[0], tokens.repeat(30)) and torch.equal(many[1], lps.repeat(30))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("at", [0.0, 1000.0, -1000.0, 1e30])
def test_temperatures_next_to_the_logits_own_rounding(dev, at):
    """42 temperatures below the largest logit is there less than its rounding, or about as much."""
    gen = torch.Generator().manual_seed(3)
    step = math.ulp(max(abs(at), 2.0 ** -10)) * 2.0 ** 29    # a unit in the last place of fp32
    x = (at + step * torch.randint(-40, 1, (8, 2500), generator=gen).double()).float().to(dev)
    for T in (0.01, 0.012, 0.02, 0.03, 0.1, 0.9, 20.0):
        _check(x, torch.rand(8, generator=gen), T=T * step)
        _check(x, torch.rand(8, generator=gen), T=T * step, p=0.9, m=0.01)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 3001])
def test_an_infinite_temperature_draws_evenly_among_what_is_left(dev, dtype, V):
    gen = torch.Generator().manual_seed(V)
    x = (torch.randn(6, V, generator=gen) * 4).to(dtype)
    x[1, ::2] = float("-inf")
    x[2, ::3] = float("nan")
    x[3, 1:] = float("-inf")
    x[4, 2:7] = torch.finfo(dtype).min
    x[5, :] = float("-inf")
    u = torch.rand(6, generator=gen)
    for k in (0, 3):
        tokens, lps = sample_rows(x.to(dev), u.to(dev), torch.full((6,), float("inf"), device=dev), torch.full((6,), k, dtype=torch.int32, device=dev))
        for i in range(5):
            row = torch.where(x[i].float().isnan(), float("-inf"), x[i].float())
            order = torch.sort(row, descending=True, stable=True).indices[:int((row > float("-inf")).sum())]
            order = order[:k] if k else order
            assert tokens[i].item() == order[int(u[i].item() * len(order))].item()
            assert abs(lps[i].item() + math.log(len(order))) <= 2.0 ** -24 * math.log(len(order)) + 1e-9
        assert tokens[5] == 0 and lps[5] == float("-inf")


@pytest.mark.parametrize("dev", DEVICES)
def test_an_engine_refuses_a_vocabulary_that_the_kernel_does_not_take(dev, monkeypatch):
    from test_adapters_together import _model

    from skyrl_isoexec_b200.engine.llm_engine import EngineConfig, LLMEngine
    from skyrl_isoexec_b200.ops import sampling

    if dev == "cuda":
        from skyrl_isoexec_b200.ops import _native

        assert _native.lib().ix_sample_rows_max_vocab() == sampling.MAX_VOCAB
    model = _model(dev)
    LLMEngine(model, EngineConfig(max_num_seqs=2, num_kv_pages=8, sample_from_numbers=True))
    monkeypatch.setattr(sampling, "MAX_VOCAB", model.cfg.vocab_size - 1)
    with pytest.raises(ValueError, match="sample_from_numbers needs a vocabulary"):
        LLMEngine(model, EngineConfig(max_num_seqs=2, num_kv_pages=8, sample_from_numbers=True))
    LLMEngine(model, EngineConfig(max_num_seqs=2, num_kv_pages=8))
