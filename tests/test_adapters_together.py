"""The per-request operators as they are used together: an adapter bank beside the shared projections of the model in serving
(every request its own adapter and sampling settings) and in training (one backward over the tokens of several tenants),
the step over all factors, and the options that reach them (sampler, LoRA trainer)."""
import math

import pytest
import torch

from skyrl_isoexec_b200.engine.llm_engine import EngineConfig, LLMEngine
from skyrl_isoexec_b200.engine.sampler import Sampler, SamplingParams
from skyrl_isoexec_b200.models.config import get_config
from skyrl_isoexec_b200.models.decoder import DecoderLM, ForwardCtx
from skyrl_isoexec_b200.ops import functional as F
from skyrl_isoexec_b200.ops.optim import TensorAdamW
from skyrl_isoexec_b200.ops.sampling import sample_rows
from skyrl_isoexec_b200.train.lora import AdapterBank, AdapterStore, LoRAAdapter, LoRAConfig, LoRATrainer

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(dev, seed=1):
    return DecoderLM(get_config("tiny-qwen3", **({} if dev == "cpu" else {"dtype": "bfloat16"})), device=dev, seed=seed)


def _adapters(model, ranks=(4, 8, 11), std=0.05):
    out = {}
    for i, r in enumerate(ranks):
        ad = LoRAAdapter.init(model, LoRAConfig(rank=r, alpha=2.0 * r, seed=i))
        g = torch.Generator().manual_seed(100 + i)
        for b in ad.B.values():
            b.copy_(torch.randn(b.shape, generator=g) * std)
        out[f"tenant{i}"] = ad
    return out


def _ctx(model, lens, lora=None):
    dev = model.device_
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(dev)
    return ForwardCtx(positions=pos, meta=F.AttnMeta.packed(lens, model.hq, model.hkv, dev), lora=lora)


@pytest.mark.parametrize("dev", DEVICES)
def test_bank_computes_what_merged_weights_compute(dev):
    """A packed batch of three tenants and the base model against four forwards, each with its adapter merged into the weights."""
    model = _model(dev)
    ads = _adapters(model)
    bank = AdapterBank(model, ads)
    assert bank.rank == 16
    gen = torch.Generator().manual_seed(0)
    lens, who = [37, 150, 64, 21, 130], ["tenant0", "tenant2", None, "tenant1", "tenant0"]
    ids = [torch.randint(0, 2048, (n,), generator=gen) for n in lens]
    per_token = [w for w, n in zip(who, lens) for _ in range(n)]
    with torch.no_grad():
        got = model(torch.cat(ids).to(dev), _ctx(model, lens, bank.batch(per_token)))
        base = model(torch.cat(ids).to(dev), _ctx(model, lens))
        store = AdapterStore(model)
        for n, ad in ads.items():
            store.register(n, ad)
        row = 0
        for x, n, w in zip(ids, lens, who):
            if w is not None:
                store.activate(w)
            else:
                store.deactivate()
            want = model(x.to(dev), _ctx(model, [n]))
            g, b = got[row:row + n], base[row:row + n]
            row += n
            if w is None:
                assert torch.equal(g, want)                  # a row without an adapter keeps the base model's bits
                continue
            # the adapters move the hidden state by far more than the two ways of adding them differ: fp32 sums in another
            # order; in bf16 the merged weights are rounded, two layers of four targets
            moved, apart = (want - b).float().norm(), (g - want).float().norm()
            assert moved > 0.05 * want.float().norm() and apart < (1e-4 if dev == "cpu" else 0.1) * moved, (w, moved, apart)
        store.deactivate()


@pytest.mark.parametrize("dev", DEVICES)
def test_engine_serves_every_request_with_its_own_adapter(dev):
    model = _model(dev)
    ads = _adapters(model)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 2048, (n,), generator=gen).tolist() for n in (9, 140, 30, 140, 30, 5)]
    prompts[3], prompts[4] = prompts[1], prompts[2]          # the same prompts under other adapters: no shared pages
    who = ["tenant0", None, "tenant2", "tenant1", "tenant2", None]
    sp = SamplingParams(max_generate_length=12, temperature=0.0, ignore_eos=True)

    def engine(**kw):
        return LLMEngine(model, EngineConfig(max_num_seqs=8, num_kv_pages=64, max_num_batched_tokens=100, **kw))

    eng = engine(enable_prefix_caching=True)
    eng.set_adapters(AdapterBank(model, ads))
    both = [eng.generate(prompts, sp, adapters=who) for _ in range(2)]
    assert [o.response_ids for o in both[0]] == [o.response_ids for o in both[1]]
    plain = engine().generate(prompts, sp)
    for o, p, w in zip(both[0], plain, who):
        if w is None:
            assert o.response_ids == p.response_ids and o.response_logprobs == p.response_logprobs
    store = AdapterStore(model)
    for n, ad in ads.items():
        store.register(n, ad)
    for i, w in enumerate(who):
        if w is None:
            continue
        store.activate(w)
        merged = engine(use_cuda_graph=False).generate([prompts[i]], sp)[0]      # (engines that come and go: their graphs would, too)
        # greedy tokens may part where two logits are closer than the two ways of adding differ; before that they agree
        a, b = both[0][i], merged
        same = next((k for k in range(12) if a.response_ids[k] != b.response_ids[k]), 12)
        if dev == "cpu":
            assert same == 12
        lps = torch.tensor([a.response_logprobs[:max(same, 1)], b.response_logprobs[:max(same, 1)]])
        assert (lps[0] - lps[1]).abs()[:same].max() < (1e-3 if dev == "cpu" else 0.15) if same else True
        assert a.response_ids != plain[i].response_ids or a.response_logprobs != plain[i].response_logprobs
    store.deactivate()
    with pytest.raises(ValueError, match="unknown adapter"):
        eng.add_request(prompts[0], sp, adapter="nobody")
    with pytest.raises(ValueError, match="unknown adapter"):
        engine().add_request(prompts[0], sp, adapter="tenant0")
    with pytest.raises(ValueError, match="adapters for"):
        eng.generate(prompts, sp, adapters=who[:2])
    eng.add_request(prompts[0], sp, adapter="tenant0")
    with pytest.raises(RuntimeError, match="in flight"):
        eng.set_adapters(None)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_one_training_step_of_several_tenants_and_then_serving(dev, bits):
    """Forward with the bank, loss over every tenant's rows, backward into the step's own buffers, one step over all factors,
    refreshed serving. The factors' gradients against the dense gradient of each tenant's merged weights, projected."""
    model = _model(dev)
    for p in model.parameters():
        p.requires_grad_(False)
    ads = _adapters(model, ranks=(8, 8))
    bank = AdapterBank(model, ads, trainable=True)
    ps = bank.parameters()
    opt = TensorAdamW(ps, grads=[torch.zeros_like(p) for p in ps], lr=1e-3, state_bits=bits)
    for p, g in zip(ps, opt.grads):
        p.grad = g
    gen = torch.Generator().manual_seed(0)
    lens, who = [40, 70, 25], ["tenant0", "tenant1", "tenant0"]
    ids = torch.cat([torch.randint(0, 2048, (n,), generator=gen) for n in lens]).to(dev)
    names = [w for w, n in zip(who, lens) for _ in range(n)]

    def loss(hidden, x):
        lp, _ = F.token_logprobs(model.logits(hidden[:-1]), x[1:])
        return -lp.sum() / 100

    total = loss(model(ids, _ctx(model, lens, bank.batch(names))), ids)
    total.backward()
    before = [p.detach().clone() for p in ps]
    rows = {w: torch.tensor([n == w for n in names], device=dev) for w in ads}
    # the same batch once per tenant with that tenant's adapter merged; its dense gradient from its own rows is dW, and the
    # factors' gradients are s B^T dW and s dW A^T. Rows of the others enter through no weight of this tenant (sequences do not
    # attend to each other), so one loss over all rows serves both
    for w in ads:
        store = AdapterStore(model)
        store.register(w, ads[w])
        store.activate(w)
        dense = {n: model.p(n) for n in bank.A}
        for p in dense.values():
            p.requires_grad_(True)
        hidden = model(ids, _ctx(model, lens))
        lp, _ = F.token_logprobs(model.logits(hidden[:-1]), ids[1:])
        grads = torch.autograd.grad(-(lp * rows[w][:-1]).sum() / 100, list(dense.values()))
        e, s = bank.names.index(w), ads[w].scale
        for (t, p), dW in zip(dense.items(), grads):
            dW = dW.float()
            for got, want in ((bank.A[t].grad[e, :8], s * ads[w].B[t].t() @ dW), (bank.B[t].grad[e, :, :8], s * dW @ ads[w].A[t].t())):
                apart = (got.float() - want).norm() / want.norm()
                assert apart < (2e-3 if dev == "cpu" else 0.1), (w, t, apart.item())
        for p in dense.values():
            p.requires_grad_(False)
        store.deactivate()
    opt.step()
    assert all(not torch.equal(a, b.detach()) for a, b in zip(before, ps)) and opt.step_count == 1
    # a step of Adam is lr times the gradient's sign where the second moment is fresh
    for p, b, g in zip(ps, before, opt.grads):
        big = g.float().abs() > 1e-4
        upd = (p.detach().float() - b.float())[big]
        assert (upd + 1e-3 * g.float()[big].sign()).abs().max() < (2e-5 if dev == "cpu" else 2.0 ** -8 * b.float().abs().max() + 2e-5)
    opt.zero_grad()
    eng = LLMEngine(model, EngineConfig(max_num_seqs=8, num_kv_pages=32, sample_from_numbers=True))
    eng.set_adapters(bank)
    sps = [SamplingParams(max_generate_length=6, temperature=0.8, top_k=20, ignore_eos=True), SamplingParams(max_generate_length=6, top_p=0.9, ignore_eos=True),
           SamplingParams(max_generate_length=6, min_p=0.1, temperature=1.5, ignore_eos=True)]
    outs = eng.generate([ids[:10].tolist()] * 3, sps, adapters=["tenant0", None, "tenant1"])
    assert all(len(o.response_ids) == 6 and all(math.isfinite(v) and v <= 0 for v in o.response_logprobs) for o in outs)


@pytest.mark.parametrize("dev", DEVICES)
def test_sampler_draws_from_numbers(dev):
    torch.manual_seed(0)
    V = 704                                                  # (the framework's log-probabilities want a multiple of 8)
    x = (torch.randn(6, V) * 2).to(torch.float32 if dev == "cpu" else torch.bfloat16).to(dev)
    ps = [SamplingParams(temperature=0.7, top_k=5), SamplingParams(top_p=0.5), SamplingParams(min_p=0.2), SamplingParams(temperature=0.0, top_k=3),
          SamplingParams(top_k=10 ** 12, top_p=0.9), SamplingParams(temperature=1.3)]
    s = Sampler(dev, 5, from_numbers=True)
    u = torch.rand(6, device=dev, generator=torch.Generator(device=dev).manual_seed(5))
    tokens, lps = s(x, ps)
    f = lambda v, dt=torch.float32: torch.tensor(v, dtype=dt, device=dev)  # noqa: E731
    want, _ = sample_rows(x, u, f([0.7, 1, 1, 0, 1, 1.3]), f([5, 0, 0, 3, 2 ** 31 - 1, 0], torch.int32), f([1, 0.5, 1, 1, 0.9, 1]), f([0, 0, 0.2, 0, 0, 0]))
    assert torch.equal(tokens, want)
    raw, _ = F.token_logprobs(x, tokens)
    assert torch.equal(lps, raw)                             # reported: the raw distribution's, as without the option
    again, _ = s(x, ps)
    s.reseed(5)
    assert torch.equal(s(x, ps)[0], tokens) and not torch.equal(again, tokens)
    # a shaped row goes through the same kernel: the banned and the favoured token
    shaped = [SamplingParams(top_k=50, logit_bias={int(x[0].argmax()): -1e9}), SamplingParams(top_k=50, logit_bias={7: 1e9})]
    before = x[:2].clone()
    for _ in range(5):
        t, _ = s(x[:2], shaped)
        assert int(t[0]) != int(x[0].argmax()) and int(t[1]) == 7
    assert torch.equal(x[:2], before)
    # every token drawn is one that the row-by-row form may draw
    row = SamplingParams(temperature=0.9, top_k=8, top_p=0.8)
    allowed = set()
    v, i = (x[0].float() / 0.9).topk(8)
    pr = torch.softmax(v, 0)
    keep = (pr.cumsum(0) - pr) < 0.8
    allowed = set(i[keep].tolist())
    drawn = {int(s(x[:1], [row])[0]) for _ in range(60)}
    assert drawn <= allowed and len(drawn) > 1


@pytest.mark.parametrize("dev", DEVICES)
def test_lora_trainer_steps_all_factors_at_once(dev):
    """The fused step against torch's Adam from the same gradients; the 8-bit one runs and resumes; other names are refused."""
    from skyrl_isoexec_b200.train import algorithms as alg
    from skyrl_isoexec_b200.train.policy_worker import PolicyWorker, WorkerConfig

    gen = torch.Generator().manual_seed(0)
    done = {}
    for kind in ("adam", "fused", "fused8"):
        model = _model(dev)
        worker = PolicyWorker(model, WorkerConfig(), alg.AlgorithmConfig(policy_loss_type="cross_entropy"))
        store = AdapterStore(model)
        store.register("t", LoRAAdapter.init(model, LoRAConfig(rank=4, lr=5e-3, optimizer=kind)))
        store.activate("t")
        tr = LoRATrainer(worker, store, "t")
        tr.set_lr(2e-3)
        gen.manual_seed(1)
        for _ in range(3):
            worker.opt.main_grad.copy_(torch.randn(worker.opt.main_grad.shape, generator=gen) * 1e-2)
            assert tr.optim_step() > 0
        done[kind] = store.adapters["t"]
        sd = tr.opt.state_dict()
        tr.opt.load_state_dict(sd)
    for name in done["adam"].A:
        for a, b in ((done["adam"].A[name], done["fused"].A[name]), (done["adam"].B[name], done["fused"].B[name])):
            # three steps of at most 2e-3 each; torch squares and divides in another order: parts of 1e-5 of a step. The
            # projection of a slightly different B differs in the second step on
            assert (a - b).abs().max() < 1e-5
        assert torch.isfinite(done["fused8"].A[name]).all() and (done["fused8"].B[name] - done["adam"].B[name]).abs().max() < 4e-3
    with pytest.raises(ValueError, match="LoRAConfig.optimizer"):
        LoRATrainer(worker, store_with(model, "sgd"), "t")


def store_with(model, kind):
    store = AdapterStore(model)
    store.register("t", LoRAAdapter.init(model, LoRAConfig(rank=2, optimizer=kind)))
    return store


def test_bank_refusals_and_round_trip():
    model = _model("cpu")
    ads = _adapters(model)
    bank = AdapterBank(model, ads)
    for n, ad in ads.items():
        back = bank.adapter(n)
        assert all(torch.equal(back.A[t], ad.A[t]) and torch.equal(back.B[t], ad.B[t]) for t in ad.A)
    with pytest.raises(ValueError, match="no adapters"):
        AdapterBank(model, {})
    other = LoRAAdapter.init(model, LoRAConfig(rank=4))
    other.A["layers.9.attn.o.weight"] = other.A["layers.0.attn.o.weight"]
    with pytest.raises(ValueError, match="no weight"):
        AdapterBank(model, {"x": other})
    with pytest.raises(ValueError, match="changed its rank"):
        bank.put("tenant0", LoRAAdapter.init(model, LoRAConfig(rank=32, alpha=64.0)))
    part = LoRAAdapter.init(model, LoRAConfig(rank=4, targets=("attn.o.weight",)))
    assert set(AdapterBank(model, {"x": part}).A) == {f"layers.{i}.attn.o.weight" for i in range(2)}


def test_bank_takes_a_scale_that_fp32_rounds_and_refuses_targets_that_are_only_merged():
    model = _model("cpu")
    ad = LoRAAdapter.init(model, LoRAConfig(rank=12, alpha=16.0))
    bank = AdapterBank(model, {"x": ad})
    bank.put("x", ad)
    assert bank.scale.item() == torch.tensor(16 / 12).item()
    wide = LoRAAdapter.init(model, LoRAConfig(rank=4, targets=("attn.o.weight", "embed.weight")))
    with pytest.raises(ValueError, match="only .* are computed"):
        AdapterBank(model, {"x": wide})
    part = AdapterBank(model, {"x": LoRAAdapter.init(model, LoRAConfig(rank=12, alpha=16.0, targets=("attn.o.weight",)))})
    with pytest.raises(ValueError, match="new targets"):
        part.put("x", ad)
    grown = LoRAAdapter.init(model, LoRAConfig(rank=15, alpha=20.0))
    bank.put("x", grown)
    assert all(torch.equal(bank.adapter("x").A[t], grown.A[t].to(bank.A[t].dtype).float()) for t in grown.A)
