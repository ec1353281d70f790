"""An adapter bank that cannot be served is refused when it is built or given to an engine, not in the middle of a step."""
import pytest
import torch
from test_adapters_together import DEVICES, _model

from skyrl_isoexec_b200.engine.llm_engine import EngineConfig, LLMEngine
from skyrl_isoexec_b200.engine.sampler import SamplingParams
from skyrl_isoexec_b200.models.config import get_config
from skyrl_isoexec_b200.models.decoder import DecoderLM
from skyrl_isoexec_b200.ops import lora as ops
from skyrl_isoexec_b200.ops.optim import TensorAdamW
from skyrl_isoexec_b200.train.lora import AdapterBank, LoRAAdapter, LoRAConfig


def test_what_the_kernels_cannot_compute_with():
    ok = dict(adapters=3, rank=16, widths=[("o", 64, 128)], dtype=torch.bfloat16)
    ops.check_bank(**ok)
    ops.check_bank(**{**ok, "adapters": ops.MAX_ADAPTERS, "rank": ops.MAX_RANK})
    for change, words in ((dict(adapters=1025), "at most 1024"), (dict(rank=136), "up to 128"), (dict(rank=12), "multiple of 8"),
                          (dict(widths=[("o", 64, 128), ("d", 60, 64)]), "d is 60 -> 64"), (dict(widths=[("d", 64, 100)]), "multiples of 8"),
                          (dict(dtype=torch.float32), "bf16")):
        with pytest.raises(ValueError, match=words):
            ops.check_bank(**{**ok, **change})


@pytest.mark.gpu
def test_a_bank_that_cannot_be_served_is_refused_when_it_is_built():
    from skyrl_isoexec_b200.ops import _native

    assert ops.MAX_ADAPTERS == _native.lib().ix_lora_max_adapters()
    model = _model("cuda")
    one = LoRAAdapter.init(model, LoRAConfig(rank=4, targets=("attn.o.weight",)))
    with pytest.raises(ValueError, match="up to 128"):
        AdapterBank(model, {"x": one, "y": LoRAAdapter.init(model, LoRAConfig(rank=129))})
    with pytest.raises(ValueError, match="at most 1024"):
        AdapterBank(model, {f"t{i}": one for i in range(1025)})
    eng = LLMEngine(model, EngineConfig(max_num_seqs=4, num_kv_pages=16))
    eng.set_adapters(AdapterBank(model, {"x": LoRAAdapter.init(model, LoRAConfig(rank=128)), **{f"t{i}": one for i in range(1023)}}))
    sp = SamplingParams(max_generate_length=3, ignore_eos=True)
    outs = eng.generate([[1, 2, 3]] * 3, sp, adapters=["x", "t1022", None])
    assert [len(o.response_ids) for o in outs] == [3, 3, 3]


@pytest.mark.parametrize("dev", DEVICES)
def test_an_engine_refuses_a_bank_of_another_model(dev):
    model = _model(dev)
    kw = {} if dev == "cpu" else {"dtype": "bfloat16"}
    other = DecoderLM(get_config("tiny-qwen3", ffn_size=384, **kw), device=dev, seed=1)
    bank = AdapterBank(other, {"x": LoRAAdapter.init(other, LoRAConfig(rank=8))})
    eng = LLMEngine(model, EngineConfig(max_num_seqs=4, num_kv_pages=16))
    with pytest.raises(ValueError, match="does not fit"):
        eng.set_adapters(bank)
    assert eng.adapters is None
    if dev == "cuda":
        host = _model("cpu")
        with pytest.raises(ValueError, match="does not fit"):
            eng.set_adapters(AdapterBank(host, {"x": LoRAAdapter.init(host, LoRAConfig(rank=8))}))
    eng.set_adapters(AdapterBank(model, {"x": LoRAAdapter.init(model, LoRAConfig(rank=8))}))
    eng.set_adapters(None)


@pytest.mark.parametrize("dev", DEVICES)
def test_factors_put_into_a_bank_under_an_optimizer(dev):
    """One tenant's factors are replaced while the bank trains: after refresh_masters() the next step starts from them, and the
    other tenant's masters keep their bits."""
    model = _model(dev)
    a, b = (LoRAAdapter.init(model, LoRAConfig(rank=8, seed=i)) for i in (1, 2))
    bank = AdapterBank(model, {"a": a, "b": b}, trainable=True)
    ps = bank.parameters()
    gen = torch.Generator().manual_seed(0)
    opt = TensorAdamW(ps, grads=[torch.randn(p.shape, generator=gen).to(dev) for p in ps], lr=1e-4)
    opt.step()
    masters = {k: v.clone() for k, v in opt.state.items() if k == "master"}
    other = {t: bank.A[t][1].detach().clone() for t in bank.A}
    new = LoRAAdapter.init(model, LoRAConfig(rank=8, seed=9))
    bank.put("a", new)
    opt.refresh_masters()
    opt.step(0.0)                                            # no step: what is written back is what the masters are
    for t in bank.A:
        assert torch.equal(bank.A[t][0], new.A[t].to(bank.A[t].dtype)) and torch.equal(bank.A[t][1], other[t])
    if masters:
        for p, o in zip(ps, opt.offsets):
            half = p[1].numel()
            assert torch.equal(opt.state["master"][o + half:o + 2 * half], masters["master"][o + half:o + 2 * half])
