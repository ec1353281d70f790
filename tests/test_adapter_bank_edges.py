"""An adapter bank that cannot be served is refused when it is built or given to an engine, not in the middle of a step."""
import pytest
import torch
from test_adapters_together import DEVICES, _model

from skyrl_isoexec_b200.engine.llm_engine import EngineConfig, LLMEngine
from skyrl_isoexec_b200.engine.sampler import SamplingParams
from skyrl_isoexec_b200.models.config import get_config
from skyrl_isoexec_b200.models.decoder import DecoderLM
from skyrl_isoexec_b200.ops import lora as ops
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
