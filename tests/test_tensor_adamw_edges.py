"""AdamW over many tensors (ops/optim.TensorAdamW): states of other tensors, replaced memory, masters of changed weights."""
import pytest
import torch

from skyrl_isoexec_b200.ops.optim import TensorAdamW

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_of_other_tensors_is_refused(dev, dt, bits):
    """Sections are padded to 256 elements, so lists of other tensors may have buffers of the same size."""
    def opt(*shapes):
        return TensorAdamW([torch.zeros(s, dtype=dt, device=dev) for s in shapes], state_bits=bits)

    a = opt((300,), (10,), (20, 30))
    for g in a.grads:
        g.fill_(0.5)
    a.step()
    sd = a.state_dict()
    for shapes in (((10,), (300,), (20, 30)), ((300,), (10,), (30, 20)), ((300,), (10,), (600,)), ((301,), (10,), (20, 30))):
        b = opt(*shapes)
        assert b.state["exp_avg"].shape == a.state["exp_avg"].shape
        with pytest.raises(ValueError, match="differ from number"):
            b.load_state_dict(sd)
        assert b.step_count == 0 and not any(v.float().any() for v in b.state.values())
    for shapes in (((300,), (10,)), ((300,), (10,), (20, 30), (0,))):
        with pytest.raises(ValueError, match="differ from number|expected"):
            opt(*shapes).load_state_dict(sd)
    with pytest.raises(ValueError, match="no step count"):
        a.load_state_dict({"state": {}, "param_groups": []})
    b = opt((300,), (10,), (20, 30))
    b.load_state_dict(sd)
    assert b.step_count == 1 and all(torch.equal(a.state[k].float(), b.state[k].float()) for k in a.state)
    sd.pop("shapes")                                         # a state that was put together elsewhere
    b.load_state_dict(sd)
