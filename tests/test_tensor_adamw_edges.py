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


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_on_the_memory_of_construction_on_every_device(dev, dt, bits):
    """A parameter's storage, a gradient buffer or an entry of ``state`` that was replaced: the step goes on with the first."""
    def run(replace):
        w, g = torch.ones(300, dtype=dt, device=dev), torch.ones(300, device=dev)
        held, opt = w.detach(), TensorAdamW([w], grads=[g], lr=0.1, state_bits=bits)
        opt.step()
        if replace:
            w.data = torch.zeros(300, dtype=dt, device=dev)
            opt.grads[0] = torch.full((300,), -7.0, device=dev)
            for k in opt.state:
                opt.state[k] = torch.zeros_like(opt.state[k])
        opt.step()
        if replace:
            assert not w.any() and not any(v.float().any() for v in opt.state.values())
        sd = opt.state_dict()
        opt.load_state_dict(sd)
        opt.step()
        return held, opt.moments(0)

    (a, am), (b, bm) = run(False), run(True)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(am, bm)) and (a.float() < 0.75).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_settings_that_a_step_does_not_see_cannot_be_set(dev):
    opt = TensorAdamW([torch.ones(8, device=dev)], weight_decay=0.1)
    assert opt.weight_decay == (0.1,)
    with pytest.raises(AttributeError):
        opt.weight_decay = [0.0]
    with pytest.raises(TypeError):
        opt.weight_decay[0] = 0.0
    a, b = (TensorAdamW([torch.ones(8, device=dev)], grads=[torch.ones(8, device=dev)], lr=lr, betas=betas) for lr, betas in ((0.5, (0.8, 0.9)), (0.1, (0.9, 0.99))))
    b.lr, b.betas = 0.5, (0.8, 0.9)
    a.step()
    b.step()
    assert torch.equal(a.params[0], b.params[0])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_refreshed_masters_take_changed_weights_and_keep_the_others(dev, bits):
    gen = torch.Generator().manual_seed(0)
    p = [torch.randn(300, generator=gen).bfloat16().to(dev), torch.randn(7, 9, generator=gen).bfloat16().to(dev), torch.tensor([-0.0, 0.0]).bfloat16().to(dev)]
    opt = TensorAdamW(p, grads=[torch.randn(t.shape, generator=gen).to(dev) for t in p], lr=1e-3, state_bits=bits)
    assert opt.state["master"][opt.offsets[2]].item() == 0.0 and torch.signbit(opt.state["master"][opt.offsets[2]])
    opt.step()
    before = opt.state["master"].clone()
    opt.refresh_masters()
    assert torch.equal(opt.state["master"], before)          # still the parameters' rounding: nothing is lost
    p[0][10:20] = 3.0
    p[1][2] = float("nan")
    opt.refresh_masters()
    now = opt.state["master"]
    at = torch.zeros_like(now, dtype=torch.bool)
    at[10:20], at[opt.offsets[1] + 18:opt.offsets[1] + 27] = True, True
    assert torch.equal(now[~at], before[~at]) and (now[10:20] == 3.0).all() and now[opt.offsets[1] + 18:opt.offsets[1] + 27].isnan().all()
    opt.step(0.0)
    assert (p[0][10:20] == 3.0).all()
