"""AdamW over many tensors (ops/optim.TensorAdamW) against the formula in 64 bits, with states in 32 bits and in 8, on the
CPU and (marked) on a GPU; the cuts between tensors, odd sizes, unaligned tensors, refusals."""
import math

import pytest
import torch

from skyrl_isoexec_b200.ops.optim import BLOCK, TensorAdamW

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SIZES = [(1,), (7,), (256,), (0,), (257,), (33, 65), (5000,), (2049,), (8,)]
U32 = 2.0 ** -24


def _make(dev, dt, gdt, seed, misalign):
    g = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for k, shape in enumerate(SIZES):
        n = math.prod(shape)
        lead = 1 if misalign and k % 2 else 0                       # every second tensor starts off a 16-byte boundary
        ps.append((torch.randn(n + lead, generator=g) * 0.05).to(dt).to(dev)[lead:].view(shape))
        gs.append(torch.zeros(n + lead, dtype=gdt, device=dev)[lead:].view(shape))
    return ps, gs, g


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt,gdt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                    (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("misalign", [False, True])
def test_steps_match_the_formula_in_64_bits(dev, bits, dt, gdt, misalign):
    ps, gs, gen = _make(dev, dt, gdt, 3, misalign)
    decay = [0.1 if i % 2 else 0.0 for i in range(len(ps))]
    b1, b2, eps, lr = 0.9, 0.97, 1e-8, 1e-2
    opt = TensorAdamW(ps, grads=gs, betas=(b1, b2), eps=eps, weight_decay=decay, state_bits=bits)
    coef = torch.tensor([0.75], device=dev)
    for t in range(1, 5):
        for g in gs:
            g.copy_(torch.randn(g.shape, generator=gen) * 10.0 ** (t - 3))
        gs[5].view(-1)[:600] = 0.0                                   # a whole scale's block without a gradient
        before = [(a.double(), b.double()) for a, b in (opt.moments(i) for i in range(len(ps)))]
        held = [(opt.state["master"][o:o + p.numel()].view(p.shape) if dt == torch.bfloat16 else p).double().clone() for p, o in zip(ps, opt.offsets)]
        opt.step(lr, grad_scale=coef)
        assert opt.step_count == t
        for i, (p, g) in enumerate(zip(ps, gs)):
            if p.numel() == 0:
                continue
            x = g.double() * 0.75
            m = b1 * before[i][0] + (1 - b1) * x
            v = b2 * before[i][1] + (1 - b2) * x * x
            upd = lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
            want = held[i] * (1 - lr * decay[i]) - upd
            got = opt.state["master"][opt.offsets[i]:opt.offsets[i] + p.numel()].view(p.shape) if dt == torch.bfloat16 else p
            # terms of m cancel: its error is counted against their magnitudes. Roundings on the way to m: the product with
            # the scale, two products, one sum, two constants; to v two more; to the update a division, a root (half of v's
            # error), four products and a sum
            mag_m = b1 * before[i][0].abs() + (1 - b1) * x.abs()
            err_m, err_v = 6 * U32 * mag_m, 9 * U32 * v
            den = (v / (1 - b2 ** t)).sqrt() + eps
            tol = 4 * U32 * held[i].abs() + 2 * U32 * want.abs() + lr / (1 - b1 ** t) * err_m / den + 14 * U32 * upd.abs() + 1e-30
            assert ((got.double() - want).abs() <= tol).all(), (i, ((got.double() - want).abs() / tol).max())
            if dt == torch.bfloat16:
                assert torch.equal(p, got.to(torch.bfloat16))
            dm, dv = (y.double() for y in opt.moments(i))
            if bits == 32:
                assert ((dm - m).abs() <= err_m + 1e-38).all() and ((dv - v).abs() <= err_v + 1e-38).all()
                continue
            o, n = opt.offsets[i], p.numel()
            per = torch.arange(o, o + n, device=dev) // BLOCK
            # codes: half a step of e4m3 (2^-4 of the value; 2^-10 of the scale below its normal numbers)
            s = opt.state["exp_avg_scale"][per].double().view(p.shape)
            assert ((dm - m).abs() <= m.abs() * 2.0 ** -4 + s * 2.0 ** -10 + 2 * err_m + 1e-37).all()
            r, sv = v.sqrt(), opt.state["exp_avg_sq_scale"][per].double().view(p.shape)
            # a root's code is never less than the smallest one, 2^-9 of the scale
            assert ((dv.sqrt() - r).abs() <= r * (2.0 ** -4 + 1e-5) + sv * 2.0 ** -9 + 1e-37).all()
            assert ((dv > 0) | (v < 1e-37) | (sv == 0)).all()
            for blk in range(o // BLOCK, -(-(o + n) // BLOCK)):
                here = m.reshape(-1)[max(0, blk * BLOCK - o):blk * BLOCK - o + BLOCK]
                assert abs(opt.state["exp_avg_scale"][blk].item() * 448 - here.abs().max().item()) <= 1e-5 * here.abs().max().item() + 1e-36
    used = torch.zeros(opt.state["exp_avg"].numel(), dtype=torch.bool, device=dev)
    for o, p in zip(opt.offsets, ps):
        used[o:o + p.numel()] = True
    for k in ("exp_avg", "exp_avg_sq"):
        assert not opt.state[k].float()[~used].any()                 # what stands between two sections stays zero


@pytest.mark.parametrize("dev", DEVICES)
def test_own_gradient_buffers_and_resume(dev):
    """Autograd fills the optimizer's buffers; a state dict taken in the middle goes on with the same bits."""
    torch.manual_seed(0)
    x = torch.randn(16, 12, device=dev)

    def run(steps, opt, w):
        for _ in range(steps):
            opt.zero_grad()
            (torch.tanh(x @ w[0] + w[1]).square().sum()).backward()
            opt.step(grad_scale=None)

    def fresh(bits):
        gen = torch.Generator().manual_seed(1)
        w = [(torch.randn(12, 9, generator=gen) * 0.3).to(dev).requires_grad_(True), torch.zeros(9, device=dev).requires_grad_(True)]
        opt = TensorAdamW(w, lr=1e-2, state_bits=bits)
        for p, g in zip(w, opt.grads):
            p.grad = g
        return w, opt

    for bits in (32, 8):
        w, opt = fresh(bits)
        run(3, opt, w)
        sd, kept = opt.state_dict(), [p.detach().clone() for p in w]
        run(3, opt, w)
        w2, opt2 = fresh(bits)
        opt2.load_state_dict(sd)
        with torch.no_grad():
            for p, k in zip(w2, kept):
                p.copy_(k)
        run(3, opt2, w2)
        assert opt2.step_count == 6 and all(torch.equal(a, b) for a, b in zip(w, w2))


def test_refusals():
    p = [torch.zeros(4, 6), torch.zeros(3)]
    bad = [
        (lambda: TensorAdamW([]), "no parameters"),
        (lambda: TensorAdamW(p, state_bits=16), "state_bits"),
        (lambda: TensorAdamW(p, betas=(1.0, 0.9)), "out of range"),
        (lambda: TensorAdamW(p, eps=0.0), "out of range"),
        (lambda: TensorAdamW(p, weight_decay=[0.1]), "weight decays"),
        (lambda: TensorAdamW(p, grads=[torch.zeros(4, 6)]), "gradients for"),
        (lambda: TensorAdamW(p, grads=[torch.zeros(6, 4), torch.zeros(3)]), "same shape"),
        (lambda: TensorAdamW([torch.zeros(6, 4).t()]), "contiguous"),
        (lambda: TensorAdamW([torch.zeros(3, dtype=torch.float16)]), "fp32 or bf16"),
        (lambda: TensorAdamW([torch.zeros(3), torch.zeros(3, dtype=torch.bfloat16)]), "one type"),
        (lambda: TensorAdamW(p, grads=[torch.zeros(4, 6, dtype=torch.float64), torch.zeros(3, dtype=torch.float64)]), "fp32 or bf16"),
        (lambda: TensorAdamW([p[0], p[0]]), "share memory"),
        (lambda: TensorAdamW([p[0], p[0].view(-1)[20:]]), "share memory"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()
    opt = TensorAdamW(p)
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step(grad_scale=torch.ones(2))
    with pytest.raises(ValueError, match="this optimizer"):
        opt.load_state_dict(TensorAdamW(p, state_bits=8).state_dict())
    with pytest.raises(ValueError, match="expected"):
        opt.load_state_dict(TensorAdamW([torch.zeros(1000)]).state_dict())
    assert opt.step_count == 0


@pytest.mark.parametrize("dev", DEVICES)
def test_replaced_storage_is_neither_stepped_nor_freed(dev):
    w = torch.ones(300, device=dev)
    opt = TensorAdamW([w], grads=[torch.ones(300, device=dev)], lr=0.1)
    w.data = torch.zeros(300, device=dev)
    junk = [torch.zeros(300, device=dev) for _ in range(8)]
    if dev == "cuda":
        opt.step()
        torch.cuda.synchronize()
        assert not w.any() and not any(j.any() for j in junk)


@pytest.mark.parametrize("dev", DEVICES)
def test_copies_are_refused_and_replaced_states_stay_allocated(dev):
    import copy

    w = torch.ones(300, device=dev)
    opt = TensorAdamW([w], grads=[torch.ones(300, device=dev)], lr=0.1, state_bits=8)
    for call in (copy.copy, copy.deepcopy):
        with pytest.raises(TypeError, match="state_dict"):
            call(opt)
    old = dict(opt.state)
    opt.state["exp_avg"] = torch.zeros_like(opt.state["exp_avg"])
    assert all(any(t is m for m in opt._memory) for t in old.values())


@pytest.mark.gpu
def test_another_stream_capture_refused_and_version_counters():
    torch.manual_seed(2)
    base = [torch.randn(5000, device="cuda"), torch.randn(31, device="cuda")]
    grads = [torch.randn_like(b) for b in base]
    out = []
    for side in (False, True):
        ps = [b.clone().requires_grad_(True) for b in base]
        opt = TensorAdamW(ps, grads=grads, lr=1e-2, state_bits=8)
        s = torch.cuda.Stream() if side else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                opt.step()
        torch.cuda.current_stream().wait_stream(s)
        out.append([p.detach().clone() for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*out))
    y = (ps[0] * ps[0]).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    n = opt.step_count
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    assert opt.step_count == n
