"""Low-rank adapters of many requests (ops/lora.py) where the usual shapes do not go: infinite numbers, every rank on both
sizes of tile, a bank that is larger than the batch's adapters, batches without a token."""
import pytest
import torch
from test_lora_many_adapters import DEVICES, _make, _reference, _tol

from skyrl_isoexec_b200.ops import functional as F
from skyrl_isoexec_b200.ops.lora import LoraPlan, lora_add, lora_linear


def _run(y, x, A, B, scale, ids, dout):
    leaves = [t.clone().requires_grad_(True) for t in (x, A, B)]
    out = lora_add(y, *leaves, scale, LoraPlan(ids, A.shape[0]))
    return dict(zip(("out", "dx", "dA", "dB"), (out.detach(), *torch.autograd.grad(out, leaves, dout))))


def _compare(got, args, shape):
    """Finite results within the derived tolerance, infinite ones equal, no number where the formula gives none."""
    T, K, N, r, E = shape
    ref, mag = _reference(*args)
    for name, g in got.items():
        want, g = ref[name], g.double()
        assert torch.equal(g.isnan(), want.isnan()), (name, "nan", g.isnan().sum().item(), want.isnan().sum().item())
        inf = want.isinf()
        assert torch.equal(g[inf], want[inf]), name
        ok = want.isfinite()
        far, tol = (g - want).abs()[ok], _tol(name, want, mag[name], T, K, N, r)[ok]
        assert (far <= tol).all(), (name, (far / tol).max().item())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("r", [8, 16, 24, 40, 72])
@pytest.mark.parametrize("T,E", [(37, 4), (700, 4)])
def test_infinite_numbers(dev, r, T, E):
    """An infinite x or gradient of one token, and an infinite number of A: what the formula says, no NaN beside it."""
    shape = (T, 72, 104, r, E)
    y, x, A, B, scale, ids, dout = _make(*shape, "shuffled", dev, seed=r)
    A, B, scale = A.abs() + 0.01, B.abs() + 0.01, scale.abs() + 0.5      # so that sums of infinite terms are infinite, not NaN
    ids[2], ids[5], ids[7], ids[9], ids[11] = 3, 0, 1, 1, 2
    inf = float("inf")
    x[5, 3], x[9, 71] = inf, -inf
    dout[7, 2], dout[11, 103], dout[9, 0] = inf, -inf, inf
    y[11, 4] = -inf
    args = (y, x, A, B, scale, ids, dout)
    _compare(_run(*args), args, shape)
    A2 = A.clone()
    A2[3, r - 1, 5] = inf                                # h is infinite where x is not zero there
    x2 = x.clone()
    x2[:, 5] = x2[:, 5].abs() + 0.01
    args = (y, x2, A2, B, scale, ids, dout)
    got = _run(*args)
    got.pop("dx")                                        # (an infinite factor of the second product gives NaN or infinity)
    _compare(got, args, shape)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("r", [8, 16, 24, 32, 48, 64, 72, 104, 128])
@pytest.mark.parametrize("T,E,mode", [(60, 12, "holes"), (230, 2, "shuffled")])
def test_every_rank_in_small_and_large_tiles(dev, r, T, E, mode):
    shape = (T, 328, 264, r, E)
    args = _make(*shape, mode, dev, seed=r)
    _compare(_run(*args), args, shape)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("r", [16, 64])
def test_a_bank_larger_than_the_batch_of_adapters(dev, r):
    """A prompt of one request in a bank of 64: the tile that the bank's size chooses gives what a bank of one gives."""
    shape = (2048, 160, 200, r, 64)
    args = _make(*shape, "one", dev, seed=1)
    got = _run(*args)
    _compare(got, args, shape)
    y, x, A, B, scale, ids, dout = args
    alone = _run(y, x, A[63:], B[63:], scale[63:], torch.zeros_like(ids), dout)
    ref, mag = _reference(*args)
    for name in ("out", "dx"):                           # another order of 32-bit sums, then the same rounding
        assert ((got[name].double() - alone[name].double()).abs() <= 2 * _tol(name, ref[name], mag[name], *shape[:4])).all()
    assert not got["dA"][:63].any() and not got["dB"][:63].any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("odd", ["x", "dout", "both"])
def test_an_empty_batch_of_rows_of_a_wider_buffer(dev, odd):
    """No token, rows with a stride that 8 does not divide: the gradients of the factors are zero."""
    y, x, A, B, scale, ids, dout = _make(40, 64, 48, 8, 2, "shuffled", dev)
    wide_x, wide_d = (torch.full((4, w + 9), float("nan"), device=dev).bfloat16() for w in (64, 48))
    none = slice(2, 2)
    leaf = (wide_x[none, 3:67] if odd != "dout" else x[:0]).detach().requires_grad_(True)
    d = wide_d[none, 5:53] if odd != "x" else dout[:0]
    leaves = [leaf, A.clone().requires_grad_(True), B.clone().requires_grad_(True)]
    out = lora_add(y[:0], *leaves, scale, LoraPlan(ids[:0], 2))
    dx, dA, dB = torch.autograd.grad(out, leaves, d)
    assert out.shape == (0, 48) and dx.shape == (0, 64) and not dA.any() and not dB.any() and dA.shape == A.shape and dB.shape == B.shape
    w = torch.zeros(48, 64, device=dev).bfloat16()
    leaves = [leaf.detach().requires_grad_(True), A.clone().requires_grad_(True), B.clone().requires_grad_(True)]
    out = lora_linear(leaves[0], w, *leaves[1:], scale, LoraPlan(ids[:0], 2))
    assert out.shape == (0, 48) and not any(g.any() for g in torch.autograd.grad(out, leaves, d))


@pytest.mark.parametrize("dev", DEVICES)
def test_on_another_device_than_the_current_one(dev, monkeypatch):
    """The calls run under their tensors' device. (Elsewhere than on two GPUs: the current device only seems to be another.)"""
    y, x, A, B, scale, ids, dout = _make(40, 64, 48, 8, 2, "shuffled", dev)
    w = torch.randn(48, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(dev)
    plan = LoraPlan(ids, 2)
    want = [lora_add(y, x, A, B, scale, plan), lora_linear(x, w, A, B, scale, plan)]
    entered, inside = [], []
    if dev == "cuda":
        seen = F.gemm_nt

        class Under:
            def __init__(self, index):
                entered.append(index)

            def __enter__(self):
                inside.append(1)

            def __exit__(self, *_):
                inside.pop()

        def gemm_nt(*a, **kw):
            assert inside, "the projection outside its tensors' device"
            return seen(*a, **kw)

        monkeypatch.setattr(torch.cuda, "current_device", lambda: plan.index if inside else 1 + plan.index)
        monkeypatch.setattr(torch.cuda, "device", Under)
        monkeypatch.setattr(F, "gemm_nt", gemm_nt)
    got = [lora_add(y, x, A, B, scale, plan), lora_linear(x, w, A, B, scale, plan)]
    leaves = [t.clone().requires_grad_(True) for t in (x, A, B)]
    out = lora_linear(leaves[0], w, *leaves[1:], scale, plan)
    monkeypatch.undo()
    assert torch.equal(out.detach(), want[1]) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(g.isfinite().all() for g in torch.autograd.grad(out, leaves, dout))
    assert dev == "cpu" or set(entered) == {plan.index}
