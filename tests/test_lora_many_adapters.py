"""Low-rank adapters of many requests beside a shared projection (ops/lora.py) against the formulas in 64 bits: output and
gradients, ragged groups, tokens without an adapter, strides, poisoned places nobody may read, refusals."""
import pytest
import torch

from skyrl_isoexec_b200.ops import functional as F
from skyrl_isoexec_b200.ops.lora import LoraPlan, lora_add, lora_linear, pad_rank

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = 2.0 ** -8          # half a step of bf16, relative
SHAPES = [(1, 64, 72, 8, 1), (5, 8, 8, 8, 3), (17, 96, 40, 16, 2), (300, 264, 520, 24, 4), (129, 1000, 128, 64, 3), (700, 512, 264, 128, 2),
          (2050, 256, 392, 32, 1), (64, 2048, 1024, 16, 64), (333, 72, 2056, 40, 1), (49, 4096, 64, 8, 1), (1000, 104, 136, 16, 12)]


def _ids(T, E, mode, gen):
    a = torch.randint(0, E, (T,), generator=gen, dtype=torch.int64)
    if mode == "sorted":
        a = a.sort().values
    elif mode == "holes":                       # no adapter, in every way a number can be out of range
        a[torch.rand(T, generator=gen) < 0.4] = -1
        a[::7] = E
        a[::11] = 2 ** 32                       # would wrap to adapter 0 in 32 bits
        a[3::13] = -(2 ** 31)
    elif mode == "none":
        a[:] = -1
    elif mode == "one":
        a[:] = E - 1
    return a


def _make(T, K, N, r, E, mode, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).bfloat16().to(dev)  # noqa: E731
    ids = _ids(T, E, mode, gen).to(dev)
    return (rnd(T, N), rnd(T, K), rnd(E, r, K, std=K ** -0.5), rnd(E, N, r, std=r ** -0.5), (torch.rand(E, generator=gen) * 2 - 0.5).to(dev), ids, rnd(T, N))


def _reference(y, x, A, B, scale, ids, dout):
    """Results in 64 bits, and for each the sum of magnitudes that its rounding errors scale with."""
    y, x, A, B, s, d = (t.double() for t in (y, x, A, B, scale, dout))
    T, E = x.shape[0], A.shape[0]
    ref = dict(out=y.clone(), dx=torch.zeros_like(x), dA=torch.zeros_like(A), dB=torch.zeros_like(B))
    mag = {k: torch.zeros_like(v) for k, v in ref.items()}
    for a in range(E):
        m = ids == a
        h, g = s[a] * x[m] @ A[a].t(), s[a] * d[m] @ B[a]
        ha, ga = abs(s[a]) * x[m].abs() @ A[a].abs().t(), abs(s[a]) * d[m].abs() @ B[a].abs()
        ref["out"][m] += h @ B[a].t()
        mag["out"][m] += ha @ B[a].abs().t()
        ref["dx"][m], mag["dx"][m] = g @ A[a], ga @ A[a].abs()
        ref["dA"][a], mag["dA"][a] = g.t() @ x[m], ga.t() @ x[m].abs()
        ref["dB"][a], mag["dB"][a] = d[m].t() @ h, d[m].abs().t() @ ha
    return ref, mag


def _tol(name, ref, mag, T, K, N, r):
    # the output's rounding; h and g as two bf16 numbers (2^-16); sums in 32 bits, at most two units of 2^-24 a term
    terms = {"out": K + r, "dx": N + r, "dA": N + T, "dB": K + T}[name]
    return HALF * ref.abs() + mag * (2.0 ** -16 + (terms + 8) * 2.0 ** -23) + 1e-30


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("mode", ["sorted", "shuffled", "holes", "none", "one"])
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_gradients(dev, shape, mode):
    T, K, N, r, E = shape
    y, x, A, B, scale, ids, dout = _make(*shape, mode, dev)
    ref, mag = _reference(y, x, A, B, scale, ids, dout)
    plan = LoraPlan(ids, E)
    served = lora_add(y, x, A, B, scale, plan)
    leaves = [t.clone().requires_grad_(True) for t in (y, x, A, B)]
    out = lora_add(*leaves, scale, plan)
    assert torch.equal(served, out.detach())
    dy, dx, dA, dB = torch.autograd.grad(out, leaves, dout)
    for name, got in (("out", out.detach()), ("dx", dx), ("dA", dA), ("dB", dB)):
        assert got.dtype == torch.bfloat16 and got.shape == ref[name].shape
        far = (got.double() - ref[name]).abs()
        assert (far <= _tol(name, ref[name], mag[name], T, K, N, r)).all(), (name, (far / _tol(name, ref[name], mag[name], T, K, N, r)).max().item())
    assert torch.equal(dy, dout)
    free = (ids < 0) | (ids >= E)
    assert torch.equal(out.detach()[free], y[free]) and not dx[free].any()
    for a in range(E):
        if not (ids == a).any():
            assert not dA[a].any() and not dB[a].any()


@pytest.mark.parametrize("dev", DEVICES)
def test_gradients_against_differences(dev):
    """The operator is linear in x, in A and in B: a difference of any size is the derivative, but for the two outputs' rounding."""
    T, K, N, r, E = 150, 64, 48, 8, 3
    y, x, A, B, scale, ids, dout = _make(T, K, N, r, E, "holes", dev, seed=4)
    plan = LoraPlan(ids, E)
    leaves = [t.clone().requires_grad_(True) for t in (x, A, B)]
    grads = torch.autograd.grad(lora_add(y, *leaves, scale, plan), leaves, dout)
    gen = torch.Generator().manual_seed(9)
    for i, (leaf, grad) in enumerate(zip((x, A, B), grads)):
        step = (torch.randn(leaf.shape, generator=gen) * leaf.float().std().item()).bfloat16().to(dev)
        # both ends must be bf16 numbers themselves: the step is what is really between them
        hi, lo = (leaf + step), (leaf - step)
        outs = [lora_add(y, *[t if j != i else e for j, t in enumerate((x, A, B))], scale, plan).double() for e in (hi, lo)]
        want = ((outs[0] - outs[1]) * dout.double()).sum()
        got = (grad.double() * (hi.double() - lo.double())).sum()
        slack = HALF * ((outs[0].abs() + outs[1].abs()) * dout.double().abs()).sum() + HALF * (grad.double().abs() * (hi.double() - lo.double()).abs()).sum()
        # roundings are independent: twelve of their standard deviations are far inside the sum of all of them
        n = outs[0].numel() + grad.numel()
        assert (want - got).abs() <= 12 * slack / n ** 0.5, (i, want.item(), got.item())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("train", [False, True])
def test_linear_with_adapters_is_the_projection_then_the_adapters(dev, train):
    T, K, N, r, E = 200, 128, 96, 16, 5
    y, x, A, B, scale, ids, dout = _make(T, K, N, r, E, "holes", dev, seed=2)
    w = (torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * K ** -0.5).bfloat16().to(dev)
    plan = LoraPlan(ids, E)
    want = lora_add(F.linear(x, w), x, A, B, scale, plan)
    if not train:
        assert torch.equal(lora_linear(x, w, A, B, scale, plan), want)
        return
    leaves = [t.clone().requires_grad_(True) for t in (x, w, A, B)]
    out = lora_linear(*leaves, scale, plan)
    assert torch.equal(out.detach(), want)
    dx, dw, dA, dB = torch.autograd.grad(out, leaves, dout)
    l2 = [t.clone().requires_grad_(True) for t in (x, w, A, B)]
    gx, gw, gA, gB = torch.autograd.grad(lora_add(F.linear(l2[0], l2[1]), l2[0], l2[2], l2[3], scale, plan), l2, dout)
    assert torch.equal(dA, gA) and torch.equal(dB, gB) and torch.equal(dw, gw)
    # apart, both parts of dx are rounded and so is their sum; together the projection's part and the sum are
    base = (dout.double() @ w.double()).abs()
    part = (gx.double().abs() + base)
    assert ((dx.double() - gx.double()).abs() <= 2 * HALF * (gx.double().abs() + part) + 1e-6).all()
    frozen = [x.clone().requires_grad_(True), w, A.clone().requires_grad_(True), B]
    dx2, dA2 = torch.autograd.grad(lora_linear(*frozen, scale, plan), (frozen[0], frozen[2]), dout)
    assert torch.equal(dx2, dx) and torch.equal(dA2, dA)
    only_b = B.clone().requires_grad_(True)
    (dB2,) = torch.autograd.grad(lora_linear(x, w, A, only_b, scale, plan), only_b, dout)
    assert torch.equal(dB2, dB)


@pytest.mark.parametrize("dev", DEVICES)
def test_strides_leading_dimensions_and_neighbours(dev):
    """Rows of wider buffers, a batch shape, an expanded x and an expanded gradient; what surrounds the rows is not touched."""
    T, K, N, r, E = 60, 64, 40, 8, 3
    y, x, A, B, scale, ids, dout = _make(T, K, N, r, E, "shuffled", dev)
    plan = LoraPlan(ids, E)
    want = lora_add(y, x, A, B, scale, plan)
    for off in (8, 3):                                   # on and off a 16-byte boundary
        wide_x, wide_y = torch.full((T, K + 24), float("nan"), device=dev).bfloat16(), torch.full((T, N + 24), float("nan"), device=dev).bfloat16()
        wide_x[:, off:off + K], wide_y[:, off:off + N] = x, y
        kept = wide_y.clone()
        assert torch.equal(lora_add(wide_y[:, off:off + N], wide_x[:, off:off + K], A, B, scale, plan), want)
        assert torch.equal(wide_y.nan_to_num(7.0), kept.nan_to_num(7.0))
    spaced = torch.full((2 * E,), float("nan"), device=dev)
    spaced[::2] = scale
    assert torch.equal(lora_add(y, x, A, B, spaced[::2], plan), want)
    assert torch.equal(lora_add(y.view(3, 20, N), x.view(3, 20, K), A, B, scale, plan), want.view(3, 20, N))
    odd = torch.full((2, K + 9), float("nan"), device=dev).bfloat16()      # a single row: contiguous, with a stride of K + 9
    odd[0, 8:8 + K] = x[3]
    p1 = LoraPlan(ids[3:4], E)
    assert torch.equal(lora_add(y[3:4], odd[:1, 8:8 + K], A, B, scale, p1), want[3:4])
    one = x[:1].expand(T, K)
    assert torch.equal(lora_add(y, one, A, B, scale, plan), lora_add(y, one.contiguous(), A, B, scale, plan))
    At, Bt = A.transpose(1, 2).contiguous().transpose(1, 2), B.transpose(1, 2).contiguous().transpose(1, 2)
    leaves = [x.clone().requires_grad_(True), At.detach().requires_grad_(True), Bt.detach().requires_grad_(True)]
    lora_add(y, *leaves, scale, plan).sum().backward()
    l2 = [t.clone().requires_grad_(True) for t in (x, A, B)]
    torch.autograd.backward(lora_add(y, *l2, scale, plan), torch.ones_like(y))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, l2))


@pytest.mark.parametrize("dev", DEVICES)
def test_values_that_are_not_finite_stay_in_their_own_rows(dev):
    T, K, N, r, E = 90, 128, 64, 8, 4
    y, x, A, B, scale, ids, dout = _make(T, K, N, r, E, "shuffled", dev)
    ids = ids.clamp(max=2)                               # nobody uses adapter 3: its factors are never read
    ids[4], ids[5] = -1, 1
    clean = lora_add(y, x, A, B, scale, LoraPlan(ids, E))
    A2, B2, x2 = A.clone(), B.clone(), x.clone()
    A2[3], B2[3] = float("nan"), float("inf")
    x2[4] = float("nan")                                 # a token without an adapter
    x2[5, 3] = float("nan")
    leaves = [x2.requires_grad_(True), A2.requires_grad_(True), B2.requires_grad_(True)]
    out = lora_add(y, *leaves, scale, LoraPlan(ids, E))
    rows = torch.arange(T, device=dev) != 5
    assert torch.equal(out.detach()[rows], clean[rows]) and out.detach()[5].isnan().all()
    dx, dA, dB = torch.autograd.grad(out, leaves, dout)
    assert dx.isfinite().all() and dA[[0, 2, 3]].isfinite().all() and dB[[0, 2, 3]].isfinite().all()
    assert dA[1, :, 3].isnan().all() and dA[1, :, :3].isfinite().all()
    assert not dA[3].any() and not dB[3].any()


@pytest.mark.parametrize("dev", DEVICES)
def test_empty_batch_and_padded_rank(dev):
    y, x, A, B, scale, ids, dout = _make(40, 64, 48, 8, 2, "shuffled", dev)
    none = LoraPlan(ids[:0], 2)
    leaves = [t.clone().requires_grad_(True) for t in (x[:0], A, B)]
    out = lora_add(y[:0], *leaves, scale, none)
    assert out.shape == (0, 48)
    grads = torch.autograd.grad(out, leaves, dout[:0])
    assert grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()
    pairs = [pad_rank(a, b, 24) for a, b in zip(A, B)]
    A2, B2 = torch.stack([p[0] for p in pairs]), torch.stack([p[1] for p in pairs])
    plan = LoraPlan(ids, 2)
    got, want = lora_add(y, x, A2, B2, scale, plan).double(), lora_add(y, x, A, B, scale, plan).double()
    ref, mag = _reference(y, x, A, B, scale, ids, dout)
    assert ((got - want).abs() <= 2 * _tol("out", ref["out"], mag["out"], 40, 64, 48, 8)).all()


def test_refusals():
    y, x, A, B, scale, ids, _ = _make(10, 16, 24, 8, 2, "shuffled", "cpu")
    plan = LoraPlan(ids, 2)
    bad = [
        (lambda: LoraPlan(ids.float(), 2), "int32 or int64"),
        (lambda: LoraPlan(ids.view(2, 5), 2), "flat"),
        (lambda: LoraPlan(ids, 0), "at least one"),
        (lambda: lora_add(y, x, A[0], B, scale, plan), "factors are"),
        (lambda: lora_add(y, x, A, B[:1], scale, plan), "factors are"),
        (lambda: lora_add(y, x, A[:, :4], B, scale, plan), "factors are"),
        (lambda: lora_add(y, x[:, :8], A, B, scale, plan), "do not fit"),
        (lambda: lora_add(y[:, :8], x, A, B, scale, plan), "do not fit"),
        (lambda: lora_add(y[:5], x, A, B, scale, plan), "do not fit"),
        (lambda: lora_add(y[:5], x[:5], A, B, scale, plan), "the plan is for"),
        (lambda: lora_add(y, x, A[:1], B[:1], scale[:1], plan), "the plan is for"),
        (lambda: lora_add(y, x, A, B, scale[:1], plan), "scale is"),
        (lambda: lora_add(y, x, A, B, scale.double(), plan), "scale is"),
        (lambda: lora_add(y, x, A, B, scale.clone().requires_grad_(True), plan), "no gradient"),
        (lambda: lora_add(y.float(), x, A, B, scale, plan), "one type"),
        (lambda: lora_linear(x, torch.zeros(24, 8).bfloat16(), A, B, scale, plan), "does not fit"),
        (lambda: pad_rank(A[0], B[0], 4), "do not fit"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


@pytest.mark.gpu
def test_refusals_on_a_gpu():
    y, x, A, B, scale, ids, _ = _make(10, 16, 24, 8, 2, "shuffled", "cuda")
    plan = LoraPlan(ids, 2)
    f = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    bad = [
        (lambda: lora_add(y.float(), x.float(), A.float(), B.float(), scale, plan), "bf16"),
        (lambda: lora_add(y, x, f(2, 4, 16), f(2, 24, 4), scale, plan), "multiple of 8"),
        (lambda: lora_add(y, x, f(2, 136, 16), f(2, 24, 136), scale, plan), "multiple of 8"),
        (lambda: lora_add(f(10, 20), x, A, f(2, 20, 8), scale, plan), "multiples of 8"),
        (lambda: lora_add(y, x, A, B, scale.cpu(), plan), "one device"),
        (lambda: lora_add(y, x, A, B, scale, LoraPlan(ids.cpu(), 2)), "one device"),
        (lambda: LoraPlan(ids, 5000), "at most"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


@pytest.mark.parametrize("dev", DEVICES)
def test_second_derivatives_are_refused(dev):
    y, x, A, B, scale, ids, _ = _make(10, 16, 24, 8, 2, "shuffled", dev)
    out = lora_add(y, x, A.requires_grad_(True), B, scale, LoraPlan(ids, 2))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(out.sum(), A, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("E,T", [(1, 1), (1, 5000), (3, 31), (33, 32), (1024, 70), (1000, 9001), (200, 100000)])
def test_plan_is_a_stable_sort_with_every_token_in_one_tile(E, T):
    gen = torch.Generator().manual_seed(E + T)
    for mode in ("shuffled", "holes", "one"):
        ids = _ids(T, E, mode, gen)
        p = LoraPlan(ids.cuda(), E)
        key = torch.where((ids < 0) | (ids >= E), E, ids)
        order = torch.sort(key, stable=True).indices
        assert torch.equal(p.perm.cpu().long(), order)
        counts = torch.bincount(key, minlength=E + 1)
        assert torch.equal(p.offsets.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]))
        for tiles, n, size in ((p.tiles_small, p.n_tiles[0], 16), (p.tiles_large, p.n_tiles[1], 64)):
            assert int(n) == int(((counts + size - 1) // size).sum()) <= tiles.numel() // 4
            rows = tiles.cpu().view(-1, 4)[:int(n)].long()
            starts = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])[:-1]
            want = [(a if a < E else -1, int(starts[a]) + i, min(size, int(counts[a]) - i)) for a in counts.nonzero()[:, 0].tolist() for i in range(0, int(counts[a]), size)]
            assert [tuple(t[:3]) for t in rows.tolist()] == want


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 900])
def test_captured_replayed_repeated_and_on_another_stream(T):
    K, N, r, E = 256, 192, 16, 6
    y, x, A, B, scale, ids, dout = _make(T, K, N, r, E, "holes", "cuda")

    def once():
        p = LoraPlan(ids, E)
        leaves = [x.detach().requires_grad_(True), A.detach().requires_grad_(True), B.detach().requires_grad_(True)]
        out = lora_add(y, *leaves, scale, p)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = once()
    assert all(torch.equal(a, b) for a, b in zip(once(), want))            # no atomics: the same bits every time
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    y2, x2, _, _, _, ids2, d2 = _make(T, K, N, r, E, "shuffled", "cuda", seed=5)
    for a, b in ((y, y2), (x, x2), (ids, ids2), (dout, d2)):
        a.copy_(b)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, once()))


@pytest.mark.parametrize("dev", DEVICES)
def test_a_plan_is_not_copied_and_may_be_dropped_while_another_stream_reads_it(dev):
    import copy

    y, x, A, B, scale, ids, _ = _make(4000, 64, 48, 8, 2, "shuffled", dev)
    plan = LoraPlan(ids, 2)
    for call in (copy.copy, copy.deepcopy):
        with pytest.raises(TypeError, match="from the ids"):
            call(plan)
    want = lora_add(y, x, A, B, scale, plan)
    if dev == "cpu":
        return plan.record_stream(None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [lora_add(y, x, A, B, scale, plan) for _ in range(20)]
    plan.record_stream(s)
    del plan
    junk = [torch.zeros(60000, dtype=torch.int32, device="cuda") for _ in range(4)]       # (zeros index nothing out of range)
    torch.cuda.current_stream().wait_stream(s)
    assert len(junk) == 4 and all(torch.equal(g, want) for g in got)
