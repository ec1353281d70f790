"""Low-rank adapters of many requests at once beside a shared projection: ``y[t] + s_a (x[t] A_a^T) B_a^T`` with the adapter
``a`` of token ``t``, and the gradients of ``x``, ``A`` and ``B``. CUDA tensors (bf16) go to csrc/lora.cu, CPU tensors to
torch in fp32 with the same roundings. ``train/lora.py`` merges ONE adapter into the weights instead; there rollouts keep the
trainer's bits, here a batch may hold a different adapter in every row.

An adapter bank is two tensors, ``A [E, r, K]`` and ``B [E, N, r]``, with ``scale [E]`` in fp32 (``alpha / rank``). Adapters of
different ranks share a bank when the smaller ones are filled up with zero rows of ``A`` and zero columns of ``B``
(``pad_rank``): the result does not change."""

from __future__ import annotations

import torch

from . import _native
from . import functional as F

MAX_RANK = 128
MAX_ADAPTERS = 1024         # in a bank (csrc/lora.cu::kMaxAdapters)


class LoraPlan:
    """The tokens of a batch grouped by adapter. ``ids``: integer [T], the adapter of every token; a number outside
    ``[0, num_adapters)`` means none. Built on the device in one launch without a look at the ids on the host (so a plan can
    be captured, and is built again by a replay); one plan serves every projection of every layer of the batch."""

    def __init__(self, ids: torch.Tensor, num_adapters: int):
        if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"LoraPlan: ids are a flat int32 or int64 tensor, not {tuple(ids.shape)} {ids.dtype}")
        if num_adapters < 1:
            raise ValueError("LoraPlan: at least one adapter")
        self.T, self.E, self.device, self.index = ids.shape[0], int(num_adapters), ids.device, ids.get_device()
        if not ids.is_cuda:
            self.ids = ids.clone()
            return
        L = _native.lib()
        if self.E > L.ix_lora_max_adapters():
            raise ValueError(f"LoraPlan: at most {L.ix_lora_max_adapters()} adapters in a batch, not {self.E}")
        if ids.dtype == torch.int64:                # a number that 32 bits would wrap into the range stays outside
            ids = torch.where((ids < 0) | (ids >= self.E), -1, ids)
        ids = ids.to(torch.int32).contiguous()
        small, large = (L.ix_lora_max_tiles(self.T, self.E, k) for k in (0, 1))
        buf = torch.empty(4 * small + 4 * large + self.T + self.E + 2 + 2, dtype=torch.int32, device=ids.device)
        self.tiles_small, self.tiles_large, self.perm, self.offsets, self.n_tiles = buf.split(
            [4 * small, 4 * large, self.T, self.E + 2, 2])
        # the addresses of the plan's own buffers: taken once, every call passes them
        self._apply_args = (self.perm.data_ptr(), self.tiles_small.data_ptr(), self.tiles_large.data_ptr(), self.n_tiles.data_ptr())
        self._offsets_ptr = self.offsets.data_ptr()
        with torch.cuda.device(ids.device):
            _native.check(L.ix_lora_plan(ids.data_ptr(), self.T, self.E, self._apply_args[0], self._offsets_ptr, *self._apply_args[1:],
                                         _native.stream()), "ix_lora_plan")

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream`` on the plan's buffers: for a plan that another stream than its own still reads
        when it is dropped."""
        if self.device.type == "cuda":
            self.perm.record_stream(stream)              # (all buffers are one allocation)

    def __reduce_ex__(self, protocol):
        raise TypeError("a LoraPlan is tied to its buffers on the device: build another one from the ids")


def pad_rank(A: torch.Tensor, B: torch.Tensor, rank: int) -> tuple[torch.Tensor, torch.Tensor]:
    """One adapter's ``A [r, K]`` and ``B [N, r]`` filled up with zeros to ``rank``."""
    r = A.shape[0]
    if A.dim() != 2 or B.dim() != 2 or B.shape[1] != r or rank < r:
        raise ValueError(f"pad_rank: A {tuple(A.shape)} and B {tuple(B.shape)} do not fit rank {rank}")
    return torch.nn.functional.pad(A, (0, 0, 0, rank - r)), torch.nn.functional.pad(B, (0, rank - r))


def check_bank(adapters: int, rank: int, widths, dtype: torch.dtype) -> None:
    """Refuse a bank that the kernels cannot compute with. ``widths``: (name, in, out) of every target."""
    if adapters > MAX_ADAPTERS:
        raise ValueError(f"lora: at most {MAX_ADAPTERS} adapters in a bank, not {adapters}")
    if rank % 8 or not 8 <= rank <= MAX_RANK:
        raise ValueError(f"lora: a bank's rank is a multiple of 8 up to {MAX_RANK}, not {rank}")
    if dtype != torch.bfloat16:
        raise ValueError(f"lora: on a GPU the factors are bf16, not {dtype}")
    for name, inn, out in widths:
        if inn % 8 or out % 8:
            raise ValueError(f"lora: {name} is {inn} -> {out}, widths are multiples of 8")


def _check(y, x, A, B, scale, plan) -> None:
    sa, sb, sx = A.shape, B.shape, x.shape
    if len(sa) != 3 or len(sb) != 3 or sa[0] != sb[0] or sa[1] != sb[2]:
        raise ValueError(f"lora: factors are A [E, r, K] and B [E, N, r], not {tuple(sa)} and {tuple(sb)}")
    E, r, K = sa
    N = sb[1]
    if sx[-1] != K or (y is not None and (y.shape[-1] != N or y.shape[:-1] != sx[:-1])):
        raise ValueError(f"lora: x {tuple(sx)} and y {None if y is None else tuple(y.shape)} do not fit factors of widths {K} and {N}")
    if plan.E != E or plan.T * K != x.numel():
        raise ValueError(f"lora: the plan is for {plan.T} tokens of {plan.E} adapters, x has {x.numel() // K} and the bank {E}")
    if scale.dtype != torch.float32 or scale.shape != (E,):
        raise ValueError(f"lora: scale is fp32 [{E}], not {tuple(scale.shape)} {scale.dtype}")
    if scale.requires_grad:
        raise ValueError("lora: scale is a constant, it has no gradient")
    dev, dt = plan.device, x.dtype
    if x.device != dev or A.device != dev or B.device != dev or scale.device != dev or (y is not None and y.device != dev):
        raise ValueError("lora: all tensors and the plan are on one device")
    if A.dtype != dt or B.dtype != dt or (y is not None and y.dtype != dt):
        raise ValueError("lora: x, y, A and B have one type")
    if x.is_cuda:
        if dt != torch.bfloat16:
            raise ValueError(f"lora: on a GPU the tensors are bf16, not {dt}")
        if r % 8 or r > MAX_RANK or K % 8 or N % 8:
            raise ValueError(f"lora: rank {r} (a multiple of 8 up to {MAX_RANK}: pad_rank) and widths {K}, {N} (multiples of 8)")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[T, width] with unit inner stride, rows on 16-byte boundaries."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    st = t.stride()
    if (st[1] != 1 or st[0] % 8 or t.data_ptr() % 16) and t.shape[0]:
        t = t.contiguous()
        if t.stride(0) % 8 or t.data_ptr() % 16:            # (a single row is contiguous whatever its stride says)
            t = t.clone(memory_format=torch.contiguous_format)
    return t


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _factor(t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _apply(x, base, out, down, up, scale, plan, want_h):
    """out = base + s (x down^T) up^T on prepared operands (csrc/lora.cu::ix_lora_apply); returns h [2, T, r] in the plan's order
    if wanted."""
    T, K = x.shape
    (E, r, _), N = down.shape, up.shape[1]
    h = torch.empty(2, T, r, dtype=torch.bfloat16, device=x.device) if want_h else None
    if T == 0:
        return h
    _native.check(
        _native.lib().ix_lora_apply(x.data_ptr(), x.stride(0), base.data_ptr(), base.stride(0), out.data_ptr(), out.stride(0), down.data_ptr(),
                                    up.data_ptr(), scale.data_ptr(), *plan._apply_args, None if h is None else h.data_ptr(), T, K, N, r, E, 0,
                                    _native.raw_stream(plan.index)),
        "ix_lora_apply")
    return h


def _backward_cuda(dy, x, A, B, scale, h, plan, base, need_x, need_a, need_b):
    (T, K), (E, N, r) = x.shape, B.shape
    if not need_x:
        base = dx = None
    else:
        dx = base if base is not None else torch.empty_like(x, memory_format=torch.contiguous_format)
    dA = torch.empty_like(A) if need_a else None
    dB = torch.empty_like(B) if need_b else None
    g = torch.empty(2, T, r, dtype=x.dtype, device=x.device) if need_a else None
    _native.check(
        _native.lib().ix_lora_backward(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), _native.ptr(base),
                                       base.stride(0) if base is not None else 0, _native.ptr(dx), dx.stride(0) if dx is not None else 0,
                                       A.data_ptr(), B.data_ptr(), scale.data_ptr(), *plan._apply_args, plan._offsets_ptr,
                                       _native.ptr(h) if need_b else None, _native.ptr(g), _native.ptr(dA), _native.ptr(dB), T, K, N, r, E,
                                       _native.raw_stream(plan.index)),
        "ix_lora_backward")
    return dx, dA, dB


def _cpu_h(x, A, scale, plan):
    """s (x A^T) of every token with its own adapter, fp32 [T, r]; zero rows without one."""
    h = torch.zeros(x.shape[0], A.shape[1])
    for a in range(plan.E):
        rows = (plan.ids == a).nonzero()[:, 0]
        h[rows] = scale[a] * (x[rows].float() @ A[a].float().t())
    return h


def _cpu_up(h, B, plan):
    out = torch.zeros(h.shape[0], B.shape[1])
    for a in range(plan.E):
        rows = (plan.ids == a).nonzero()[:, 0]
        out[rows] = h[rows] @ B[a].float().t()
    return out


def _cpu_grad(h, z, plan):
    return torch.stack([h[plan.ids == a].t() @ z[plan.ids == a].float() for a in range(plan.E)])


def _forward(y, x, A, B, scale, plan, inplace: bool, want_h: bool):
    """(out, h) on rows; ``inplace``: out is y."""
    if x.is_cuda:
        out = y if inplace else torch.empty_like(y, memory_format=torch.contiguous_format)
        if torch.cuda.current_device() == plan.index:        # (the usual case: no context manager in a small call)
            return out, _apply(x, y, out, A, B, scale, plan, want_h)
        with torch.cuda.device(plan.index):
            return out, _apply(x, y, out, A, B, scale, plan, want_h)
    h = _cpu_h(x, A, scale, plan)
    hit = ((plan.ids >= 0) & (plan.ids < plan.E))[:, None]
    out = torch.where(hit, (y.float() + _cpu_up(h, B, plan)).to(y.dtype), y)
    return (y.copy_(out) if inplace else out), h


def _backward(dy, x, A, B, scale, h, plan, base, need_x: bool, need_a: bool, need_b: bool):
    """(dx, dA, dB); ``base``: the other part of dx, added to in place."""
    dx = dA = dB = None
    if x.is_cuda:
        if torch.cuda.current_device() == plan.index:
            return _backward_cuda(dy, x, A, B, scale, h, plan, base, need_x, need_a, need_b)
        with torch.cuda.device(plan.index):
            return _backward_cuda(dy, x, A, B, scale, h, plan, base, need_x, need_a, need_b)
    g = _cpu_h(dy, B.transpose(1, 2), scale, plan)
    if need_x:
        dx = _cpu_up(g, A.transpose(1, 2), plan)
        dx = (dx if base is None else base.float() + dx).to(x.dtype)
    if need_a:
        dA = _cpu_grad(g, x, plan).to(A.dtype)
    if need_b:
        dB = _cpu_grad(h, dy, plan).transpose(1, 2).contiguous().to(B.dtype)
    return dx, dA, dB


def _first_order_only() -> None:
    # (what autograd's decorator for this does, without the 15 us that it costs a call)
    if torch.is_grad_enabled():
        raise RuntimeError("lora: the backward pass is not differentiable itself (create_graph=True)")


class _LoraAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, A, B, scale, plan):
        x2, A2, B2 = _rows(x), _factor(A), _factor(B)
        out, h = _forward(_rows(y), x2, A2, B2, scale, plan, False, ctx.needs_input_grad[3])
        ctx.save_for_backward(x2, A2, B2, scale, h)
        ctx.plan, ctx.xshape = plan, x.shape
        return out if y.dim() == 2 else out.view(y.shape)

    @staticmethod
    def backward(ctx, dout):
        _first_order_only()
        x, A, B, scale, h = ctx.saved_tensors
        ny, nx, na, nb = ctx.needs_input_grad[:4]
        dx, dA, dB = _backward(_rows(dout), x, A, B, scale, h, ctx.plan, None, nx, na, nb)
        return (dout if ny else None), (dx.view(ctx.xshape) if nx and len(ctx.xshape) != 2 else dx), dA, dB, None, None


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, A, B, scale, plan):
        x2, A2, B2 = _rows(x), _factor(A), _factor(B)
        out, h = _forward(F.gemm_nt(x2, w), x2, A2, B2, scale, plan, True, ctx.needs_input_grad[3])
        ctx.save_for_backward(x2, w, A2, B2, scale, h)
        ctx.plan, ctx.xshape = plan, x.shape
        return out.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dout):
        _first_order_only()
        x, w, A, B, scale, h = ctx.saved_tensors
        nx, nw, na, nb = ctx.needs_input_grad[:4]
        dy = _rows(dout)
        base = F.gemm_nn(dy, w) if nx else None
        dx, dA, dB = _backward(dy, x, A, B, scale, h, ctx.plan, base, nx, na, nb)
        dw = F.gemm_tn(dy, x) if nw else None
        return (dx.view(ctx.xshape) if nx and len(ctx.xshape) != 2 else dx), dw, dA, dB, None, None


def lora_add(y: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, scale: torch.Tensor, plan: LoraPlan) -> torch.Tensor:
    """``y + s_a (x A_a^T) B_a^T`` for every token's own adapter: x [..., K], y [..., N], A [E, r, K], B [E, N, r], scale [E].
    One rounding, of the result; a token without an adapter gets y's bits. Differentiable in y, x, A and B. An infinite x, A or
    gradient does what the formula says. An infinite number in the factor of the second product (B; A in the gradient of x) makes
    infinity or NaN on a GPU: x A^T enters there as the sum of two numbers, whose signs may differ."""
    _check(y, x, A, B, scale, plan)
    scale = _flat(scale)
    if torch.is_grad_enabled() and (A.requires_grad or B.requires_grad or x.requires_grad or y.requires_grad):
        return _LoraAdd.apply(y, x, A, B, scale, plan)
    out = _forward(_rows(y), _rows(x), _factor(A), _factor(B), scale, plan, False, False)[0]
    return out if y.dim() == 2 else out.view(y.shape)


def lora_linear(x: torch.Tensor, w: torch.Tensor, A: torch.Tensor, B: torch.Tensor, scale: torch.Tensor, plan: LoraPlan) -> torch.Tensor:
    """``F.linear(x, w)`` with the tokens' adapters added into its result in place (``lora_add`` without the second buffer).
    Differentiable in x, w, A and B; a frozen ``w`` costs no product in the backward."""
    _check(None, x, A, B, scale, plan)
    if w.dim() != 2 or w.shape != (B.shape[1], A.shape[2]) or w.dtype != x.dtype or w.device != x.device:
        raise ValueError(f"lora: w {tuple(w.shape)} {w.dtype} does not fit factors of widths {A.shape[2]} and {B.shape[1]}")
    if x.is_cuda and torch.cuda.current_device() != plan.index:      # (the projection launches on the current device)
        with torch.cuda.device(plan.index):
            return lora_linear(x, w, A, B, scale, plan)
    scale = _flat(scale)
    if torch.is_grad_enabled() and (A.requires_grad or B.requires_grad or x.requires_grad or w.requires_grad):
        return _LoraLinear.apply(x, w, A, B, scale, plan)
    x2 = _rows(x)
    return _forward(F.gemm_nt(x2, w), x2, _factor(A), _factor(B), scale, plan, True, False)[0].view(*x.shape[:-1], w.shape[0])
