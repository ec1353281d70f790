"""AdamW over many tensors at once: the factors of an adapter, or any list of weights that is not one flat buffer (for that
one there is ``train/policy_worker.FlatAdamW``). One launch of csrc/tensor_adamw.cu steps all of them; CPU tensors take the
same formulas in torch, rounded in the same places."""

from __future__ import annotations

import struct

import torch

from . import _native

BLOCK = 256             # elements that share one scale of an 8-bit state
FP8 = torch.float8_e4m3fn


def _encode(v: torch.Tensor, root: bool):
    """(e4m3 codes, fp32 scale per ``BLOCK``) of a flat tensor of whole blocks; ``root``: a positive value keeps a positive code."""
    s = v.view(-1, BLOCK).abs().amax(-1) * (1.0 / 448.0)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    each = s.repeat_interleave(BLOCK)
    q = torch.where(each > 0, v / torch.where(each > 0, each, torch.ones_like(each)), torch.zeros_like(v))
    if root:
        q = torch.where(q > 0, q.clamp(min=2.0 ** -9), q)
    return q.clamp(-448.0, 448.0).to(FP8), s


class TensorAdamW:
    """AdamW with decoupled weight decay over a list of contiguous tensors of one type (fp32, or bf16 with fp32 masters kept
    here) on one device.

    Gradients are read from ``grads``, one buffer per parameter that the program fills again for every step (autograd, a
    projection, ``F.gemm_tn(out=...)``); without the argument they are made here, fp32 zeros in one allocation
    (``zero_grad`` clears them). The memory of parameters and gradients is fixed at construction (and kept alive): a step does
    no per-tensor work on the host, and does not see a ``p.data`` or an entry of ``params``, ``grads`` or ``state`` that was replaced.

    ``state_bits=8``: both moments in e4m3 with one scale per 256 elements, the second by its square root, 2 bytes and a bit
    per element instead of 8. ``state`` holds flat buffers in which tensor ``i`` starts at ``offsets[i]`` (a multiple of
    256): ``exp_avg``, ``exp_avg_sq``, with 8 bits ``exp_avg_scale`` and ``exp_avg_sq_scale``, with bf16 parameters
    ``master``. What stands between two sections stays zero.

    A step cannot be captured into a CUDA graph: its bias corrections are numbers of the host's step count."""

    def __init__(self, params, grads=None, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.0, state_bits: int = 32):
        params = list(params)
        if not params:
            raise ValueError("TensorAdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"TensorAdamW: state_bits must be 32 or 8, not {state_bits!r}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps > 0.0:
            raise ValueError(f"TensorAdamW: betas {betas} / eps {eps} out of range")
        decay = [float(weight_decay)] * len(params) if not hasattr(weight_decay, "__len__") else [float(w) for w in weight_decay]
        if len(decay) != len(params):
            raise ValueError(f"TensorAdamW: {len(decay)} weight decays for {len(params)} parameters")
        dev, dt = params[0].device, params[0].dtype          # (a tensor's device always carries its index)
        if dt not in (torch.float32, torch.bfloat16):
            raise ValueError(f"TensorAdamW: parameters are fp32 or bf16, not {dt}")
        self.device, self.lr, self.betas, self.eps, self._decay, self.state_bits = dev, lr, tuple(betas), eps, tuple(decay), state_bits
        self.params = params
        self.offsets, total = [], 0
        for p in params:
            self.offsets.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        self._own_grad = None
        if grads is None:
            self._own_grad = torch.zeros(total, dtype=torch.float32, device=dev)
            grads = [self._own_grad[o:o + p.numel()].view(p.shape) for o, p in zip(self.offsets, params)]
        self.grads = list(grads)
        if len(self.grads) != len(params):
            raise ValueError(f"TensorAdamW: {len(self.grads)} gradients for {len(params)} parameters")
        for p, g in zip(params, self.grads):
            if p.device != dev or g.device != dev or p.dtype != dt or g.dtype != self.grads[0].dtype:
                raise ValueError("TensorAdamW: parameters share one type and one device, and so do gradients")
            if p.shape != g.shape or not p.is_contiguous() or not g.is_contiguous():
                raise ValueError("TensorAdamW: parameters and gradients are contiguous and of the same shape")
        if self.grads[0].dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"TensorAdamW: gradients are fp32 or bf16, not {self.grads[0].dtype}")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("TensorAdamW: two of the parameters share memory")
        # what a step writes and reads: stays allocated, and is what it was at construction on either device
        self._params, self._grads = [p.detach() for p in params], [g.detach() for g in self.grads]
        self._memory = [*self._params, *self._grads]
        self.step_count = 0
        st = FP8 if state_bits == 8 else torch.float32
        self.state = {"exp_avg": torch.zeros(total, dtype=st, device=dev), "exp_avg_sq": torch.zeros(total, dtype=st, device=dev)}
        if state_bits == 8:
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                self.state[k] = torch.zeros(total // BLOCK, dtype=torch.float32, device=dev)
        if dt == torch.bfloat16:
            self.state["master"] = torch.zeros(total, dtype=torch.float32, device=dev)
            for p, o in zip(self._params, self.offsets):
                self.state["master"][o:o + p.numel()].copy_(p.reshape(-1))
        self._buffers = dict(self.state)
        self._memory += self.state.values()
        if dev.type == "cuda":
            self._tables()

    def __reduce_ex__(self, protocol):
        raise TypeError("TensorAdamW is tied to the memory of its parameters: build another one and pass state_dict() on")

    @property
    def weight_decay(self) -> tuple:
        """Per parameter. Fixed at construction (it stands in the table on the device); ``lr``, ``betas`` and ``eps`` may be set."""
        return self._decay

    def _tables(self) -> None:
        chunk = _native.lib().ix_tensor_adamw_chunk()
        rows = bytearray()
        for p, g, off, wd in zip(self._params, self._grads, self.offsets, self._decay):
            vec = int(p.data_ptr() % 16 == 0 and g.data_ptr() % 16 == 0)
            rows += struct.pack("<QQqqfi24x", p.data_ptr(), g.data_ptr(), p.numel(), off, wd, vec)
        n = torch.tensor([-(-p.numel() // chunk) for p in self.params])
        tensor = torch.repeat_interleave(torch.arange(len(self.params)), n)
        piece = torch.arange(len(tensor)) - (n.cumsum(0) - n)[tensor]
        self._table = torch.frombuffer(rows, dtype=torch.uint8).to(self.device)
        self._chunks = torch.stack([tensor, piece], 1).to(torch.int32).to(self.device)
        st = self._buffers
        # everything a step passes that does not change: the buffers are this object's own
        self._args = (self._table.data_ptr(), self._chunks.data_ptr(), len(tensor), int(self.params[0].dtype == torch.float32),
                      int(self.grads[0].dtype == torch.float32), int(self.state_bits == 8), _native.ptr(st.get("master")), st["exp_avg"].data_ptr(),
                      st["exp_avg_sq"].data_ptr(), _native.ptr(st.get("exp_avg_scale")), _native.ptr(st.get("exp_avg_sq_scale")))

    @torch.no_grad()
    def refresh_masters(self) -> None:
        """Take the masters from the bf16 parameters again where these are no longer the masters' rounding (after weights were
        loaded, or one adapter's factors put into a bank): the next step would write the old ones back. Others keep their bits."""
        if "master" in self._buffers:
            for p, o in zip(self._params, self.offsets):
                m, now = self._buffers["master"][o:o + p.numel()], p.reshape(-1)
                changed = m.to(torch.bfloat16).view(torch.int16) != now.view(torch.int16)
                m.copy_(torch.where(changed, now.float(), m))

    @torch.no_grad()
    def zero_grad(self) -> None:
        if self._own_grad is not None:
            self._own_grad.zero_()
        else:
            torch._foreach_zero_(self._grads)

    @torch.no_grad()
    def step(self, lr: float | None = None, grad_scale: torch.Tensor | None = None) -> None:
        """One step with ``lr`` (default: the constructor's). ``grad_scale``: a device scalar multiplied into every gradient
        (a clip coefficient); nothing is read back. A gradient that is not finite goes into its own element's moments, and
        with 8-bit states into the 256 elements of its scale: the caller skips such a step."""
        lr = self.lr if lr is None else float(lr)
        if grad_scale is not None and (grad_scale.device != self.device or grad_scale.dtype != torch.float32 or grad_scale.numel() != 1):
            raise ValueError("TensorAdamW: grad_scale is one fp32 number on the parameters' device")
        if self.device.type != "cuda":
            self.step_count += 1
            return self._step_cpu(lr, grad_scale)
        if torch.cuda.current_device() == self.device.index:
            self._step_cuda(lr, grad_scale)
        else:
            with torch.cuda.device(self.device):
                self._step_cuda(lr, grad_scale)

    def _step_cuda(self, lr, grad_scale) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("TensorAdamW.step cannot be captured into a graph: its bias corrections follow the host's step count")
        self.step_count += 1
        _native.check(_native.lib().ix_tensor_adamw(*self._args, _native.ptr(grad_scale), lr, self.betas[0], self.betas[1], self.eps,
                                                    self.step_count, _native.raw_stream(self.device.index)), "ix_tensor_adamw")
        torch.autograd.graph.increment_version(self.params)

    def _step_cpu(self, lr, grad_scale) -> None:
        b1, b2 = self.betas
        st, t = self._buffers, self.step_count
        for i, (p, g, o) in enumerate(zip(self._params, self._grads, self.offsets)):
            n = p.numel()
            e = o + -(-n // BLOCK) * BLOCK
            x = torch.nn.functional.pad(g.reshape(-1).float(), (0, e - o - n))
            if grad_scale is not None:
                x = x * grad_scale
            m, v = st["exp_avg"][o:e].float(), st["exp_avg_sq"][o:e].float()
            if self.state_bits == 8:
                m = m * st["exp_avg_scale"][o // BLOCK:e // BLOCK].repeat_interleave(BLOCK)
                v = (v * st["exp_avg_sq_scale"][o // BLOCK:e // BLOCK].repeat_interleave(BLOCK)).square()
            m = b1 * m + (1 - b1) * x
            v = b2 * v + (1 - b2) * x * x
            master = st["master"][o:o + n] if "master" in st else p.view(-1)
            upd = lr / (1 - b1 ** t) * m[:n] / (v[:n].sqrt() / (1 - b2 ** t) ** 0.5 + self.eps)
            master.copy_(master * (1 - lr * self._decay[i]) - upd)
            if "master" in st:
                p.view(-1).copy_(master)
            if self.state_bits == 8:
                for k, y, root in (("exp_avg", m, False), ("exp_avg_sq", v.sqrt(), True)):
                    st[k][o:e], st[k + "_scale"][o // BLOCK:e // BLOCK] = _encode(y, root)
            else:
                st["exp_avg"][o:e], st["exp_avg_sq"][o:e] = m, v

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(mean, second moment) of parameter ``i`` in fp32, decoded."""
        o, n, st = self.offsets[i], self._params[i].numel(), self._buffers
        m, v = st["exp_avg"][o:o + n].float(), st["exp_avg_sq"][o:o + n].float()
        if self.state_bits == 8:
            per = torch.arange(o, o + n, device=m.device) // BLOCK
            m, v = m * st["exp_avg_scale"][per], (v * st["exp_avg_sq_scale"][per]).square()
        return m.view(self._params[i].shape), v.view(self._params[i].shape)

    def _shapes(self) -> list:
        return [tuple(p.shape) for p in self._params]

    def state_dict(self) -> dict:
        return {"step": self.step_count, "shapes": self._shapes(), **{k: v.clone() for k, v in self._buffers.items()}}

    @torch.no_grad()
    def load_state_dict(self, sd: dict) -> None:
        """Take a ``state_dict()`` of the same tensors in the same order. (``shapes`` says which they were; a state that was
        put together elsewhere may come without, its buffers laid out by ``offsets``.)"""
        sd = dict(sd)
        if "step" not in sd:
            raise ValueError("TensorAdamW: not a state of this optimizer (no step count)")
        step, shapes = int(sd.pop("step")), sd.pop("shapes", None)
        if set(sd) != set(self._buffers):
            raise ValueError(f"TensorAdamW: state has {sorted(sd)}, this optimizer {sorted(self._buffers)}")
        for k, v in sd.items():
            if v.shape != self._buffers[k].shape or v.dtype != self._buffers[k].dtype:
                raise ValueError(f"TensorAdamW: {k} is {tuple(v.shape)} {v.dtype}, expected {tuple(self._buffers[k].shape)} {self._buffers[k].dtype}")
        if shapes is not None and [tuple(x) for x in shapes] != self._shapes():
            at = next((i for i, (a, b) in enumerate(zip(shapes, self._shapes())) if tuple(a) != b), min(len(shapes), len(self.params)))
            raise ValueError(f"TensorAdamW: the state is of {len(shapes)} tensors, this optimizer has {len(self.params)}, and they differ from number {at} on")
        for k, v in sd.items():
            self._buffers[k].copy_(v)
        self.step_count = step
