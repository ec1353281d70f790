"""LoRA adapters over the flat-parameter model and a multi-tenant adapter store (reference:
B/workers/megatron/adapter_store.py multi-tenant LoRA; R/tx/layers/lora.py).

The model computes with ONE weight buffer (shared with the colocated engine), so an adapter is applied by merging
``W += (alpha / r) * B @ A`` into the target weights and removed by restoring the saved base rows exactly; the
engine needs no LoRA-aware kernel and rollouts under an adapter stay bitwise equal to the trainer's scoring.
Training an adapter: the base weights are frozen; the dense weight gradient dW that the backward already
produces is projected onto the factors, dA = (alpha/r) * B^T dW, dB = (alpha/r) * dW A^T, and only A, B step.

Several adapters at once: an ``AdapterBank`` holds their factors side by side, and a batch whose tokens use different ones
(``ForwardCtx.lora = bank.batch(...)``, ``LLMEngine.set_adapters``) adds each token's own beside the shared projections with
``ops/lora.py``, in serving and, differentiably, in training: one forward and backward over the sequences of many tenants, no
dense weight gradient.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

DEFAULT_TARGETS = ("attn.qkv.weight", "attn.q_b.weight", "attn.kv_b.weight", "attn.o.weight", "mlp.gate_up.weight", "mlp.down.weight")


@dataclass
class LoRAConfig:
    rank: int = 8
    alpha: float = 16.0
    targets: tuple = DEFAULT_TARGETS
    lr: float = 1e-4
    seed: int = 0
    optimizer: str = "adam"     # "adam": torch's; "fused" / "fused8": ops/optim.TensorAdamW, one launch for all factors, moments in 32 or 8 bits


@dataclass
class LoRAAdapter:
    cfg: LoRAConfig
    A: dict = field(default_factory=dict)     # name -> [r, in]   (fp32)
    B: dict = field(default_factory=dict)     # name -> [out, r]  (fp32, zeros at init: the adapter starts as a no-op)

    @property
    def scale(self) -> float:
        return self.cfg.alpha / self.cfg.rank

    @staticmethod
    def init(model, cfg: LoRAConfig) -> "LoRAAdapter":
        ad = LoRAAdapter(cfg)
        g = torch.Generator().manual_seed(cfg.seed)
        for name, w in model.named_weights():
            if w.dim() == 2 and name.endswith(tuple(cfg.targets)):
                out, inn = w.shape
                ad.A[name] = (torch.randn(cfg.rank, inn, generator=g) / math.sqrt(inn)).to(w.device)
                ad.B[name] = torch.zeros(out, cfg.rank, device=w.device)
        if not ad.A:
            raise ValueError(f"no parameter matches the LoRA targets {cfg.targets}")
        return ad

    def delta(self, name: str) -> torch.Tensor:
        return self.scale * (self.B[name] @ self.A[name])

    def num_parameters(self) -> int:
        return sum(a.numel() + b.numel() for a, b in zip(self.A.values(), self.B.values()))

    def state_dict(self) -> dict:
        return {"cfg": vars(self.cfg), "A": {k: v.cpu() for k, v in self.A.items()}, "B": {k: v.cpu() for k, v in self.B.items()}}

    @staticmethod
    def from_state_dict(sd: dict, device="cpu") -> "LoRAAdapter":
        ad = LoRAAdapter(LoRAConfig(**{**sd["cfg"], "targets": tuple(sd["cfg"]["targets"])}))
        ad.A = {k: v.to(device) for k, v in sd["A"].items()}
        ad.B = {k: v.to(device) for k, v in sd["B"].items()}
        return ad


class AdapterStore:
    """Named adapters for one base model; at most one is merged into the weights at a time."""

    def __init__(self, model):
        self.model = model
        self.adapters: dict[str, LoRAAdapter] = {}
        self.active: str | None = None
        self._base: dict[str, torch.Tensor] = {}

    def register(self, tenant: str, adapter: LoRAAdapter) -> None:
        if tenant in self.adapters:
            raise ValueError(f"adapter {tenant!r} already registered")
        self.adapters[tenant] = adapter

    def remove(self, tenant: str) -> None:
        if self.active == tenant:
            self.deactivate()
        del self.adapters[tenant]

    @torch.no_grad()
    def activate(self, tenant: str) -> None:
        """Merge ``tenant``'s delta into the model weights (after un-merging whichever adapter was active)."""
        if self.active == tenant:
            return
        self.deactivate()
        ad = self.adapters[tenant]
        views = dict(self.model.named_weights())
        for name in ad.A:
            w = views[name]
            self._base[name] = w.detach().clone()
            w.copy_((w.float() + ad.delta(name).to(w.device)).to(w.dtype))
        self.active = tenant

    @torch.no_grad()
    def deactivate(self) -> None:
        """Restore the base weights bit for bit."""
        if self.active is None:
            return
        views = dict(self.model.named_weights())
        for name, base in self._base.items():
            views[name].copy_(base)
        self._base.clear()
        self.active = None

    @torch.no_grad()
    def refresh(self) -> None:
        """Re-merge the active adapter after its factors changed (an optimizer step)."""
        t = self.active
        if t is not None:
            self.deactivate()
            self.activate(t)


class AdapterBank:
    """The factors of several adapters side by side, per target weight ``A [E, r, in]`` and ``B [E, out, r]`` in the model's type:
    ``r`` is the largest rank, rounded up to a multiple of 8, smaller adapters are filled up with zeros, and an adapter without
    a target has zeros there. ``trainable``: the factors take gradients (``parameters()``), in their own type like any
    parameter; bf16 ones are summed over micro-batches in bf16."""

    def __init__(self, model, adapters: dict[str, LoRAAdapter], trainable: bool = False):
        if not adapters:
            raise ValueError("AdapterBank: no adapters")
        views = dict(model.named_weights())
        self.names = list(adapters)
        self.cfgs = [ad.cfg for ad in adapters.values()]
        self.rank = max(-(-c.rank // 8) * 8 for c in self.cfgs)
        dev = model.store.flat.device
        self.scales = [ad.scale for ad in adapters.values()]
        self.scale = torch.tensor(self.scales, dtype=torch.float32, device=dev)
        self.A: dict[str, torch.Tensor] = {}
        self.B: dict[str, torch.Tensor] = {}
        targets = [n for n in views if any(n in ad.A for ad in adapters.values())]
        if dev.type == "cuda":               # refused here, not in the middle of an engine's step
            from ..ops.lora import check_bank

            check_bank(len(adapters), self.rank, [(t, *reversed(views[t].shape)) for t in targets], model.store.flat.dtype)
        for t in targets:
            out, inn = views[t].shape
            self.A[t] = torch.zeros(len(adapters), self.rank, inn, dtype=views[t].dtype, device=dev)
            self.B[t] = torch.zeros(len(adapters), out, self.rank, dtype=views[t].dtype, device=dev)
        for name, ad in adapters.items():
            missing = [t for t in ad.A if t not in self.A]
            if missing:
                raise ValueError(f"AdapterBank: the model has no weight {missing[0]!r} that adapter {name!r} was made for")
            merged_only = [t for t in ad.A if not t.endswith(DEFAULT_TARGETS)]
            if merged_only:
                raise ValueError(f"AdapterBank: adapter {name!r} has factors of {merged_only[0]!r}; beside the projections only "
                                 f"{', '.join(DEFAULT_TARGETS)} are computed (AdapterStore merges any weight)")
            self.put(name, ad)
        for t in self.parameters():
            t.requires_grad_(trainable)

    @torch.no_grad()
    def put(self, name: str, ad: LoRAAdapter) -> None:
        """Take the factors of ``ad`` again (after it stepped on its own) in the place of adapter ``name``. An optimizer that steps
        this bank's factors and keeps masters of them (``TensorAdamW`` on bf16) has to take them, too: ``refresh_masters()``;
        its moments of ``name`` are still those of the factors before."""
        e, r = self.names.index(name), ad.cfg.rank
        if r > self.rank or ad.scale != self.scales[e]:
            raise ValueError(f"AdapterBank: {name!r} changed its rank or scale; build a new bank")
        if any(t not in self.A for t in ad.A):
            raise ValueError(f"AdapterBank: {name!r} has new targets; build a new bank")
        self.cfgs[e] = ad.cfg                                    # (its rank may be another one, under the same scale)
        for t in self.A:
            self.A[t][e].zero_()
            self.B[t][e].zero_()
            if t in ad.A:
                self.A[t][e, :r].copy_(ad.A[t])
                self.B[t][e, :, :r].copy_(ad.B[t])

    def adapter(self, name: str) -> LoRAAdapter:
        """The factors of one adapter at its own rank: what the bank holds, in fp32 (rounded to the model's type where that is
        bf16; an optimizer's fp32 masters stay with the optimizer)."""
        e = self.names.index(name)
        r = self.cfgs[e].rank
        ad = LoRAAdapter(self.cfgs[e])
        for t in self.A:
            if t.endswith(tuple(ad.cfg.targets)):
                ad.A[t], ad.B[t] = self.A[t][e, :r].detach().float().clone(), self.B[t][e, :, :r].detach().float().contiguous().clone()
        return ad

    def parameters(self) -> list[torch.Tensor]:
        return [t for pair in zip(self.A.values(), self.B.values()) for t in pair]

    def batch(self, ids) -> "LoraBatch":
        """The adapters of a batch's tokens for ``ForwardCtx.lora``. ``ids``: a device tensor of places (negative: none), or a
        list of names and None, one per token."""
        if not isinstance(ids, torch.Tensor):
            ids = torch.tensor([-1 if n is None else self.names.index(n) for n in ids], dtype=torch.int32, device=self.scale.device)
        return LoraBatch(self, ids)


class LoraBatch:
    """One batch's tokens grouped by adapter (``ops/lora.LoraPlan``, built once) with the bank they compute with."""

    def __init__(self, bank: AdapterBank, ids: torch.Tensor):
        from ..ops import lora as ops

        self._ops, self.bank, self.plan = ops, bank, ops.LoraPlan(ids, len(bank.names))

    def __contains__(self, target: str) -> bool:
        return target in self.bank.A

    def linear(self, x, w, target: str):
        return self._ops.lora_linear(x, w, self.bank.A[target], self.bank.B[target], self.bank.scale, self.plan)

    def add(self, y, x, target: str):
        return self._ops.lora_add(y, x, self.bank.A[target], self.bank.B[target], self.bank.scale, self.plan)


class LoRATrainer:
    """Adam on the factors of one adapter, fed by the dense main gradients of a ``PolicyWorker``."""

    def __init__(self, worker, store: AdapterStore, tenant: str):
        self.worker, self.store, self.tenant = worker, store, tenant
        self.ad = store.adapters[tenant]
        params = []
        for name in self.ad.A:
            self.ad.A[name].requires_grad_(False)
            self.ad.B[name].requires_grad_(False)
            params += [self.ad.A[name], self.ad.B[name]]
        if self.ad.cfg.optimizer == "adam":
            self.opt = torch.optim.Adam(params, lr=self.ad.cfg.lr)
        elif self.ad.cfg.optimizer in ("fused", "fused8"):
            from ..ops.optim import TensorAdamW

            self.opt = TensorAdamW(params, lr=self.ad.cfg.lr, state_bits=8 if self.ad.cfg.optimizer == "fused8" else 32)
            for p, g in zip(params, self.opt.grads):
                p.grad = g
        else:
            raise ValueError(f"LoRAConfig.optimizer is 'adam', 'fused' or 'fused8', not {self.ad.cfg.optimizer!r}")

    def set_lr(self, lr: float) -> None:
        if isinstance(self.opt, torch.optim.Optimizer):
            for group in self.opt.param_groups:
                group["lr"] = float(lr)
        else:
            self.opt.lr = float(lr)

    @torch.no_grad()
    def optim_step(self) -> float:
        """Project the accumulated dense gradients onto (A, B), step them, re-merge; the base weights never move."""
        model, opt = self.worker.model, self.worker.opt
        sq = 0.0
        for name in self.ad.A:
            s = model.store.specs[name]
            n = 1
            for d in s.shape:
                n *= d
            dW = opt.main_grad[s.offset:s.offset + n].view(s.shape).float()
            A, B = self.ad.A[name], self.ad.B[name]
            if isinstance(self.opt, torch.optim.Optimizer):
                A.grad = self.ad.scale * (B.t() @ dW)
                B.grad = self.ad.scale * (dW @ A.t())
            else:                                  # into the optimizer's own buffers
                torch.mul(B.t() @ dW, self.ad.scale, out=A.grad)
                torch.mul(dW @ A.t(), self.ad.scale, out=B.grad)
            sq += float(A.grad.square().sum() + B.grad.square().sum())
        self.opt.step()
        opt.zero_grad()
        self.store.refresh()
        return math.sqrt(sq)
