"""One token per row of logits from one given random number per row, each row with its own temperature, top-k, top-p and
min-p. CUDA rows go to csrc/sample_rows.cu (no sort, no host synchronisation), CPU rows to the sorted form in torch.

The tokens of a row are ordered by logit, largest first, and by index where logits are equal; token i weighs
``exp((x_i - max x) / temperature)``. Kept are the first ``top_k``; of these those that weigh at least ``min_p`` (of the
heaviest, which weighs 1); of these those in front of which less than ``top_p`` of the whole kept weight stands, the first
token always. The token drawn is the one in whose stretch of the kept weight ``u`` falls, so a row's outcome is a function of
its own logits, settings and number alone: not of the batch, the stream or the number of calls before it."""

from __future__ import annotations

import torch

from . import _native

MAX_VOCAB = 1 << 19         # tokens of a row on a GPU (csrc/sample_rows.cu::ix_sample_rows_max_vocab)


def _setting(t, name, rows, dtype, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.shape != (rows,) or t.dtype != dtype or t.device != device:
        raise ValueError(f"sample_rows: {name} is None or {str(dtype)[6:]} [{rows}] on the logits' device")
    return t if t.is_contiguous() else t.contiguous()


def sample_rows(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
                top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens int64 [rows], log-probabilities fp32 [rows]).

    ``logits`` [rows, V] bf16 or fp32 (on a GPU V is at most ``MAX_VOCAB``); ``u`` fp32 [rows] in ``[0, 1)`` (a number outside is moved to the nearer end, NaN to 0). ``temperature`` fp32 (default
    1; at or below 0: the largest logit), ``top_k`` int32 (at or below 0: off), ``top_p`` fp32 (1 or more: off), ``min_p`` fp32 (at
    or below 0: off), each [rows] or None. A logit of -inf or NaN is never drawn; a row that has no other gives token 0 with
    log-probability -inf. The log-probability is that of the token in the kept, renormalised distribution, the one it was
    drawn from (0 for a greedy row), not that of the raw logits (``functional.token_logprobs``)."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"sample_rows: logits are bf16 or fp32 [rows, V], not {tuple(logits.shape)} {logits.dtype}")
    rows, V = logits.shape
    if V < 1:
        raise ValueError("sample_rows: an empty vocabulary")
    dev = logits.device
    if u is None:
        raise ValueError("sample_rows: one number u per row is needed")
    u = _setting(u, "u", rows, torch.float32, dev)
    temperature = _setting(temperature, "temperature", rows, torch.float32, dev)
    top_k = _setting(top_k, "top_k", rows, torch.int32, dev)
    top_p = _setting(top_p, "top_p", rows, torch.float32, dev)
    min_p = _setting(min_p, "min_p", rows, torch.float32, dev)
    if logits.requires_grad:
        logits = logits.detach()
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if not logits.is_cuda:
        return _sample_cpu(logits, u, temperature, top_k, top_p, min_p)
    if torch.cuda.current_device() != logits.get_device():
        with torch.cuda.device(dev):
            return _sample_cuda(logits, u, temperature, top_k, top_p, min_p)
    return _sample_cuda(logits, u, temperature, top_k, top_p, min_p)


def _sample_cuda(logits, u, temperature, top_k, top_p, min_p):
    rows, V = logits.shape
    L = _native.lib()
    if V > MAX_VOCAB:
        raise ValueError(f"sample_rows: a vocabulary of at most {MAX_VOCAB}, not {V}")
    tokens = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    bf16 = logits.dtype == torch.bfloat16
    marked = torch.empty(rows, dtype=torch.int32, device=logits.device) if bf16 else None
    esize, ld = logits.element_size(), logits.stride(0)
    settings = (u, temperature, top_k, top_p, min_p)
    for lo in range(0, rows, 65535):                      # one launch's limit of rows
        n, at = min(65535, rows - lo), lambda t: None if t is None else t.data_ptr() + lo * t.element_size()  # noqa: B023
        _native.check(L.ix_sample_rows(logits.data_ptr() + lo * ld * esize, ld, n, V, int(not bf16), *(at(t) for t in settings), at(tokens),
                                       at(logprobs), at(marked), _native.raw_stream(logits.get_device())), "ix_sample_rows")
    return tokens, logprobs


def _sample_cpu(logits, u, temperature, top_k, top_p, min_p):
    rows, V = logits.shape
    one, off = torch.ones(rows), torch.zeros(rows)
    x = logits.float()
    x = torch.where(x.isnan(), float("-inf"), x) + 0.0
    u = u.nan_to_num(0.0).clamp(0.0, 1.0 - 2.0 ** -24)
    vals, order = torch.sort(x, dim=-1, descending=True, stable=True)
    vals = vals.double()
    top = vals[:, :1]
    t = (one if temperature is None else temperature).double()[:, None]
    w = torch.exp((vals - top) / torch.where(t > 0, t, 1.0))
    w = torch.where(vals == top, 1.0, torch.where(top.isposinf() | vals.isneginf(), 0.0, w))      # (also where T is infinite)
    place = torch.arange(V)[None, :]
    if top_k is not None:
        k = top_k.long()[:, None]
        w = torch.where((place < k) | (k <= 0), w, 0.0)
    m = (off if min_p is None else min_p).double()[:, None]
    w = torch.where((w >= m) | ~(m > 0) | (place == 0), w, 0.0)
    c = w.cumsum(-1)
    p = (one if top_p is None else top_p).double()[:, None]
    w = torch.where((c - w < p * c[:, -1:]) | ~(p < 1) | (place == 0), w, 0.0)
    c = w.cumsum(-1)
    at = (c <= u.double()[:, None] * c[:, -1:]).sum(-1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(-1, keepdim=True) - 1)
    greedy, nothing = ~(t > 0), torch.isneginf(top)
    at = torch.where(greedy, 0, at)
    lp = torch.where(greedy, 0.0, torch.log(w.gather(1, at) / c[:, -1:]))
    tokens = torch.where(nothing, 0, order.gather(1, at))
    return tokens[:, 0], torch.where(nothing, float("-inf"), lp)[:, 0].float()
