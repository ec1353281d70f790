"""Operators of a service that many tenants share, each with a low-rank adapter of its own, as cases to measure:

* ``lora``    the adapters of many requests beside a shared projection: ``out[t] = y[t] + s[a] * (x[t] A[a]^T) B[a]^T`` with
              ``a = ids[t]`` (negative: no adapter), and the gradients of ``x``, ``A`` and ``B``;
* ``sample``  one token per row of logits from one given random number per row, with a temperature, top-k, top-p and min-p of
              the row's own, and the token's log-probability under the distribution that it was drawn from;
* ``adamw``   one AdamW step over many tensors at once, with the two moments in 32 bits or in 8.

``own`` false: the plain forms (elementary torch operations). ``own`` true: the calls of this package."""

from __future__ import annotations

import torch

own = False
BLOCK = 256                 # elements that share a scale of an 8-bit state; every tensor's section of a flat buffer starts at a multiple of it
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.95, 1e-8, 0.05, 3e-4


def listed():
    return [
        # one token of one request with an adapter: the latency of a decode step's projection (2048-wide model, small rank)
        dict(name="lora one token", op="lora", train=False, tokens=1, k=2048, n=4096, rank=8, adapters=4, base=0.0),
        # a decode batch of 48 requests over 32 adapters, a few without: fused q|k|v of a 4096-wide model
        dict(name="lora decode 48", op="lora", train=False, tokens=48, k=4096, n=6144, rank=16, adapters=32, base=0.1),
        # chunked prefill of a few requests, ragged, large rank: the output projection
        dict(name="lora prefill 4093", op="lora", train=False, tokens=4093, k=4096, n=4096, rank=64, adapters=5, base=0.2),
        # a training micro-batch of several tenants with ragged shares: gradients of every adapter
        dict(name="lora train 6 tenants", op="lora", train=True, tokens=2777, k=2560, n=9216, rank=8, adapters=6, base=0.0),
        # a training micro-batch of one tenant: gate|up of a 4096-wide model
        dict(name="lora train 8192", op="lora", train=True, tokens=8192, k=4096, n=24576, rank=16, adapters=1, base=0.0),
        # one sequence alone, usual chat settings
        dict(name="sample one row", op="sample", rows=1, vocab=151936, dtype="bfloat16", settings="chat", masked=0.0),
        # a decode batch whose requests all have settings of their own, no setting and greedy ones among them
        dict(name="sample 67 mixed", op="sample", rows=67, vocab=128256, dtype="bfloat16", settings="mixed", masked=0.0),
        # a large rollout batch, nucleus sampling
        dict(name="sample 512 top-p", op="sample", rows=512, vocab=151936, dtype="bfloat16", settings="top_p", masked=0.0),
        # logits after penalties and a grammar's mask: 32 bits, most of the vocabulary closed, a long vocabulary
        dict(name="sample 24 masked f32", op="sample", rows=24, vocab=248320, dtype="float32", settings="mixed", masked=0.97),
        # the factors of a small adapter: latency
        dict(name="adamw small adapter", op="adamw", tensors="factors", layers=2, hidden=256, inner=768, rank=8, bits=32, params="float32", grads="float32"),
        # the factors of an adapter on every projection of a 36-layer, 4096-wide model
        dict(name="adamw adapter 36 layers", op="adamw", tensors="factors", layers=36, hidden=4096, inner=12288, rank=16, bits=32, params="bfloat16", grads="float32"),
        # full weights of a 4096-wide layer, odd small tensors among them, states in 8 bits
        dict(name="adamw layer 8 bits", op="adamw", tensors="weights", layers=1, hidden=4096, inner=12288, rank=0, bits=8, params="bfloat16", grads="bfloat16"),
    ]


def _log(rng, lo, hi):
    return lo * (hi / lo) ** rng.random()


def draw(rng):
    op = rng.choice(["lora", "lora", "sample", "adamw"])
    if op == "lora":
        while True:
            c = dict(op="lora", train=rng.random() < 0.5, tokens=int(_log(rng, 1, 8192.99)), k=8 * int(_log(rng, 8, 1536)),
                     n=8 * int(_log(rng, 8, 3071)), rank=8 * rng.randint(1, 8), adapters=int(_log(rng, 1, 64.99)),
                     base=rng.choice([0.0, 0.1, 0.5]))
            if c["tokens"] * (c["k"] + c["n"]) <= 8192 * 28672 // 2:
                return c
    if op == "sample":
        while True:
            c = dict(op="sample", rows=int(_log(rng, 1, 512.99)), vocab=int(_log(rng, 1000, 262145)), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                     settings=rng.choice(["chat", "mixed", "top_p", "plain"]), masked=rng.choice([0.0, 0.0, 0.5, 0.97]))
            if c["rows"] * c["vocab"] * (2 if c["dtype"] == "float32" else 1) <= 512 * 151936:
                return c
    while True:
        c = dict(op="adamw", tensors=rng.choice(["factors", "weights"]), layers=int(_log(rng, 1, 48.99)), hidden=8 * int(_log(rng, 8, 512.99)),
                 inner=8 * int(_log(rng, 8, 1536.99)) + rng.choice([0, 0, 1, 5]), rank=rng.choice([4, 8, 13, 16, 32, 64]), bits=rng.choice([32, 8]),
                 params=rng.choice(["float32", "bfloat16"]), grads=rng.choice(["float32", "bfloat16"]))
        if _work_adamw(c)["bytes"] <= 3_000_000_000:
            return c


# ------------------------------------------------------------------------------------------------ low-rank adapters
def _prepare_lora(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, K, N, r, E = c["tokens"], c["k"], c["n"], c["rank"], c["adapters"]

    def rand(*shape, std=1.0):
        return torch.empty(*shape, device="cuda", dtype=torch.bfloat16).normal_(0.0, std, generator=g)

    # requests or tenants follow one another with ragged shares; a decode batch (few tokens for its adapters) mixes them
    cuts = torch.rand(E, generator=g, device="cuda").add(0.2)
    edge = (cuts.cumsum(0) / cuts.sum() * T).round()
    ids = torch.searchsorted(edge, torch.arange(T, device="cuda").float(), right=True).clamp(max=E - 1).to(torch.int32)
    if T < 16 * E:
        ids = ids[torch.randperm(T, generator=g, device="cuda")]
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < c["base"], -1, ids).to(torch.int32)
    s = {"op": "lora", "train": c["train"], "y": rand(T, N), "x": rand(T, K), "A": rand(E, r, K, std=K ** -0.5), "B": rand(E, N, r, std=0.3 * r ** -0.5),
         "scale": torch.rand(E, generator=g, device="cuda") + 0.5, "ids": ids}
    if c["train"]:
        s["dout"] = rand(T, N)
    if own:
        from skyrl_isoexec_b200.ops.lora import LoraPlan

        s["plan"] = LoraPlan(ids, E)            # one per batch, kept for every projection of every layer
        if c["train"]:
            for k in ("x", "A", "B"):
                s[k].requires_grad_(True)
    return s


def _run_lora(s):
    if own:
        from skyrl_isoexec_b200.ops.lora import lora_add

        out = lora_add(s["y"], s["x"], s["A"], s["B"], s["scale"], s["plan"])
        if not s["train"]:
            return {"out": out}
        dx, dA, dB = torch.autograd.grad(out, (s["x"], s["A"], s["B"]), s["dout"])
        return {"out": out.detach(), "dx": dx, "dA": dA, "dB": dB}
    # all adapters side by side: one product gives every token's coordinates in every adapter, those of its own are kept
    E, r, K = s["A"].shape
    N = s["B"].shape[1]
    x, A = s["x"].float(), s["A"].float().reshape(E * r, K)
    B = s["B"].float().transpose(0, 1).reshape(N, E * r)
    mine = s["ids"][:, None] == torch.arange(E, device=x.device, dtype=torch.int32)[None, :]
    mine = torch.where(mine, s["scale"][None, :], 0.0).repeat_interleave(r, dim=1)
    h = (x @ A.t()) * mine
    out = (s["y"].float() + h @ B.t()).to(s["y"].dtype)
    if not s["train"]:
        return {"out": out}
    dy = s["dout"].float()
    dh = (dy @ B) * mine
    return {"out": out, "dx": (dh @ A).to(s["x"].dtype), "dA": (dh.t() @ x).reshape(E, r, K).to(s["A"].dtype),
            "dB": (dy.t() @ h).reshape(N, E, r).transpose(0, 1).to(s["B"].dtype)}


def _exact_lora(c, seed):
    s = _prepare_lora(c, seed)
    E = c["adapters"]
    out = s["y"].detach().double()
    res = {"out": out}
    if c["train"]:
        res |= {"dx": torch.zeros_like(s["x"], dtype=torch.float64), "dA": torch.zeros_like(s["A"], dtype=torch.float64), "dB": torch.zeros_like(s["B"], dtype=torch.float64)}
    for a in range(E):
        rows = (s["ids"] == a).nonzero()[:, 0]
        A, B, f = s["A"][a].detach().double(), s["B"][a].detach().double(), float(s["scale"][a])
        x = s["x"].detach()[rows].double()
        h = torch.einsum("tk,rk->tr", x, A)
        out[rows] += f * torch.einsum("tr,nr->tn", h, B)
        if c["train"]:
            dy = s["dout"][rows].double()
            dh = f * torch.einsum("tn,nr->tr", dy, B)
            res["dx"][rows] = torch.einsum("tr,rk->tk", dh, A)
            res["dA"][a] = torch.einsum("tr,tk->rk", dh, x)
            res["dB"][a] = f * torch.einsum("tn,tr->nr", dy, h)
    return res


def _work_lora(c):
    T, K, N, r, E = c["tokens"], c["k"], c["n"], c["rank"], c["adapters"]
    used = min(E, T)
    factors = 2 * used * r * (K + N)
    w = {"bytes": 2 * T * (K + 2 * N) + factors + 4 * T, "flops": 2 * T * r * (K + N)}
    if c["train"]:                       # backward: dout read, x again, dx written; the factors' gradients written
        w["bytes"] += 2 * T * (N + 2 * K) + factors + 2 * E * r * (K + N)
        w["flops"] += 4 * T * r * (K + N)
    return w


# ------------------------------------------------------------------------------------------------ sampling
def _prepare_sample(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, V = c["rows"], c["vocab"]

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    x = torch.empty(n, V, device="cuda").normal_(0.0, 2.0, generator=g)
    x += 6.0 * (rand(n, V) < 20.0 / V)                                        # a few likely tokens in every row
    if c["masked"]:
        x.masked_fill_(rand(n, V) < c["masked"], float("-inf"))
    x = x.to(getattr(torch, c["dtype"]))
    one = torch.ones(n, device="cuda")
    off = torch.zeros(n, device="cuda", dtype=torch.int32)
    s = {"op": "sample", "logits": x, "u": rand(n), "temperature": one, "top_k": off, "top_p": one, "min_p": 0 * one}
    if c["settings"] == "chat":
        s |= {"temperature": 0.6 * one, "top_k": off + 20, "top_p": 0.95 * one}
    elif c["settings"] == "top_p":
        s |= {"top_p": 0.9 * one}
    elif c["settings"] == "mixed":
        pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(len(values), (n,), generator=g, device="cuda")]  # noqa: E731
        s |= {"temperature": pick([0.0, 0.3, 0.7, 1.0, 1.5]), "top_k": pick([0, 0, 1, 40, 200, 5000]).to(torch.int32), "top_p": pick([1.0, 0.99, 0.9, 0.5]),
              "min_p": pick([0.0, 0.0, 0.02, 0.1])}
    return s


def _run_sample(s):
    if own:
        from skyrl_isoexec_b200.ops.sampling import sample_rows

        tokens, logprobs = sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    # order: logit descending, then index ascending. A sum over a whole vocabulary decides which token a number falls on, so
    # weights and sums are held in 64 bits.
    x = s["logits"].float()
    V = x.shape[1]
    x = torch.where(x.isnan(), float("-inf"), x) + 0.0
    vals, order = torch.sort(x, dim=-1, descending=True, stable=True)
    del x
    top = vals[:, :1]
    t = s["temperature"].double()[:, None]
    w = torch.where(vals == top, 1.0, torch.exp((vals.double() - top.double()) / torch.where(t > 0, t, 1.0)))
    rank = torch.arange(V, device=w.device)[None, :]
    k = s["top_k"].long()[:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    mp = s["min_p"].double()[:, None]
    w = torch.where((w >= mp) | ~(mp > 0), w, 0.0)
    c = w.cumsum(-1)
    p = s["top_p"].double()[:, None]
    w = torch.where((c - w < p * c[:, -1:]) | ~(p < 1) | (rank == 0), w, 0.0)
    c = w.cumsum(-1)
    at = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(-1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(-1, keepdim=True) - 1)
    greedy, nothing = ~(t > 0), torch.isneginf(top)
    at = torch.where(greedy, 0, at)
    lp = torch.where(greedy, 0.0, torch.log(w.gather(1, at) / c[:, -1:]))
    tokens = torch.where(nothing, 0, order.gather(1, at))
    return {"tokens": tokens[:, 0], "logprobs": torch.where(nothing, float("-inf"), lp)[:, 0].float()}


def _exact_sample(c, seed):
    import numpy as np

    s = {k: (v.float() if k == "logits" else v).cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in _prepare_sample(c, seed).items()}
    n = c["rows"]
    tokens, lps = np.zeros(n, np.int64), np.zeros(n, np.float64)
    for i in range(n):
        row = s["logits"][i].astype(np.float64)
        row = np.where(np.isnan(row), -np.inf, row)
        best = row.max()
        if best == -np.inf:
            lps[i] = -np.inf
            continue
        if not s["temperature"][i] > 0:
            tokens[i] = int(row.argmax())
            continue
        live = np.flatnonzero(row > -np.inf)                       # ascending, so the stable sort keeps the lower index first
        live = live[np.argsort(-row[live], kind="stable")]
        if s["top_k"][i] > 0:
            live = live[: int(s["top_k"][i])]
        with np.errstate(invalid="ignore"):
            e = (row[live] - best) / float(s["temperature"][i])
        w = np.exp(np.where(row[live] == best, 0.0, e))
        m = int(np.count_nonzero(w >= float(s["min_p"][i]))) if s["min_p"][i] > 0 else len(w)
        w = w[:m]
        if s["top_p"][i] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            w = w[: max(1, int(np.count_nonzero(before < float(s["top_p"][i]) * w.sum())))]
        c_ = np.cumsum(w)
        j = min(int(np.searchsorted(c_, float(s["u"][i]) * c_[-1], side="right")), int(np.count_nonzero(w)) - 1)
        tokens[i], lps[i] = live[j], np.log(w[j]) - np.log(c_[-1])
    return {"tokens": torch.from_numpy(tokens), "logprobs": torch.from_numpy(lps)}


def _work_sample(c):
    e = 4 if c["dtype"] == "float32" else 2
    return {"bytes": c["rows"] * (c["vocab"] * e + 4 * 5 + 12), "flops": 2 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------ AdamW over many tensors
def _sizes(c):
    """Elements of every tensor: an adapter's factors, or a layer's weights with its norms and a few odd ones."""
    h, f, r = c["hidden"], c["inner"], c["rank"]
    qkv = h + h // 2
    if c["tensors"] == "factors":
        return [m * r for _ in range(c["layers"]) for m in (h, qkv, h, h, h, 2 * f, f, h)]
    return [m for _ in range(c["layers"]) for m in (h, qkv * h, h * h, 127, 1, h, 2 * f * h, h * f)]


def _offsets(c):
    at, off = 0, []
    for m in _sizes(c):
        off.append(at)
        at += -(-m // BLOCK) * BLOCK
    return off, at


def _spread(scale):
    return scale.repeat_interleave(BLOCK)


def _to_8_bits(v):
    """(e4m3 codes, one scale a block): the block's largest magnitude becomes 448; blocks below the normal numbers are zero."""
    s = v.abs().reshape(-1, BLOCK).amax(-1) / 448.0
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    q = torch.where(_spread(s) > 0, v / _spread(torch.where(s > 0, s, 1.0)), 0.0)
    return q, s


def _prepare_adamw(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes, (off, total) = _sizes(c), _offsets(c)
    real = torch.zeros(total, device="cuda", dtype=torch.bool)
    for o, m in zip(off, sizes):
        real[o:o + m] = True

    def rand(std, dtype=torch.float32):
        return torch.where(real, torch.empty(total, device="cuda").normal_(0.0, std, generator=g), 0.0).to(dtype)

    s = {"op": "adamw", "bits": c["bits"], "t": 7, "p": rand(0.02, getattr(torch, c["params"])), "g": rand(1e-2, getattr(torch, c["grads"])),
         "grad_scale": torch.rand(1, device="cuda", generator=g) * 0.5 + 0.5}
    m = rand(4e-3)
    v = rand(8e-3).square()
    if c["params"] == "bfloat16":
        s["master"] = s["p"].float()
    if c["bits"] == 8:
        q, s["m_scale"] = _to_8_bits(m)
        s["m"] = q.to(torch.float8_e4m3fn)
        q, s["v_scale"] = _to_8_bits(v.sqrt())
        s["v"] = torch.where(q > 0, q.clamp(min=2.0 ** -9), 0.0).to(torch.float8_e4m3fn)
    else:
        s |= {"m": m, "v": v}
    if own:
        from skyrl_isoexec_b200.ops.optim import TensorAdamW

        views = lambda t: [t[o:o + n] for o, n in zip(off, sizes)]  # noqa: E731
        opt = TensorAdamW(views(s["p"]), grads=views(s["g"]), betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=c["bits"])
        state = {"exp_avg": s["m"], "exp_avg_sq": s["v"]}
        if c["bits"] == 8:
            state |= {"exp_avg_scale": s["m_scale"], "exp_avg_sq_scale": s["v_scale"]}
        if c["params"] == "bfloat16":
            state["master"] = s["master"]
        opt.load_state_dict({"step": s["t"], **state})
        return {"op": "adamw", "opt": opt, "p": s["p"], "grad_scale": s["grad_scale"]}
    return s


def _run_adamw(s):
    if own:
        opt = s["opt"]
        opt.step(LR, grad_scale=s["grad_scale"])
        return {"p": s["p"], **opt.state}
    s["t"] += 1
    g = s["g"].float() * s["grad_scale"]
    m, v = s["m"], s["v"]
    if s["bits"] == 8:                     # e4m3 codes; the second moment is held by its square root
        m = m.float() * _spread(s["m_scale"])
        v = (v.float() * _spread(s["v_scale"])).square()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = s["master"] if "master" in s else s["p"]
    p = p * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** s["t"])) / ((v / (1 - BETA2 ** s["t"])).sqrt() + EPS)
    if s["bits"] == 8:
        q, s["m_scale"] = _to_8_bits(m)
        s["m"] = q.to(torch.float8_e4m3fn)
        q, s["v_scale"] = _to_8_bits(v.sqrt())
        s["v"] = torch.where(q > 0, q.clamp(min=2.0 ** -9), 0.0).to(torch.float8_e4m3fn)   # never zero beside a moving mean
    else:
        s["m"], s["v"] = m, v
    if "master" in s:
        s["master"] = p
        s["p"] = p.to(s["p"].dtype)
    else:
        s["p"] = p
    out = {"p": s["p"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}
    if s["bits"] == 8:
        out |= {"exp_avg_scale": s["m_scale"], "exp_avg_sq_scale": s["v_scale"]}
    if "master" in s:
        out["master"] = s["master"]
    return out


def _e4m3(x):
    """Nearest e4m3 value, ties to even, by its definition: three bits behind the leading one down to 2^-6, steps of 2^-9 below."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_adamw(c, seed):
    s = _prepare_adamw(c, seed)
    if "opt" in s:
        return None
    f = torch.float64
    per = torch.arange(s["p"].numel(), device="cuda") // BLOCK
    g = s["g"].to(f) * s["grad_scale"].to(f)
    m, v = s["m"].to(torch.float32).to(f), s["v"].to(torch.float32).to(f)
    if c["bits"] == 8:
        m = m * s["m_scale"].to(f)[per]
        v = (v * s["v_scale"].to(f)[per]) ** 2
    t = s["t"] + 1
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    p = (s["master"] if "master" in s else s["p"]).to(f)
    p = p - LR * (DECAY * p + m / (1 - BETA1 ** t) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS))
    out = {"p": p, "exp_avg": m, "exp_avg_sq": v}
    if "master" in s:
        out["master"] = p
    if c["bits"] == 8:
        for name, x in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
            scale = x.abs().view(-1, BLOCK).max(dim=1).values / 448
            y = torch.nan_to_num(x / scale[per])
            code = _e4m3(y)
            if name == "exp_avg_sq":
                code = torch.where((y > 0) & (code == 0), 2.0 ** -9, code)
            out[name], out[name + "_scale"] = code, scale
    return out


def _work_adamw(c):
    size = {"float32": 4, "bfloat16": 2}
    a_number = size[c["grads"]] + (8 + 2 if c["params"] == "bfloat16" else 8) + (4 * (1 + 2 / BLOCK * 4) if c["bits"] == 8 else 16)
    n = sum(_sizes(c))
    return {"bytes": int(n * a_number), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ what is called from outside
def prepare(case, seed):
    return {"lora": _prepare_lora, "sample": _prepare_sample, "adamw": _prepare_adamw}[case["op"]](case, seed)


def run(state):
    return {"lora": _run_lora, "sample": _run_sample, "adamw": _run_adamw}[state["op"]](state)


def exact(case, seed):
    return {"lora": _exact_lora, "sample": _exact_sample, "adamw": _exact_adamw}[case["op"]](case, seed)


def work(case):
    return {"lora": _work_lora, "sample": _work_sample, "adamw": _work_adamw}[case["op"]](case)
