"""What the ragged expert path and the gradient clipping are measured on.

Four kinds of case:

- ``layout``: the router's choice -> rows of each expert (``ragged_layout``)
- ``linear``: one product grouped by expert, without gradients, as serving and
  evaluation call it (``grouped_linear``)
- ``train``:  the same product and its three gradients
- ``step``:   the norm over many gradients and the clipped step of the fp32
  masters (``grad_clip_scale`` and ``master_sgd_step_``)

``run`` computes each in its plain form, or by the framework's own kernels
where ``own`` is true.
"""
import math

import torch

own = False

DEV = "cuda:0"


def _layout(name, **kw):
    return {"kind": "layout", "masked": 0.0, **kw, **({"name": name} if name else {})}


def _linear(name, **kw):
    return {"kind": "linear", "masked": 0.0, "gelu": False, "skew": 0.7, **kw, **({"name": name} if name else {})}


def _train(name, **kw):
    return {**_linear(name, **kw), "kind": "train"}


def _step(name, **kw):
    return {"kind": "step", "momentum": 0.0, "decay": 0.0, **kw, **({"name": name} if name else {})}


def listed():
    return [
        # eight tokens in flight of a serving loop: latency alone
        _layout("layout-decode", T=8, k=4, E=256),
        # a training step of the 256-expert model: 96 sequences of 1024
        _layout("layout-step", T=98304, k=4, E=256),
        # the single-expert router of the 1024-expert model, a tenth of the tokens padding
        _layout("layout-switch", T=65537, k=1, E=1024, masked=0.1),
        # one decoded token through the first product of its four experts
        _linear("decode-1", T=1, k=4, E=256, K=1024, N=4096, gelu=True, skew=0.0),
        # 32 sequences decoded together, second product
        _linear("decode-32", T=32, k=4, E=256, K=4096, N=1024, skew=0.0),
        # a prompt batch: a few dozen rows for each expert, ragged
        _linear("prompt-2k", T=2051, k=4, E=256, K=1024, N=4096, gelu=True),
        # the forward product of a training step, many rows for each expert
        _linear("forward-64k", T=65536, k=4, E=256, K=1024, N=4096, gelu=True),
        # small experts with sizes off every tile, some tokens masked out
        _train("train-odd", T=999, k=2, E=12, K=136, N=328, gelu=True, masked=0.05),
        # the single-expert model's second product: 1024 experts, few rows for each
        _train("train-switch", T=32768, k=1, E=1024, K=2048, N=512),
        # the largest: the 256-expert model's first product and its gradients
        _train("train-64k", T=65536, k=4, E=256, K=1024, N=4096),
        # the trunk of the 256-expert model: 44 bf16 tensors with fp32 masters
        _step("step-trunk", d=1024, layers=6, vocab=32000, grads="bf16", tensors=0, size=0),
        # expert stacks: a few large fp32 gradients, momentum and decay
        _step("step-experts", d=0, layers=0, vocab=0, grads="fp32", tensors=4, size=67108864, momentum=0.9, decay=0.01),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layout", "linear", "linear", "train", "train", "step"])
    masked = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.4), 3)])
    if kind == "layout":
        k = rng.choice([1, 2, 4, 8])
        E = _log(rng, k, 4096)
        return _layout("", T=_log(rng, 1, min(393216 // k, (1 << 28) // E)), k=k, E=E, masked=masked)
    if kind == "step":
        tensors = _log(rng, 1, 200)
        return _step("", d=0, layers=0, vocab=0, grads=rng.choice(["bf16", "fp32"]), tensors=tensors,
                     size=_log(rng, 16, 200_000_000 // tensors), momentum=rng.choice([0.0, 0.9]),
                     decay=rng.choice([0.0, 0.01]))
    k = rng.choice([1, 2, 4])
    E = _log(rng, max(2, k), 1024)
    K, N = 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512)
    while E * K * N > 1 << 30:
        E = max(k, E // 2)
    most = min(262144, (1 << 40) // (K * N), (1 << 30) // max(K, N))  # rows: no more work than the largest listed case
    T = _log(rng, 1, max(1, most // k))
    return (_linear if kind == "linear" else _train)(
        "", T=T, k=k, E=E, K=K, N=N, gelu=rng.choice([True, False]), masked=masked, skew=round(rng.uniform(0.0, 1.2), 2))


def _tensor_sizes(c):
    """Element counts of the tensors of a step: a transformer's trunk, or so many ragged ones."""
    if c["layers"]:
        d = c["d"]
        return [c["vocab"] * d, 1024 * d] + c["layers"] * [d, d, 3 * d * d, d * d, d, d, 256 * d] + [d, d]
    return [max(1, c["size"] - (i * 37) % max(1, c["size"] // 3)) for i in range(c["tensors"])]


def _choose(c, g):
    """A router's choice: k experts a token by the largest logits, some experts liked more than others."""
    bias = torch.randn(c["E"], device=DEV, generator=g) * c.get("skew", 0.7)
    logits = torch.randn(c["T"], c["E"], device=DEV, generator=g) + bias
    ids = logits.topk(c["k"], dim=-1).indices.to(torch.int32)
    if c["masked"]:  # padding tokens choose no expert
        gone = torch.rand(c["T"], device=DEV, generator=g) < c["masked"]
        ids = ids.masked_fill(gone[:, None], -1)
    return ids


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    if c["kind"] == "layout":
        return {"case": c, "ids": _choose(c, g)}
    if c["kind"] == "step":
        sizes = _tensor_sizes(c)
        gt = torch.bfloat16 if c["grads"] == "bf16" else torch.float32
        masters = [rand(n, scale=0.02, dtype=torch.float32) for n in sizes]
        s = {"case": c, "masters": masters, "params": [m.bfloat16() for m in masters],
             "grads": [rand(n, scale=0.01 * (1 + i % 3), dtype=gt) for i, n in enumerate(sizes)], "bufs": None}
        if c["momentum"]:
            s["bufs"] = [rand(n, scale=0.01, dtype=torch.float32) for n in sizes]
        return s
    E, K, N, R = c["E"], c["K"], c["N"], c["T"] * c["k"]
    ids = _choose(c, g).flatten()
    counts = torch.bincount(ids[ids >= 0].long(), minlength=E)
    ends = torch.cumsum(counts, 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    grad = c["kind"] == "train"
    s = {"case": c, "offsets": offsets, "bounds": offsets.tolist(),
         "x": rand(R, K).requires_grad_(grad),
         "w": torch.empty(E, N, K, device=DEV, dtype=torch.bfloat16),
         "b": rand(E, N, scale=0.1).requires_grad_(grad)}
    for e in range(0, E, 64):  # in parts: the fp32 numbers before the rounding are twice the size
        part = s["w"][e:e + 64]
        part.copy_(rand(*part.shape, scale=1.0 / math.sqrt(K)))
    s["w"].requires_grad_(grad)
    if grad:
        s["dy"] = rand(R, N)
    return s


# ---- the plain forms ------------------------------------------------------------

def _plain_layout(ids, E):
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    offsets = torch.cat([torch.zeros_like(counts[:1]), torch.cumsum(counts, 0)])
    order = torch.where(key[order] < E, order, -1)
    rows = torch.where(key < E, rows, -1)
    return {"offsets": offsets.to(torch.int32), "order": order.to(torch.int32),
            "rows": rows.to(torch.int32).view(ids.shape)}


def _gelu(u):
    t = torch.tanh(0.7978845608028654 * (u + 0.044715 * u * u * u))
    return 0.5 * u * (1 + t), t


def _gelu_slope(u, t):
    return 0.5 * (1 + t) + 0.5 * u * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * u * u)


def _plain_linear(s):
    c, x, w, b, at = s["case"], s["x"], s["w"], s["b"], s["bounds"]
    train = c["kind"] == "train"
    y = torch.zeros(x.shape[0], c["N"], device=x.device, dtype=x.dtype)
    if train:
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for e in range(c["E"]):  # each expert has rows and weights of its own
        lo, hi = at[e], at[e + 1]
        if lo == hi:
            continue
        xe, we = x[lo:hi].float(), w[e].float()
        u = xe @ we.t() + b[e].float()
        v, t = _gelu(u) if c["gelu"] else (u, None)
        y[lo:hi] = v.to(y.dtype)
        if train:
            du = s["dy"][lo:hi].float()
            if c["gelu"]:
                du = du * _gelu_slope(u, t)
            dx[lo:hi] = (du @ we).to(x.dtype)
            dw[e] = (du.t() @ xe).to(w.dtype)
            db[e] = du.sum(0).to(b.dtype)
    return {"y": y, "dx": dx, "dw": dw, "db": db} if train else {"y": y}


LR, MAX_NORM = 0.01, 1.0


def _plain_step(s):
    c = s["case"]
    squares = [g.float().square().sum(dtype=torch.float64) for g in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    scale = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    bufs = s["bufs"] or [None] * len(s["grads"])
    for p, m, g, v in zip(s["params"], s["masters"], s["grads"], bufs):
        u = g.float() * scale
        if c["decay"]:
            u = u + c["decay"] * m
        if v is not None:
            v.mul_(c["momentum"]).add_(u)
            u = v
        m.sub_(LR * u)
        p.copy_(m)
    return {"norm": norm.float(), "scale": scale}


@torch.no_grad()
def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "layout":
        return _plain_layout(s["ids"], s["case"]["E"])
    return _plain_step(s) if kind == "step" else _plain_linear(s)


# ---- the framework's operators ---------------------------------------------------

def _run_own(s):
    from learning_at_home_amd.ops import functional as ops

    c = s["case"]
    act = "gelu" if c.get("gelu") else None
    if c["kind"] == "layout":
        layout = ops.ragged_layout(s["ids"], c["E"])
        return {"offsets": layout.offsets, "order": layout.order, "rows": layout.rows}
    if c["kind"] == "step":
        norm, scale = ops.grad_clip_scale(s["grads"], MAX_NORM)
        ops.master_sgd_step_(s["params"], s["masters"], s["grads"], lr=LR, momentum=c["momentum"],
                             weight_decay=c["decay"], momentum_bufs=s["bufs"], grad_scale=scale)
        return {"norm": norm, "scale": scale}
    y = ops.grouped_linear(s["x"], s["w"], s["offsets"], s["b"], activation=act)
    if c["kind"] == "linear":
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def run(state):
    out = _run_own(state) if own else _run_plain(state)
    if state["case"]["kind"] == "step":
        # the first tensors whole, the last ones too: an answer holds 64 outputs at most
        ends = range(len(state["params"]))
        ends = [i for i in ends if i < 12 or i >= len(state["params"]) - 8]
        out["masters"] = [state["masters"][i] for i in ends]
        out["params"] = [state["params"][i] for i in ends]
        if state["bufs"] is not None:
            out["bufs"] = [state["bufs"][i] for i in ends]
    return out


def work(case):
    c = case
    if c["kind"] == "layout":
        n = c["T"] * c["k"]
        return {"bytes": 12 * n + 4 * (c["E"] + 1), "flops": 0}
    if c["kind"] == "step":
        n = sum(_tensor_sizes(c))
        each = (2 if c["grads"] == "bf16" else 4) + 8 + 2 + (8 if c["momentum"] else 0)
        return {"bytes": each * n, "flops": 8 * n}
    R, N, K, E = c["T"] * c["k"] * (1 - c["masked"]), c["N"], c["K"], c["E"]
    active = E * (1 - (1 - c["k"] / E) ** (c["T"] * (1 - c["masked"])))  # experts with a row at all, if all are liked alike
    bytes_ = 2 * (c["T"] * c["k"] * (K + N) + active * (N * K + N))
    flops = 2 * R * N * K
    if c["kind"] == "train":
        bytes_ += 2 * (c["T"] * c["k"] * (K + N) + E * (N * K + N))  # dy in, dx out, dw and db out
        flops *= 3
    return {"bytes": int(bytes_), "flops": int(flops)}


# ---- in 64 bits, apart from the plain forms --------------------------------------

def _exact_linear(s):
    c, f64 = s["case"], torch.float64
    x, w, b = (s[n].detach() for n in ("x", "w", "b"))
    of_row = torch.searchsorted(s["offsets"][1:].long(), torch.arange(x.shape[0], device=x.device), right=True)
    train = c["kind"] == "train"
    out = {"y": torch.zeros(x.shape[0], c["N"], device=x.device, dtype=f64)}
    if train:
        out.update(dx=torch.zeros(x.shape, device=x.device, dtype=f64), dw=torch.zeros(w.shape, device=x.device, dtype=f64),
                   db=torch.zeros(b.shape, device=x.device, dtype=f64))
    for e in of_row.unique().tolist():
        if e >= c["E"]:
            continue
        mine = (of_row == e).nonzero().squeeze(1)
        xe, we = x[mine].to(f64), w[e].to(f64)
        u = torch.addmm(b[e].to(f64), xe, we.T)
        slope = None
        if c["gelu"]:  # (1 + tanh(a)) / 2 = sigmoid(2 a)
            z = math.sqrt(8 / math.pi) * (u + 0.044715 * u ** 3)
            q = torch.sigmoid(z)
            slope = q + u * q * (1 - q) * math.sqrt(8 / math.pi) * (1 + 0.134145 * u ** 2)
            u = u * q
        out["y"].index_copy_(0, mine, u)
        if train:
            du = s["dy"][mine].to(f64)
            du = du if slope is None else du * slope
            out["dx"].index_copy_(0, mine, du.mm(we))
            out["dw"][e] = du.T.mm(xe)
            out["db"][e] = du.T.mv(torch.ones(len(mine), device=x.device, dtype=f64))
    return out


def _exact_step(s):
    c, f64 = s["case"], torch.float64
    norm = math.sqrt(sum(float(torch.dot(g.to(f64), g.to(f64))) for g in s["grads"]))
    scale = min(1.0, MAX_NORM / (norm + 1e-6))
    last = len(s["params"])
    keep = [i for i in range(last) if i < 12 or i >= last - 8]
    out = {"norm": torch.tensor(norm, dtype=f64), "scale": torch.tensor(scale, dtype=f64), "masters": [], "params": []}
    if c["momentum"]:
        out["bufs"] = []
    for i in keep:
        m = s["masters"][i].to(f64)
        u = s["grads"][i].to(f64) * scale + c["decay"] * m
        if c["momentum"]:
            u = c["momentum"] * s["bufs"][i].to(f64) + u
            out["bufs"].append(u)
        m = m - LR * u
        out["masters"].append(m)
        out["params"].append(m)
    return out


@torch.no_grad()
def exact(case, seed):
    if case["kind"] == "layout":
        return None  # whole numbers, and no rounding in them
    s = prepare(case, seed)
    return _exact_step(s) if case["kind"] == "step" else _exact_linear(s)
