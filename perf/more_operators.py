"""The products of a program's own experts, by size: the gated feed-forward block and the
product after it in 16 bits, both with their gradients, and products in 8-bit integers.

listed() holds fixed cases, draw() more of the same ranges; prepare() makes the
inputs from a seed; run() is one pass, in elementary torch operations or, with
`own`, through constellation_amd.engine; exact() restates it in 64 bits.

Sizes are the DeepSeek-V3 MoE geometry that bench.py measures (hidden 7168, inter
2048, top 8) over the experts of one node, and odd ones.  `experts` 0 is one matrix for all
rows; otherwise rows are token-expert pairs sorted by expert, and those without an expert
(`drop`) lie last.  Kinds:
  gated         h = silu(x G^T) * (x U^T); `keep`: also x G^T and x U^T, for the gradient
  product       y = x W^T
  gated_grad    from dh, x and what was kept: the gradients at x and at G and U.  The
                gradients at x G^T and x U^T are rounded to x's type in between
  product_grad  the gradients of product at x and W
  int8          rows of x to 8-bit integers with a scale per row, and their product with
                8-bit weights with a scale per channel; `gated` as above
"""
import math

import torch

own = False

HIDDEN, INTER, TOP_K = 7168, 2048, 8
LARGEST = 4096   # rows or tokens of one call
PAIRS = 16384    # token-expert pairs of one call
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one new token through an expert that every token takes
        {"name": "gated_token", "kind": "gated", "tokens": 1, "hidden": HIDDEN, "inter": INTER, "experts": 0, "top_k": 1, "dtype": "bf16", "drop": 0.0, "keep": False, "ordered": False},
        # sizes that neither a vector load nor a tile divides, with what a gradient needs
        {"name": "gated_ragged", "kind": "gated", "tokens": 357, "hidden": 1411, "inter": 333, "experts": 8, "top_k": 3, "dtype": "fp16", "drop": 0.2, "keep": True, "ordered": False},
        # a training batch on a node with 32 experts
        {"name": "gated_batch", "kind": "gated", "tokens": 2048, "hidden": HIDDEN, "inter": INTER, "experts": 32, "top_k": TOP_K, "dtype": "bf16", "drop": 0.0, "keep": True, "ordered": False},
        # a decode batch's rows through the experts' down projections
        {"name": "product_decode", "kind": "product", "tokens": 29, "hidden": HIDDEN, "inter": INTER, "experts": 64, "top_k": TOP_K, "dtype": "bf16", "drop": 0.0},
        # a long, ragged prompt through one expert's
        {"name": "product_prompt", "kind": "product", "tokens": 3001, "hidden": HIDDEN, "inter": INTER, "experts": 0, "top_k": 1, "dtype": "bf16", "drop": 0.0},
        # gradients where a fifth of the pairs is another node's
        {"name": "gated_grad_ragged", "kind": "gated_grad", "tokens": 509, "hidden": 2001, "inter": 357, "experts": 16, "top_k": 6, "dtype": "fp16", "drop": 0.2},
        # gradients of a training batch: gate and up
        {"name": "gated_grad_batch", "kind": "gated_grad", "tokens": 2048, "hidden": HIDDEN, "inter": INTER, "experts": 32, "top_k": TOP_K, "dtype": "bf16", "drop": 0.0},
        # one expert that every token takes, its weights' gradient in fp32
        {"name": "product_grad_shared", "kind": "product_grad", "tokens": 1000, "hidden": 2048, "inter": 1040, "experts": 0, "top_k": 1, "dtype": "bf16", "drop": 0.0, "dw": "f32"},
        # gradients of a training batch: down
        {"name": "product_grad_batch", "kind": "product_grad", "tokens": 2048, "hidden": HIDDEN, "inter": INTER, "experts": 32, "top_k": TOP_K, "dtype": "bf16", "drop": 0.0, "dw": "bf16"},
        # one new token through an 8-bit expert's gate and up
        {"name": "int8_token", "kind": "int8", "tokens": 1, "hidden": HIDDEN, "inter": INTER, "experts": 0, "top_k": 1, "dtype": "bf16", "drop": 0.0, "gated": True},
        # a long, ragged prompt through one 8-bit down projection
        {"name": "int8_prompt", "kind": "int8", "tokens": 3001, "hidden": HIDDEN, "inter": INTER, "experts": 0, "top_k": 1, "dtype": "bf16", "drop": 0.0, "gated": False},
        # a prefill chunk through the gates and ups of a node's 64 experts
        {"name": "int8_experts", "kind": "int8", "tokens": 1024, "hidden": HIDDEN, "inter": INTER, "experts": 64, "top_k": TOP_K, "dtype": "bf16", "drop": 0.0, "gated": True},
    ]


def _log(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(["gated", "gated", "product", "gated_grad", "gated_grad", "product_grad", "int8", "int8", "int8"])
    tokens, hidden, inter = _log(rng, 1, LARGEST), _log(rng, 64, HIDDEN), _log(rng, 16, INTER)
    if rng.random() < 0.6:
        hidden = max(64, hidden // 64 * 64)
    if rng.random() < 0.6:
        inter = max(16, inter // 16 * 16)
    experts = rng.choice([0, 0, 8, 16, 24, 32])
    top_k = rng.randint(1, 8) if experts else 1
    case = {"kind": kind, "tokens": min(tokens, PAIRS // top_k), "hidden": hidden, "inter": inter, "experts": experts, "top_k": top_k,
            "dtype": rng.choice(["bf16", "fp16"]), "drop": rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.75), 3)]) if experts else 0.0}
    if kind == "gated":
        case["keep"] = rng.random() < 0.5
        case["ordered"] = experts > 0 and not case["keep"]
    elif kind == "product_grad":
        case["dw"] = rng.choice(["f32", case["dtype"]])
    elif kind == "int8":
        case["gated"] = rng.random() < 0.5
    return case


class State:
    def __init__(self, case):
        self.case, self.ctx = dict(case), None
        if own:
            from constellation_amd.engine import Context
            self.ctx = Context(0)

    def __del__(self):
        if self.ctx is not None:
            self.ctx.close()


def _dealt(s, gen):
    """The pairs of a batch by expert: `order` (a pair's token is order // top_k; complements without an
    expert), `offsets` on the GPU and `cuts`, the same on the host."""
    c = s.case
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    if e == 0:
        s.order = s.offsets = None
        s.cuts = [0, t]
        return
    lean = torch.randn(e, generator=gen, device="cuda") * 0.3  # some experts are taken more often
    ids = (torch.rand(t, e, generator=gen, device="cuda") + lean).topk(k, dim=1).indices
    lost = torch.rand(t, k, generator=gen, device="cuda") < c["drop"]
    flat = torch.where(lost, e, ids).reshape(-1)
    order = torch.argsort(flat, stable=True).to(torch.int32)
    s.order = torch.where(flat[order.long()] == e, ~order, order)
    s.offsets = (flat[None, :] < torch.arange(e + 1, device="cuda")[:, None]).sum(1).to(torch.int32)
    s.cuts = s.offsets.tolist()


def prepare(case, seed):
    s = State(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, h, i = case["kind"], DTYPES[case["dtype"]], case["hidden"], case["inter"]
    pairs = case["tokens"] * case["top_k"]
    _dealt(s, gen)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    def weights(rows, cols):
        w = torch.empty(max(1, case["experts"]), rows, cols, dtype=dtype, device="cuda")
        for m in range(w.shape[0]):
            w[m] = normal(rows, cols, std=0.02)
        return w if case["experts"] else w[0]

    if kind == "gated":
        s.x = normal(case["tokens"] if case["ordered"] else pairs, h)
        s.w = weights(2 * i, h)
    elif kind == "product":
        s.x, s.w = normal(pairs, i), weights(h, i)
    elif kind == "gated_grad":
        s.x, s.w, s.dy = normal(pairs, h), weights(2 * i, h), normal(pairs, i, std=0.1)
        s.pre = normal(pairs, 2 * i, std=0.02 * math.sqrt(h))
    elif kind == "product_grad":
        s.x, s.w, s.dy = normal(pairs, i), weights(h, i), normal(pairs, h, std=0.1)
    else:
        rows, cols = (2 * i, h) if case["gated"] else (h, i)
        s.x = normal(case["tokens"], cols)
        mats = max(1, case["experts"])
        s.w = torch.empty(mats, rows, cols, dtype=torch.int8, device="cuda")
        for m in range(mats):  # as a normal weight's quantisation gives them
            s.w[m] = torch.randn(rows, cols, generator=gen, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s.ws = (0.02 / 32) * (0.8 + 0.4 * torch.rand(mats, rows, generator=gen, device="cuda"))
        if not case["experts"]:
            s.w, s.ws = s.w[0], s.ws[0]
    return s


# -- the plain forms ------------------------------------------------------------

def _silu_mul(v):
    gate, up = v.chunk(2, 1)
    return gate / (1 + torch.exp(-gate)) * up


def _each(s):
    """(matrix, its first row, the row behind its last) of the matrices that have rows."""
    return [(m, a, b) for m, (a, b) in enumerate(zip(s.cuts, s.cuts[1:])) if b > a]


def _stack(t):
    return t if t.dim() == 3 else t.unsqueeze(0)


def _products(s, x, weights):
    """x W^T in fp32, the rows behind the last matrix's zeros."""
    y = torch.zeros(x.shape[0], weights.shape[1], device=x.device)
    for m, a, b in _each(s):
        torch.matmul(x[a:b].float(), weights[m].float().T, out=y[a:b])
    return y


def _gate_grad(dh, pre):
    """The gradient of silu(g) * u at pre = [g, u]."""
    g, u = pre.float().chunk(2, 1)
    sig = 1 / (1 + torch.exp(-g))
    return torch.cat((dh.float() * u * sig * (1 + g * (1 - sig)), dh.float() * g * sig), 1)


def _rows8(x):
    """8-bit integers of the rows of x, and their scales."""
    scale = (x.float().abs().amax(1) / torch.full((), 127.0, device=x.device)).clamp_min(1e-12)
    return torch.round(x.float() / scale[:, None]).clamp(-127, 127).to(torch.int8), scale


def _picked(s, x):
    """The pairs' rows of x."""
    pair = torch.where(s.order < 0, ~s.order, s.order).long()
    return x[pair // s.case["top_k"]]


def run(s):
    c = s.case
    kind = c["kind"]
    if own:
        ctx = s.ctx
        if kind == "gated":
            by = {"order": s.order, "top_k": c["top_k"]} if c["ordered"] else {}
            if not c["keep"]:
                return ctx.matmul(s.x, s.w, gated=True, offsets=s.offsets, **by)
            h, pre = ctx.matmul(s.x, s.w, gated=True, keep=True, offsets=s.offsets, **by)
            return {"h": h, "pre": pre}
        if kind == "product":
            return ctx.matmul(s.x, s.w, offsets=s.offsets)
        if kind == "gated_grad":
            dx, dw = ctx.matmul_grad(s.dy, s.x, s.w, pre=s.pre, offsets=s.offsets)
            return {"dx": dx, "dw": dw}
        if kind == "product_grad":
            dx, dw = ctx.matmul_grad(s.dy, s.x, s.w, offsets=s.offsets, dw_dtype=DTYPES[c["dw"]])
            return {"dx": dx, "dw": dw}
        q, scale = ctx.quantize_i8(s.x)
        y = ctx.i8_matmul(q, scale, s.w, s.ws, gated=c["gated"], offsets=s.offsets, order=s.order, top_k=c["top_k"],
                          out_dtype=DTYPES[c["dtype"]])
        return {"y": y, "scale": scale}
    dtype = s.x.dtype
    if kind == "gated":
        pre = _products(s, _picked(s, s.x) if c["ordered"] else s.x, _stack(s.w))
        h = _silu_mul(pre).to(dtype)
        return {"h": h, "pre": pre.to(dtype)} if c["keep"] else h
    if kind == "product":
        return _products(s, s.x, _stack(s.w)).to(dtype)
    if kind in ("gated_grad", "product_grad"):
        dy = _gate_grad(s.dy, s.pre).to(dtype) if kind == "gated_grad" else s.dy
        w = _stack(s.w)
        dw = torch.zeros(w.shape, dtype=DTYPES[c.get("dw", c["dtype"])], device="cuda")
        dx = torch.zeros_like(s.x)
        for m, a, b in _each(s):
            d = dy[a:b].float()
            dx[a:b] = d @ w[m].float()
            dw[m] = d.T @ s.x[a:b].float()
        return {"dx": dx, "dw": dw.view(s.w.shape)}
    q, scale = _rows8(s.x)
    x = q.float() * scale[:, None]
    y = _products(s, x if s.order is None else _picked(s, x), _stack(s.w))
    ws = s.ws if c["experts"] else s.ws[None]
    for m, a, b in _each(s):
        y[a:b] *= ws[m]
    return {"y": (_silu_mul(y) if c["gated"] else y).to(dtype), "scale": scale}


def work(case):
    kind, h, i, e = case["kind"], case["hidden"], case["inter"], case["experts"]
    pairs = case["tokens"] * case["top_k"]
    rows = pairs * (1 - case["drop"])
    active = e * (1 - (1 - 1 / e) ** rows) if e else 1
    if kind == "int8":
        n, k = (2 * i, h) if case["gated"] else (h, i)
        out = pairs * (i if case["gated"] else h) * 2
        return {"bytes": active * (n * k + 4 * n) + case["tokens"] * (2 * k + 4) + out, "flops": 2 * rows * n * k}
    n, k = (2 * i, h) if kind.startswith("gated") else (h, i)
    weights, x = active * n * k * 2, (case["tokens"] if case.get("ordered") else rows) * k * 2
    if kind == "gated":
        return {"bytes": weights + x + pairs * i * 2 * (3 if case["keep"] else 1), "flops": 2 * rows * n * k}
    if kind == "product":
        return {"bytes": weights + x + pairs * n * 2, "flops": 2 * rows * n * k}
    dw = max(1, e) * n * k * (4 if case.get("dw") == "f32" else 2)
    dy = rows * (3 * i if kind == "gated_grad" else n) * 2
    return {"bytes": weights + x + dy + dw + pairs * k * 2, "flops": 4 * rows * n * k}


# -- the definitions in 64 bits ---------------------------------------------------

def _plain_state(case, seed):
    """prepare()'s inputs, without the engine."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def exact(case, seed):
    s = _plain_state(case, seed)
    kind, i = case["kind"], case["inter"]
    w = s.w if case["experts"] else s.w[None]
    spans = [(m, s.cuts[m], s.cuts[m + 1]) for m in range(w.shape[0])]
    pairs = case["tokens"] * case["top_k"]

    def f64(*shape):
        return torch.zeros(*shape, dtype=torch.float64, device="cuda")

    if kind in ("gated", "product", "int8"):
        x, factor = s.x.double(), None
        scale = None
        if kind == "int8":
            scale = torch.clamp((x.abs().max(1).values / 127).float(), min=1e-12)
            x = torch.round((x / scale.double()[:, None]).float()).double() * scale.double()[:, None]
            factor = s.ws.double() if case["experts"] else s.ws.double()[None]
        if case.get("ordered") or (kind == "int8" and case["experts"]):
            x = x[(s.order ^ (s.order >> 31)).long() // case["top_k"]]
        y = f64(pairs, w.shape[1])
        for m, a, b in spans:
            y[a:b] = x[a:b] @ w[m].double().T
            if factor is not None:
                y[a:b] *= factor[m]
        if kind == "product":
            return y
        if kind == "gated" or case["gated"]:
            h = y[:, :i] * torch.sigmoid(y[:, :i]) * y[:, i:]
            if kind == "gated":
                return {"h": h, "pre": y} if case["keep"] else h
            y = h
        return {"y": y, "scale": scale}
    dy = s.dy.double()
    if kind == "gated_grad":
        g, u = s.pre[:, :i].double(), s.pre[:, i:].double()
        t = torch.sigmoid(g)
        dy = torch.cat((dy * u * (t + g * t * (1 - t)), dy * g * t), 1).to(s.x.dtype).double()
    dx, dw = f64(*s.x.shape), f64(*w.shape)
    for m, a, b in spans:
        dx[a:b] = dy[a:b] @ w[m].double()
        dw[m] = dy[a:b].T @ s.x[a:b].double()
    return {"dx": dx, "dw": dw.view(s.w.shape)}
