"""The operators of an expert block as cases to time and compare.

An expert block is ``x + combine(down(gelu(up(dispatch(layer_norm(x))))))``: a norm, a router, ragged
products grouped by expert, and the rows' way to the experts and back.  Its operators are

    norm      layer_norm, and its gradients to x, weight and bias
    route     the k largest of each token's logits, their softmax, the assignments' order by expert
    shuffle   dispatch (tokens to rows sorted by expert) and combine (weighted rows back to tokens)
    product   expert_mm, and its gradients to the rows and to the experts' weights

``own = False`` computes them in elementary torch operations in 32 bits, rounded once; ``own = True`` calls
the package.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # one token of a decoding step, 4096 wide: what a call costs
        dict(name="norm_token", kind="norm", dtype="bf16", rows=1, cols=4096, train=False),
        # one block of the pipeline benchmark: 8 x 512 tokens, 2048 wide
        dict(name="norm_block", kind="norm", dtype="bf16", rows=4096, cols=2048, train=True),
        # an FP32 model of odd width, whose rows start at any multiple of 4 bytes
        dict(name="norm_odd_fp32", kind="norm", dtype="fp32", rows=2021, cols=897, train=True),
        # a batch of long sequences, 4096 wide
        dict(name="norm_long", kind="norm", dtype="bf16", rows=65536, cols=4096, train=True),
        # one token of a decoding step among 64 experts
        dict(name="route_token", kind="route", dtype="bf16", tokens=1, experts=64, top_k=4, normalize=True, train=False),
        # a training batch among 128 experts, FP32 logits as routers are usually kept
        dict(name="route_batch", kind="route", dtype="fp32", tokens=32768, experts=128, top_k=8, normalize=True, train=True),
        # a few decoding sequences of an FP32 model of odd width
        dict(name="shuffle_few", kind="shuffle", dtype="fp32", tokens=7, experts=8, top_k=2, hidden=897, train=False),
        # a training batch, 2048 wide, four experts a token
        dict(name="shuffle_batch", kind="shuffle", dtype="bf16", tokens=16384, experts=64, top_k=4, hidden=2048, train=True),
        # one token of a decoding step: 8 rows, each with its own expert's 1536 x 2048 weights
        dict(name="product_token", kind="product", dtype="bf16", rows=8, experts=64, n=1536, k=2048, train=False),
        # the pipeline's tokens, two of 8 experts each, its own 2048 -> 8192
        dict(name="product_block", kind="product", dtype="bf16", rows=8192, experts=8, n=8192, k=2048, train=True),
        # many narrow experts and a large batch
        dict(name="product_fine", kind="product", dtype="bf16", rows=65536, experts=64, n=1536, k=2048, train=True),
        # an FP32 model of odd sizes
        dict(name="product_odd_fp32", kind="product", dtype="fp32", rows=1237, experts=5, n=193, k=333, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, its logarithm uniform."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A size of a layer: half of them multiples of 64, the others any number."""
    n = _spread(rng, lo, hi)
    n = max(64, n // 64 * 64) if rng.random() < 0.5 else n
    return n + 1 if n == 3072 else n


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["norm", "route", "shuffle", "product", "product"])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.7)
    if kind == "norm":
        case["cols"] = _width(rng, 33, 16384)
        case["rows"] = min(_spread(rng, 1, 65536), (1 << 28) // case["cols"])
        return case
    if kind == "product":
        case["experts"] = _spread(rng, 1, 128)
        case["n"], case["k"] = _width(rng, 16, 8192), _width(rng, 16, 8192)
        case["rows"] = _spread(rng, 1, 65536)
        while case["experts"] * case["n"] * case["k"] > 2e8:
            case["experts"] = max(1, case["experts"] // 2)
        most = 2e11 if case["dtype"] == "bf16" else 1.2e10
        case["rows"] = max(1, min(case["rows"], int(most / (case["n"] * case["k"]))))
        return case
    case["tokens"] = _spread(rng, 1, 32768)
    case["experts"] = _spread(rng, 2, 256)
    case["top_k"] = min(case["experts"], rng.choice([1, 2, 4, 6, 8]))
    if kind == "route":
        case["normalize"] = rng.random() < 0.6
    else:
        case["hidden"] = _width(rng, 33, 8192)
        case["tokens"] = max(1, min(case["tokens"], (1 << 27) // (case["hidden"] * case["top_k"])))
    return case


# ---------------------------------------------------------------------- inputs

def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device=DEVICE) * scale


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # a residual stream: not centred, and some features much larger than the others
        x = torch.empty(rows, cols, dtype=dtype, device=DEVICE).normal_(0.2, 1.5, generator=gen)
        x[:, :: max(1, cols // 8)] *= 6.0
        s.update(x=x, weight=(1.0 + _normal(gen, cols, scale=0.1)).to(dtype), bias=_normal(gen, cols, scale=0.1).to(dtype))
        if case["train"]:
            s["gout"] = torch.empty(rows, cols, dtype=dtype, device=DEVICE).normal_(0.0, 0.01, generator=gen)
        leaves = ("x", "weight", "bias")
    elif case["kind"] == "route":
        tokens, experts = case["tokens"], case["experts"]
        popular = _normal(gen, experts, scale=0.7)   # some experts are chosen more often
        s["logits"] = (_normal(gen, tokens, experts, scale=1.5) + popular).to(dtype)
        if case["train"]:
            s["gout"] = _normal(gen, tokens, case["top_k"], scale=0.01)
        leaves = ("logits",)
    elif case["kind"] == "shuffle":
        tokens, k, hidden = case["tokens"], case["top_k"], case["hidden"]
        logits = _normal(gen, tokens, case["experts"], scale=1.5) + _normal(gen, case["experts"], scale=0.7)
        weights, chosen = torch.topk(torch.softmax(logits, 1), k, 1)
        order = torch.sort(chosen.reshape(-1), stable=True).indices
        position = torch.empty_like(order)
        position[order] = torch.arange(tokens * k, device=DEVICE)
        s.update(weights=weights, experts=chosen.int(), order=order.int(), position=position.int().view(tokens, k),
                 ends=torch.bincount(chosen.reshape(-1), minlength=case["experts"]).cumsum(0).int())
        s.update(x=_normal(gen, tokens, hidden).to(dtype), y=_normal(gen, tokens * k, hidden).to(dtype))
        if case["train"]:
            s.update(grows=_normal(gen, tokens * k, hidden, scale=0.01).to(dtype),
                     gout=_normal(gen, tokens, hidden, scale=0.01).to(dtype))
        leaves = ("x", "y", "weights")
    else:
        rows, experts, n, k = case["rows"], case["experts"], case["n"], case["k"]
        popular = torch.softmax(_normal(gen, experts, scale=0.7), 0)
        if experts > 2:
            popular[experts // 2] = 0.0   # an expert that no token chose
        chosen = torch.multinomial(popular, rows, replacement=True, generator=gen)
        s["ends"] = torch.bincount(chosen, minlength=experts).cumsum(0).int()
        s["x"] = _normal(gen, rows, k).to(dtype)
        s["weight"] = torch.empty(experts, n, k, dtype=dtype, device=DEVICE).normal_(0.0, 0.02, generator=gen)
        if case["train"]:
            s["gout"] = _normal(gen, rows, n, scale=0.01).to(dtype)
        leaves = ("x", "weight")
    if case["train"]:
        for name in leaves:
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------ runs

def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    dtype = s["x"].dtype
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(dtype)
    if not s["case"]["train"]:
        return y
    g = s["gout"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return y, dx.to(dtype), (g * xh).sum(0).to(dtype), g.sum(0).to(dtype)


def _plain_route(s):
    case, logits = s["case"], s["logits"].float()
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    values, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    values, chosen = values[:, :k], chosen[:, :k]
    if case["normalize"]:
        e = torch.exp(values - values[:, :1])
        weights = e / e.sum(1, keepdim=True)
    else:
        p = torch.exp(logits - values[:, :1])
        p = p / p.sum(1, keepdim=True)
        weights = torch.gather(p, 1, chosen)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(tokens * k, device=DEVICE)
    ends = (flat[:, None] == torch.arange(experts, device=DEVICE)).sum(0).cumsum(0)
    out = [weights, chosen.int(), ends.int(), order.int(), position.view(tokens, k).int()]
    if case["train"]:
        seed = weights * s["gout"]
        total = seed.sum(1, keepdim=True)
        if case["normalize"]:
            grad = torch.zeros_like(logits).scatter(1, chosen, seed - weights * total)
        else:
            grad = torch.zeros_like(logits).scatter(1, chosen, seed) - p * total
        out.append(grad.to(s["logits"].dtype))
    return out


def _plain_shuffle(s):
    case, dtype = s["case"], s["x"].dtype
    k = case["top_k"]
    token, place = s["order"].long() // k, s["position"].long()
    rows = s["x"][token]
    y = s["y"].float()[place]
    w = s["weights"]
    out = (y * w[:, :, None]).sum(1).to(dtype)
    if not case["train"]:
        return rows, out
    dx = s["grows"].float()[place].sum(1).to(dtype)
    g = s["gout"].float()
    dy = (w.reshape(-1)[s["order"].long()][:, None] * g[token]).to(dtype)
    dw = (y * g[:, None, :]).sum(2)
    return rows, out, dx, dy, dw


def _plain_product(s):
    """Each expert's rows padded to the longest of them, and batched products of the padded rows."""
    case, dtype = s["case"], s["x"].dtype
    rows, experts = case["rows"], case["experts"]
    ends = s["ends"].long()
    starts = torch.cat((ends.new_zeros(1), ends[:-1]))
    most = int((ends - starts).max())
    at = torch.arange(rows, device=DEVICE)
    expert = (at[:, None] >= ends).sum(1)
    place = at - starts[expert]
    x = torch.zeros(experts, most, case["k"], device=DEVICE)
    x[expert, place] = s["x"].float()
    w = s["weight"].float()
    out = torch.bmm(x, w.transpose(1, 2))[expert, place].to(dtype)
    if not case["train"]:
        return out
    g = torch.zeros(experts, most, case["n"], device=DEVICE)
    g[expert, place] = s["gout"].float()
    dx = torch.bmm(g, w)[expert, place].to(dtype)
    dw = torch.bmm(g.transpose(1, 2), x).to(dtype)
    return out, dx, dw


def _own_norm(ab, s):
    y = ab.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not s["case"]["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["gout"]))


def _own_route(ab, s):
    case = s["case"]
    r = ab.route(s["logits"], case["top_k"], normalize=case["normalize"])
    out = [r.weights.detach(), r.experts, r.ends, r.order, r.position]
    if case["train"]:
        out += torch.autograd.grad(r.weights, (s["logits"],), s["gout"])
    return out


def _own_shuffle(ab, s):
    r = ab.Routing(s["weights"], s["experts"], s["ends"], s["order"], s["position"])
    rows, out = ab.dispatch(s["x"], r), ab.combine(s["y"], r)
    if not s["case"]["train"]:
        return rows, out
    grads = torch.autograd.grad((rows, out), (s["x"], s["y"], s["weights"]), (s["grows"], s["gout"]))
    return (rows.detach(), out.detach(), *grads)


def _own_product(ab, s):
    out = ab.expert_mm(s["x"], s["weight"], s["ends"])
    if not s["case"]["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["x"], s["weight"]), s["gout"]))


_PLAIN = dict(norm=_plain_norm, route=_plain_route, shuffle=_plain_shuffle, product=_plain_product)
_OWN = dict(norm=_own_norm, route=_own_route, shuffle=_own_shuffle, product=_own_product)


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _PLAIN[case["kind"]](state)
    import adambridge_amd as ab
    if case["train"]:
        return _OWN[case["kind"]](ab, state)
    with torch.no_grad():
        return _OWN[case["kind"]](ab, state)


# ------------------------------------------------------------------- 64 bits

def _exact_norm(case, s):
    """The definition, differentiated by autograd, in slices of rows."""
    outs, dxs, dw, db = [], [], 0.0, 0.0
    for lo in range(0, case["rows"], 8192):
        x = s["x"].detach()[lo:lo + 8192].double().requires_grad_()
        w, b = (s[n].detach().double().requires_grad_() for n in ("weight", "bias"))
        with torch.enable_grad():
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            y = (x - mean) / (var + EPS).sqrt() * w + b
        outs.append(y.detach())
        if case["train"]:
            gx, gw, gb = torch.autograd.grad(y, (x, w, b), s["gout"][lo:lo + 8192].double())
            dxs.append(gx)
            dw, db = dw + gw, db + gb
    if not case["train"]:
        return torch.cat(outs)
    return torch.cat(outs), torch.cat(dxs), dw, db


def _exact_route(case, s):
    logits = s["logits"].detach().double().requires_grad_()
    experts, k = case["experts"], case["top_k"]
    # the k largest one by one, the lowest index of equal ones
    left, chosen = logits.detach().clone(), []
    for _ in range(k):
        best = left.amax(1, keepdim=True)
        index = torch.arange(experts, device=DEVICE).expand_as(left)
        at = torch.where(left == best, index, experts).amin(1)
        chosen.append(at)
        left[torch.arange(case["tokens"], device=DEVICE), at] = -torch.inf
    chosen = torch.stack(chosen, 1)
    with torch.enable_grad():
        if case["normalize"]:
            weights = torch.softmax(torch.gather(logits, 1, chosen), 1)
        else:
            weights = torch.gather(torch.softmax(logits, 1), 1, chosen)
    # an assignment's row: the rows of earlier experts, and earlier tokens of its own
    hot = torch.zeros(case["tokens"], experts, dtype=torch.int64, device=DEVICE).scatter_(1, chosen, 1)
    ends = hot.sum(0).cumsum(0)
    position = (ends - hot.sum(0))[chosen] + torch.gather(hot.cumsum(0) - hot, 1, chosen)
    order = torch.argsort(position.reshape(-1))
    out = [weights.detach(), chosen, ends, order, position]
    if case["train"]:
        out += torch.autograd.grad(weights, (logits,), s["gout"].double())
    return out


def _exact_shuffle(case, s):
    k = case["top_k"]
    x, y, w = (s[n].detach().double() for n in ("x", "y", "weights"))
    place = s["position"].long()
    rows = torch.empty_like(y)
    out = torch.zeros_like(x)
    for j in range(k):
        rows[place[:, j]] = x
        out += w[:, j:j + 1] * y[place[:, j]]
    if not case["train"]:
        return rows, out
    grows, gout = s["grows"].double(), s["gout"].double()
    dx, dy, dw = torch.zeros_like(x), torch.empty_like(y), torch.empty_like(w)
    for j in range(k):
        dx += grows[place[:, j]]
        dy[place[:, j]] = w[:, j:j + 1] * gout
        dw[:, j] = (gout * y[place[:, j]]).sum(1)
    return rows, out, dx, dy, dw


def _exact_product(case, s):
    """Expert by expert."""
    x, weight = s["x"].detach(), s["weight"].detach()
    out = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=DEVICE)
    dx = torch.zeros(case["rows"], case["k"], dtype=torch.float64, device=DEVICE) if case["train"] else None
    dw = torch.zeros(weight.shape, dtype=torch.float64, device=DEVICE) if case["train"] else None
    lo = 0
    for e, hi in enumerate(s["ends"].tolist()):
        if hi > lo:
            xe, we = x[lo:hi].double(), weight[e].double()
            out[lo:hi] = xe @ we.t()
            if case["train"]:
                ge = s["gout"][lo:hi].double()
                dx[lo:hi] = ge @ we
                dw[e] = ge.t() @ xe
        lo = hi
    return (out, dx, dw) if case["train"] else out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return dict(norm=_exact_norm, route=_exact_route, shuffle=_exact_shuffle, product=_exact_product)[case["kind"]](case, s)


# ------------------------------------------------------------------------ work

def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    train = case["train"]
    if case["kind"] == "norm":
        n, cols = case["rows"] * case["cols"], case["cols"]
        return dict(bytes=size * ((4 * n + 4 * cols) if train else (2 * n + 2 * cols)), flops=(18 if train else 8) * n)
    if case["kind"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        small = t * k * 16 + e * 4
        return dict(bytes=size * t * e * (2 if train else 1) + small + (t * k * 4 if train else 0), flops=(8 if train else 4) * t * e)
    if case["kind"] == "shuffle":
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        indexes = t * k * 12
        return dict(bytes=size * h * (t + t * k) * (4 if train else 2) + indexes + (t * k * 4 if train else 0),
                    flops=(6 if train else 2) * t * k * h)
    m, n, k = case["rows"], case["n"], case["k"]
    # the experts that have rows: all where rows are many, at most one a row
    active = min(case["experts"], m)
    if train:
        moved = 2 * m * (n + k) + active * n * k + case["experts"] * n * k
    else:
        moved = m * (n + k) + active * n * k
    return dict(bytes=size * moved, flops=(6 if train else 2) * m * n * k)
