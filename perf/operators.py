"""What the sparsely gated layer's operators are measured on: ``layer_norm``, ``route_rows``,
``grouped_matmul`` and ``combine_rows`` over the sizes they are used at.

A case is a dict: ``op`` (which operator), ``train`` (the backward pass too), ``dtype`` of the
operands and the sizes: N rows, E experts of which each row takes ``top_k``, D features in,
F features out.  ``prepare`` makes what a program holds before the call, ``run`` is the call
(``own``: the package's kernels, else the plain form in elementary torch operations, in 32
bits), ``exact`` is the same from the definitions in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # One row of a serving step: the launch is all it costs.
        dict(name="norm_one_row", op="norm", train=False, dtype="float16", N=1, D=1024),
        # A training step's rows, wide: bytes.
        dict(name="norm_train_wide", op="norm", train=True, dtype="bfloat16", N=16_384, D=4096),
        # A table of fp32 features whose width is no power of two, odd row count.
        dict(name="norm_train_f32_d100", op="norm", train=True, dtype="float32", N=100_003, D=100),
        # The gate of three rows in a serving step.
        dict(name="route_three_rows", op="route", train=False, dtype="bfloat16", N=3, E=64, top_k=2, masked=False,
             renormalize=True),
        # A training step's gate: some scores masked out, some rows without any.
        dict(name="route_train_masked", op="route", train=True, dtype="float32", N=65_537, E=64, top_k=8, masked=True,
             renormalize=True),
        # A fitted mixture as the gate: log densities of 500 components, responsibilities kept as they are.
        dict(name="route_mixture_k500", op="route", train=True, dtype="float32", N=100_000, E=500, top_k=4,
             masked=False, renormalize=False),
        # Four rows in a serving step through their experts: the chosen weights' bytes.
        dict(name="experts_four_rows", op="experts", train=False, dtype="bfloat16", N=4, E=16, top_k=2, D=1024,
             F=2048),
        # A whole prompt through its experts, unevenly chosen.
        dict(name="experts_prompt", op="experts", train=False, dtype="float16", N=4099, E=16, top_k=2, D=2048,
             F=1024),
        # A training step of the expert products: the largest of the matrix work.
        dict(name="experts_train", op="experts", train=True, dtype="bfloat16", N=16_384, E=32, top_k=2, D=1024,
             F=2048),
        # Local linear models, one for each of 200 clusters, fp32 and odd sizes.
        dict(name="experts_train_f32_local", op="experts", train=True, dtype="float32", N=100_003, E=200, top_k=1,
             D=100, F=77),
        # Eight rows' results added up in a serving step.
        dict(name="combine_eight_rows", op="combine", train=False, dtype="bfloat16", N=8, E=16, top_k=2, F=1024),
        # A training step's results added up, with the gates' gradient.
        dict(name="combine_train", op="combine", train=True, dtype="bfloat16", N=16_384, E=32, top_k=4, F=2048),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "route", "experts", "combine"))
    case = dict(op=op, train=rng.random() < 0.6, dtype=rng.choice(("float32", "bfloat16", "float16")))
    wide = case["dtype"] == "float32"     # (as many bytes as the listed ones, not more)
    if op == "norm":
        case["D"] = _log_uniform(rng, 16, 8192)
        case["N"] = min(_log_uniform(rng, 1, 200_000), (1 << (25 if wide else 26)) // case["D"])
    elif op == "route":
        case["E"] = _log_uniform(rng, 2, 1024)
        case["top_k"] = rng.randint(1, min(8, case["E"]))
        case["N"] = min(_log_uniform(rng, 1, 200_000), (1 << 26) // case["E"])
        case["masked"], case["renormalize"] = rng.random() < 0.5, rng.random() < 0.5
    elif op == "experts":
        case["E"] = _log_uniform(rng, 2, 256)
        case["top_k"] = rng.randint(1, min(4, case["E"]))
        case["D"], case["F"] = (_log_uniform(rng, 16, 2048) for _ in range(2))
        if rng.random() < 0.5:   # half of them as layers are mostly sized
            case["D"], case["F"] = (-(-case[v] // 64) * 64 for v in "DF")
        # no more weights, and no more products, than the largest listed case
        case["E"] = max(case["top_k"], min(case["E"], (1 << 26) // (case["D"] * case["F"])))
        case["N"] = min(_log_uniform(rng, 1, 131_072), (1 << 36) // (case["D"] * case["F"] * case["top_k"]),
                        (1 << 25) // (max(case["D"], case["F"]) * case["top_k"]))
    else:
        case["E"] = _log_uniform(rng, 2, 256)
        case["top_k"] = rng.randint(1, min(8, case["E"]))
        case["F"] = _log_uniform(rng, 16, 4096)
        case["N"] = min(_log_uniform(rng, 1, 131_072), (1 << (26 if wide else 27)) // (case["F"] * case["top_k"]))
    return case


# --- inputs -----------------------------------------------------------------

def _generator(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return dev, torch.Generator(device=dev).manual_seed(int(seed))


def _scores(case, g, dev):
    """Gate scores with some experts liked more than others; a mixture's log densities where the gates are
    responsibilities; masked ones at -inf, or at the type's lowest value in every third row."""
    n, e = case["N"], case["E"]
    if case.get("renormalize", True):
        s = torch.randn((n, e), generator=g, device=dev) + 0.7 * torch.randn((e,), generator=g, device=dev)
    else:
        s = -60.0 + 8.0 * torch.randn((n, e), generator=g, device=dev)
    s = s.to(getattr(torch, case["dtype"]))
    if case.get("masked"):
        off = torch.rand((n, e), generator=g, device=dev) < 0.25
        off |= (torch.arange(n, device=dev) % 97 == 5)[:, None]
        s = s.masked_fill(off, -math.inf)
        low = off & (torch.arange(n, device=dev) % 3 == 0)[:, None]
        s = s.masked_fill(low, torch.finfo(s.dtype).min)
    return s


def _groups(case, g, dev):
    """A routing of N rows as a program holds it: experts and gates of each row, the groups' offsets, the row at
    each grouped position, the position of each choice."""
    n, e, k = case["N"], case["E"], case["top_k"]
    score = torch.randn((n, e), generator=g, device=dev) + 0.3 * torch.randn((e,), generator=g, device=dev)
    top, experts = score.topk(k, dim=1)
    flat = experts.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=dev)
    offsets[1:] = torch.cumsum(torch.bincount(flat, minlength=e), 0)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k, device=dev)
    return dict(experts=experts.int(), gates=torch.softmax(top, 1), offsets=offsets.int(),
                rows=torch.div(order, k, rounding_mode="floor").int(), slots=slots.reshape(n, k).int(),
                largest=int((offsets[1:] - offsets[:-1]).max()))


def prepare(case, seed):
    dev, g = _generator(seed)
    dt = getattr(torch, case["dtype"])
    randn = lambda *s: torch.randn(s, generator=g, device=dev)    # noqa: E731
    n = case["N"]
    s = dict(case)
    if case["op"] == "norm":
        d = case["D"]
        s.update(x=(randn(n, d) * (0.5 + torch.rand((n, 1), generator=g, device=dev)) + randn(n, 1)).to(dt),
                 weight=(1.0 + 0.1 * randn(d)).to(dt), bias=(0.1 * randn(d)).to(dt))
        if case["train"]:
            s["dy"] = randn(n, d).to(dt)
    elif case["op"] == "route":
        s["scores"] = _scores(case, g, dev)
        if case["train"]:
            s["dgates"] = randn(n, case["top_k"])
    elif case["op"] == "experts":
        e, d, f = case["E"], case["D"], case["F"]
        s.update(_groups(case, g, dev), x=randn(n, d).to(dt), weight=(randn(e, d, f) / math.sqrt(d)).to(dt),
                 bias=(0.1 * randn(e, f)).to(dt))
        if case["train"]:
            s["dy"] = randn(n * case["top_k"], f).to(dt)
    else:
        s.update(_groups(case, g, dev), y=randn(n * case["top_k"], case["F"]).to(dt))
        if case["train"]:
            s["dout"] = randn(n, case["F"]).to(dt)
    return s


# --- the package's operators ------------------------------------------------

def _leaf(t):
    return t.detach().requires_grad_()


def _routing(s):
    import gmmxx_amd

    return gmmxx_amd.Routing(s["experts"], s["gates"], s["offsets"], s["rows"], s["slots"])


def _own_norm(s):
    import gmmxx_amd

    if not s["train"]:
        return gmmxx_amd.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
    y = gmmxx_amd.layer_norm(x, w, b, eps=EPS)
    return (y, *torch.autograd.grad(y, (x, w, b), s["dy"]))


def _own_route(s):
    import gmmxx_amd

    if not s["train"]:
        return tuple(gmmxx_amd.route_rows(s["scores"], s["top_k"], renormalize=s["renormalize"]))
    scores = _leaf(s["scores"])
    r = gmmxx_amd.route_rows(scores, s["top_k"], renormalize=s["renormalize"])
    return (*r, *torch.autograd.grad(r.gates, (scores,), s["dgates"]))


def _own_experts(s):
    import gmmxx_amd

    if not s["train"]:
        return gmmxx_amd.grouped_matmul(s["x"], s["weight"], _routing(s), bias=s["bias"])
    x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
    y = gmmxx_amd.grouped_matmul(x, w, _routing(s), bias=b)
    return (y, *torch.autograd.grad(y, (x, w, b), s["dy"]))


def _own_combine(s):
    import gmmxx_amd

    if not s["train"]:
        return gmmxx_amd.combine_rows(s["y"], _routing(s))
    y, gates = _leaf(s["y"]), _leaf(s["gates"])
    out = gmmxx_amd.combine_rows(y, _routing(s), gates)
    return (out, *torch.autograd.grad(out, (y, gates), s["dout"]))


# --- their plain form -------------------------------------------------------

def _plain_norm(s):
    x, w = s["x"].float(), s["weight"].float()
    dt = s["x"].dtype
    d = x.shape[1]
    c = x - x.sum(1, keepdim=True) / d
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / d + EPS)
    xh = c * rstd
    y = (xh * w + s["bias"].float()).to(dt)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.sum(1, keepdim=True) / d - xh * ((gw * xh).sum(1, keepdim=True) / d))
    return y, dx.to(dt), (dy * xh).sum(0).to(dt), dy.sum(0).to(dt)


def _plain_route(s):
    scores, k = s["scores"], s["top_k"]
    n, e = scores.shape
    v = scores.float()
    ranked, index = torch.sort(v, dim=1, descending=True, stable=True)
    top, index = ranked[:, :k], index[:, :k]
    there = top > -math.inf
    best = torch.where(there[:, :1], top[:, :1], 0.0)
    weight = torch.exp(top - best)
    whole = (weight if s["renormalize"] else torch.exp(v - best)).sum(1, keepdim=True)
    whole = torch.where(there[:, :1], whole, 1.0)
    gates = weight / whole
    experts = torch.where(there, index, -1).int()
    flat = torch.where(there, index, e).reshape(-1)       # absent choices come last
    order = torch.sort(flat, stable=True).indices
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=v.device)
    offsets[1:] = torch.searchsorted(flat[order], torch.arange(e, device=v.device), right=True)
    rows = torch.div(order, k, rounding_mode="floor").int()
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k, device=v.device)
    out = (experts, gates, offsets, rows, slots.reshape(n, k).int())
    if not s["train"]:
        return out
    dg = s["dgates"]
    mean = (gates * dg).sum(1, keepdim=True)
    if s["renormalize"]:
        ds = torch.zeros_like(v).scatter_(1, index, gates * (dg - mean))
    else:
        ds = (-mean * torch.exp(v - best) / whole).scatter_add_(1, index, gates * dg)
    return (*out, ds.to(scores.dtype))


def _plain_experts(s):
    dt, x, bias = s["x"].dtype, s["x"].float(), s["bias"].float()
    rows, slots, offsets = s["rows"].long(), s["slots"].long(), s["offsets"].long()
    m, e, f = rows.shape[0], s["E"], s["F"]
    at = torch.arange(m, device=x.device)
    expert = torch.searchsorted(offsets[1:], at, right=True)
    if not s["train"] and m <= e:      # few positions: each one's own matrix
        return (torch.bmm(x[rows][:, None, :], s["weight"][expert].float())[:, 0] + bias[expert]).to(dt)
    w = s["weight"].float()
    # the groups side by side, filled up to the largest with rows of zeros
    place = expert * s["largest"] + at - offsets[expert]
    xg = x.new_zeros((e * s["largest"], x.shape[1]))
    xg[place] = x[rows]
    xg = xg.reshape(e, s["largest"], -1)
    y = (torch.bmm(xg, w) + bias[:, None, :]).reshape(-1, f)[place].to(dt)
    if not s["train"]:
        return y
    dyg = x.new_zeros((e * s["largest"], f))
    dyg[place] = s["dy"].float()
    dyg = dyg.reshape(e, s["largest"], f)
    dxg = torch.bmm(dyg, w.transpose(1, 2)).reshape(e * s["largest"], -1)
    dx = dxg[place[slots]].sum(1)
    return y, dx.to(dt), torch.bmm(xg.transpose(1, 2), dyg).to(dt), dyg.sum(1).to(dt)


def _plain_combine(s):
    y, gates, slots = s["y"], s["gates"], s["slots"].long()
    picked = y[slots].float()
    out = (picked * gates[:, :, None]).sum(1).to(y.dtype)
    if not s["train"]:
        return out
    dout = s["dout"].float()
    dy = torch.empty_like(y)
    dy[slots.reshape(-1)] = (dout[:, None, :] * gates[:, :, None]).reshape(y.shape).to(y.dtype)
    return out, dy, (picked * dout[:, None, :]).sum(2)


_OWN = {"norm": _own_norm, "route": _own_route, "experts": _own_experts, "combine": _own_combine}
_PLAIN = {"norm": _plain_norm, "route": _plain_route, "experts": _plain_experts, "combine": _plain_combine}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# --- the definitions in 64 bits ---------------------------------------------

def _exact_norm(s):
    leaves = [s[v].double().requires_grad_() for v in ("x", "weight", "bias")]
    var, mean = torch.var_mean(leaves[0], dim=1, keepdim=True, unbiased=False)
    y = (leaves[0] - mean) * torch.rsqrt(var + EPS) * leaves[1] + leaves[2]
    if not s["train"]:
        return y
    return (y, *torch.autograd.grad(y, leaves, s["dy"].double()))


def _exact_route(s):
    v, k = s["scores"].double(), s["top_k"]
    left, gates = v.clone(), []
    full = torch.where((left > -math.inf).any(1, keepdim=True), torch.log_softmax(v, 1), -math.inf)
    for _ in range(k):
        i = left.argmax(1, keepdim=True)     # (a tie's value is the same whichever of them is taken)
        gates.append(torch.where(left.gather(1, i) > -math.inf, full.gather(1, i), -math.inf))
        left = left.scatter(1, i, -math.inf)
    logs = torch.cat(gates, 1)
    p = torch.exp(logs)
    if s["renormalize"]:
        # (over the chosen alone, from differences to the largest: the sum over all may vanish beside them)
        best = torch.where(logs[:, :1] > -math.inf, logs[:, :1], 0.0)
        w = torch.exp(logs - best)
        p = w / torch.where(logs[:, :1] > -math.inf, w.sum(1, keepdim=True), 1.0)
    out = (None, p, None, None, None)
    if not s["train"]:
        return out
    # the gradient from its formula at the gates above, row by row; a tie's lower index comes first
    dg = s["dgates"].double()
    mean = (p * dg).sum(1, keepdim=True)
    place = torch.argsort(-v, dim=1, stable=True)[:, :k]
    if s["renormalize"]:
        ds = torch.zeros_like(v).scatter_(1, place, p * (dg - mean))
    else:
        ds = -mean * torch.exp(full)
        ds.scatter_(1, place, ds.gather(1, place) + p * dg)
    return (*out, ds)


def _exact_experts(s):
    x, w, b = (s[v].double() for v in ("x", "weight", "bias"))
    ends, rows = s["offsets"].tolist(), s["rows"].long()
    y = x.new_zeros((rows.shape[0], s["F"]))
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for e in range(s["E"]):
        at = slice(ends[e], ends[e + 1])
        xe = x[rows[at]]
        y[at] = xe @ w[e] + b[e]
        if s["train"]:
            de = s["dy"][at].double()
            dx.index_add_(0, rows[at], de @ w[e].t())
            dw[e] = xe.t() @ de
            db[e] = de.sum(0)
    return (y, dx, dw, db) if s["train"] else y


def _exact_combine(s):
    y, g, slots = s["y"].double(), s["gates"].double(), s["slots"].long()
    out = y.new_zeros((slots.shape[0], y.shape[1]))
    for j in range(slots.shape[1]):
        out += g[:, j, None] * y[slots[:, j]]
    if not s["train"]:
        return out
    dout, dy, dg = s["dout"].double(), torch.zeros_like(y), torch.zeros_like(g)
    for j in range(slots.shape[1]):
        dy[slots[:, j]] = g[:, j, None] * dout
        dg[:, j] = (dout * y[slots[:, j]]).sum(1)
    return out, dy, dg


def exact(case, seed):
    with torch.enable_grad():
        out = {"norm": _exact_norm, "route": _exact_route, "experts": _exact_experts,
               "combine": _exact_combine}[case["op"]](prepare(case, seed))
    return tuple(v if v is None else v.detach() for v in out) if isinstance(out, tuple) else out.detach()


# --- what a pass cannot do without ------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    n, train = case["N"], case["train"]
    if case["op"] == "norm":
        nd = n * case["D"]
        return {"bytes": size * ((4 if train else 2) * nd + (4 if train else 2) * case["D"]),
                "flops": (19 if train else 8) * nd}
    k, e = case["top_k"], case["E"]
    m = n * k
    if case["op"] == "route":
        return {"bytes": size * n * e * (2 if train else 1) + 4 * m * (5 if train else 4) + 4 * (e + 1),
                "flops": n * e * (3 if train else 2)}
    f = case["F"]
    if case["op"] == "experts":
        d, used = case["D"], min(e, m)
        floats = n * d + used * (d + 1) * f + m * f
        if train:
            floats += n * d + e * (d + 1) * f + m * f
        return {"bytes": size * floats + 4 * (e + 1) + 4 * m * (2 if train else 1),
                "flops": 2 * m * d * f * (3 if train else 1)}
    return {"bytes": size * f * ((2 * n + 2 * m) if train else (n + m)) + 4 * m * (3 if train else 2),
            "flops": m * f * (5 if train else 2)}
