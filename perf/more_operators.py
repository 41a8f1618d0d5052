"""What the token operators are measured on: ``embed_rows``, ``dropout``, ``log_probs`` and
``quantized_matmul`` over the sizes they are used at.

A case is a dict: ``op`` (which operator), ``train`` (the backward pass too), ``dtype`` of the
operands and the sizes: N positions (rows), V tokens, D features in, F features out.  ``prepare``
makes what a program holds before the call, ``run`` is the call (``own``: the package's kernels,
else the plain form in elementary torch operations, in 32 bits), ``exact`` is the same from the
definitions in 64 bits.
"""

import math

import torch

own = False

MASK32 = 0xFFFFFFFF


def listed():
    return [
        # One token of a serving step: the launch is all it costs.
        dict(name="embed_one_token", op="embed", train=False, dtype="float16", N=1, V=32_768, D=1024, skewed=True,
             padded=False, scale=32.0),
        # A training step's tokens, the first few of them in most places, padding at the end of every sequence.
        dict(name="embed_train", op="embed", train=True, dtype="bfloat16", N=16_384, V=65_536, D=2048, skewed=True,
             padded=True, scale=1.0),
        # Labels of a mixture of 500 components as codes, each a hundred odd fp32 features, 200 places for every code.
        dict(name="embed_train_f32_codes", op="embed", train=True, dtype="float32", N=100_003, V=500, D=100,
             skewed=False, padded=False, scale=0.1),
        # A training step's rows dropped and added to what passed by: bytes.
        dict(name="dropout_train_residual", op="dropout", train=True, dtype="bfloat16", N=16_384, D=4096, p=0.1,
             residual=True),
        # fp32 features of odd width and count.
        dict(name="dropout_train_f32_d77", op="dropout", train=True, dtype="float32", N=100_003, D=77, p=0.5,
             residual=False),
        # A serving step's one row: the sampled token's log probability and the alternatives beside it.
        dict(name="logp_one_row", op="logp", train=False, dtype="float16", N=1, V=65_536, top_k=5, masked=False),
        # A serving step's rows in fp32, an odd vocabulary, some tokens forbidden, many alternatives.
        dict(name="logp_top_masked", op="logp", train=False, dtype="float32", N=130, V=32_001, top_k=20, masked=True),
        # The loss of a training step over a large vocabulary, with an entropy term.
        dict(name="logp_train", op="logp", train=True, dtype="bfloat16", N=8192, V=65_536, top_k=0, masked=False),
        # The loss over a mixture's 500 codes: many short rows.
        dict(name="logp_train_f32_codes", op="logp", train=True, dtype="float32", N=100_003, V=500, top_k=0,
             masked=False),
        # Four rows in a serving step: the weights' bytes.
        dict(name="int8_four_rows", op="int8", train=False, dtype="bfloat16", N=4, D=4096, F=8192, bias=True),
        # A prompt, odd in all sizes.
        dict(name="int8_prompt_odd", op="int8", train=False, dtype="float16", N=1531, D=1000, F=1777, bias=True),
        # Many rows: the largest of the matrix work.
        dict(name="int8_many_rows", op="int8", train=False, dtype="bfloat16", N=16_384, D=4096, F=8192, bias=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embed", "dropout", "logp", "int8"))
    case = dict(op=op, train=rng.random() < 0.6, dtype=rng.choice(("float32", "bfloat16", "float16")))
    wide = case["dtype"] == "float32"     # (as many bytes as the listed ones, not more)
    if op == "embed":
        case["D"] = _log_uniform(rng, 16, 4096)
        case["V"] = min(_log_uniform(rng, 2, 131_072), (1 << (26 if wide else 27)) // case["D"])
        case["N"] = min(_log_uniform(rng, 1, 131_072), (1 << (24 if wide else 25)) // case["D"])
        case["skewed"], case["padded"] = rng.random() < 0.7, rng.random() < 0.5
        case["scale"] = rng.choice((1.0, 0.1, math.sqrt(case["D"])))
    elif op == "dropout":
        case["D"] = _log_uniform(rng, 16, 8192)
        case["N"] = min(_log_uniform(rng, 1, 200_000), (1 << (25 if wide else 26)) // case["D"])
        case["p"], case["residual"] = round(rng.uniform(0.0, 0.9), 3), rng.random() < 0.5
    elif op == "logp":
        case["V"] = _log_uniform(rng, 2, 131_072)
        case["top_k"] = rng.choice((0, 0, rng.randint(1, min(20, case["V"]))))
        most = (1 << 24) if case["top_k"] else (1 << (28 if wide else 29))
        case["N"] = max(1, min(_log_uniform(rng, 1, 200_000), most // case["V"]))
        case["masked"] = rng.random() < 0.5
    else:
        case["train"] = False
        case["D"], case["F"] = (_log_uniform(rng, 16, 8192) for _ in range(2))
        if rng.random() < 0.5:   # half of them as layers are mostly sized
            case["D"], case["F"] = (-(-case[v] // 64) * 64 for v in "DF")
        case["N"] = max(1, min(_log_uniform(rng, 1, 65_536), (1 << 39) // (case["D"] * case["F"]),
                               (1 << 27) // max(case["D"], case["F"])))
        case["bias"] = rng.random() < 0.5
    return case


# --- inputs -----------------------------------------------------------------

def _generator(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return dev, torch.Generator(device=dev).manual_seed(int(seed))


def _tokens(case, g, dev):
    """Tokens: uniform, or the lower the likelier (v with probability log((v + 2) / (v + 1)) / log(V + 1))."""
    n, v = case["N"], case["V"]
    u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    t = torch.floor(torch.exp(u * math.log(v + 1.0)) - 1.0) if case.get("skewed", True) else torch.floor(u * v)
    return t.long().clamp_(0, v - 1)


def _scores(case, g, dev, index):
    """Scores with some tokens liked more than others; masked ones at -inf, or at the type's lowest value in every
    third row, but not the given ones; some rows without any."""
    n, v = case["N"], case["V"]
    dt = getattr(torch, case["dtype"])
    s = torch.randn((n, v), generator=g, device=dev).mul_(2.0)
    s += 1.5 * torch.randn((v,), generator=g, device=dev)
    s = s.to(dt)
    if case["masked"]:
        off = torch.rand((n, v), generator=g, device=dev) < 0.25
        off.scatter_(1, index[:, None], False)
        off |= (torch.arange(n, device=dev) % 97 == 5)[:, None]
        s.masked_fill_(off, -math.inf)
        s.masked_fill_(off & (torch.arange(n, device=dev) % 3 == 0)[:, None], torch.finfo(dt).min)
    return s


def _quantized(w):
    """A matrix's rows in 8 bits, and their scales: laid out as the package's quantize_rows does, in rows of whole
    128 bytes."""
    f, d = w.shape
    values, scales = _plain_quantize(w)
    room = torch.zeros((f, -(-d // 128) * 128), dtype=torch.int8, device=w.device)
    room[:, :d] = values.to(torch.int8)
    return room[:, :d], scales


def prepare(case, seed):
    dev, g = _generator(seed)
    dt = getattr(torch, case["dtype"])
    randn = lambda *s: torch.randn(s, generator=g, device=dev)    # noqa: E731
    n = case["N"]
    s = dict(case)
    if case["op"] == "embed":
        v, d = case["V"], case["D"]
        s.update(table=randn(v, d).to(dt), index=_tokens(case, g, dev))
        if case["padded"]:      # sequences of 512 places, an eighth of each on average unused
            used = 512 - torch.randint(0, 129, (-(-n // 512),), generator=g, device=dev)
            at = torch.arange(n, device=dev)
            s["index"] = torch.where(at % 512 < used[at // 512], s["index"], -1)
        if case["train"]:
            s["dy"] = randn(n, d).to(dt)
    elif case["op"] == "dropout":
        d = case["D"]
        s.update(x=randn(n, d).to(dt), seed=int(torch.randint(0, 1 << 62, (1,), generator=torch.Generator().manual_seed(
            int(seed)))), offset=int(seed) % 1000)
        s["passed"] = randn(n, d).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(n, d).to(dt)
    elif case["op"] == "logp":
        s["index"] = _tokens(case, g, dev)
        s["scores"] = _scores(case, g, dev, s["index"])
        s["index"][torch.arange(n, device=dev) % 31 == 7] = -1       # places that do not count
        if case["train"]:
            s.update(dchosen=-torch.rand(n, generator=g, device=dev), dentropy=0.1 * randn(n),
                     dtop=randn(n, case["top_k"]))
    else:
        d, f = case["D"], case["F"]
        s["x"] = (randn(n, d) * (0.5 + torch.rand((n, 1), generator=g, device=dev))).to(dt)
        s["values"], s["scales"] = _quantized(randn(f, d) / math.sqrt(d))
        s["b"] = (0.1 * randn(f)).to(dt) if case["bias"] else None
    return s


# --- the package's operators ------------------------------------------------

def _leaf(t):
    return t.detach().requires_grad_()


def _own_embed(s):
    import gmmxx_amd

    if not s["train"]:
        return gmmxx_amd.embed_rows(s["table"], s["index"], scale=s["scale"])
    table = _leaf(s["table"])
    y = gmmxx_amd.embed_rows(table, s["index"], scale=s["scale"])
    return (y, *torch.autograd.grad(y, (table,), s["dy"]))


def _own_dropout(s):
    import gmmxx_amd

    if not s["train"]:
        return gmmxx_amd.dropout(s["x"], s["p"], s["seed"], offset=s["offset"], residual=s["passed"])
    leaves = [_leaf(t) for t in (s["x"], s["passed"]) if t is not None]
    y = gmmxx_amd.dropout(leaves[0], s["p"], s["seed"], offset=s["offset"],
                          residual=leaves[1] if s["residual"] else None)
    return (y, *torch.autograd.grad(y, leaves, s["dy"]))


def _own_logp(s):
    import gmmxx_amd

    if not s["train"]:
        return tuple(gmmxx_amd.log_probs(s["scores"], s["index"], top_k=s["top_k"]))
    scores = _leaf(s["scores"])
    r = gmmxx_amd.log_probs(scores, s["index"], top_k=s["top_k"])
    some = s["top_k"] > 0
    ds, = torch.autograd.grad((r.chosen, r.entropy) + ((r.top,) if some else ()), (scores,),
                              (s["dchosen"], s["dentropy"]) + ((s["dtop"],) if some else ()))
    return (*r, ds)


def _own_int8(s):
    import gmmxx_amd

    return gmmxx_amd.quantized_matmul(s["x"], gmmxx_amd.Quantized(s["values"], s["scales"]), s["b"])


# --- their plain form -------------------------------------------------------

def _plain_embed(s):
    table, index = s["table"], s["index"]
    there = (index >= 0) & (index < s["V"])
    at = torch.where(there, index, 0)
    y = torch.where(there[:, None], table[at].float() * s["scale"], 0.0).to(table.dtype)
    if not s["train"]:
        return y
    dy = torch.where(there[:, None], s["dy"].float(), 0.0)
    dtable = torch.zeros(table.shape, dtype=torch.float32, device=table.device).index_add_(0, at, dy)
    return y, (dtable * s["scale"]).to(table.dtype)


def _plain_words(count, seed, offset, device):
    """The first `count` words of Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) with key `seed`: word i is
    word i % 4 of counter (i / 4, offset)."""
    c0 = torch.arange(-(-count // 4), device=device)
    c1 = c0 >> 32
    c0 = c0 & MASK32
    c2, c3 = torch.full_like(c0, offset & MASK32), torch.full_like(c0, (offset >> 32) & MASK32)
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57        # (mod 2^64: the high word is that of the true product)
        c0, c1, c2, c3 = ((q >> 32) & MASK32) ^ c1 ^ k0, q & MASK32, ((p >> 32) & MASK32) ^ c3 ^ k1, p & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:count]


def _plain_dropout(s):
    x = s["x"]
    border = round(s["p"] * 2.0 ** 32)      # kept: words from here on
    keep = (_plain_words(x.numel(), s["seed"], s["offset"], x.device) >= border).reshape(x.shape)
    scale = 1.0 / (1.0 - s["p"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"]:
        y = y + s["passed"].float()
    y = y.to(x.dtype)
    if not s["train"]:
        return y
    dx = torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)
    return (y, dx, s["dy"]) if s["residual"] else (y, dx)


def _plain_logp(s):
    scores, index, k = s["scores"], s["index"], s["top_k"]
    n, v = scores.shape
    x = scores.float()
    there = x > -math.inf                      # candidates: neither -inf nor NaN
    x = torch.where(there, x, -math.inf)
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    d = torch.where(x == m, 0.0, x - m)        # (where there are none, or +inf)
    d = torch.where(there, d, -math.inf)
    w = torch.exp(d)
    z = torch.where(some, w.sum(1, keepdim=True), 1.0)
    logz = torch.log(z)
    u = torch.where(w > 0, w * d, 0.0).sum(1, keepdim=True)
    entropy = torch.where(some, logz - u / z, 0.0)
    counts = ((index >= 0) & (index < v))[:, None]
    at = torch.where(counts[:, 0], index, 0)[:, None]
    chosen = torch.where(counts, d.gather(1, at) - logz, 0.0)[:, 0]
    if k:
        top, place = torch.sort(x, dim=1, descending=True, stable=True)
        place = place[:, :k]
        top = d.gather(1, place) - logz
        place = torch.where(top > -math.inf, place, -1).int()
        # (a candidate whose difference to the largest passes fp32 still is one)
        place = torch.where(there.gather(1, place.clamp(min=0).long()), place, -1)
    else:
        top, place = torch.zeros((n, 0), device=x.device), torch.zeros((n, 0), dtype=torch.int32, device=x.device)
    out = (chosen, entropy[:, 0], top, place)
    if not s["train"]:
        return out
    p = w / z
    dc = torch.where(counts & some, s["dchosen"][:, None], 0.0)
    dt = torch.where(place >= 0, s["dtop"], 0.0)
    whole = dc + dt.sum(1, keepdim=True)
    ds = p * (-whole - s["dentropy"][:, None] * (torch.where(p > 0, d - logz, 0.0) + entropy))
    ds.scatter_add_(1, at, torch.where(there.gather(1, at), dc, 0.0))
    if k:
        ds.scatter_add_(1, place.clamp(min=0).long(), dt)
    return (*out, ds.to(scores.dtype))


def _plain_quantize(x):
    """Whole numbers from -127 to 127 (as floats) and the scale of each row."""
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    by = torch.where(most > 0, 127.0 / most, 0.0)
    return torch.round(x * by), (most / 127.0)[:, 0]


def _plain_int8(s):
    q, scale = _plain_quantize(s["x"])
    w = s["values"].float()
    # (a product of more than 1040 pairs can pass 2^24: parts that are exact, added in 64 bits)
    y = torch.zeros((q.shape[0], w.shape[0]), dtype=torch.float64, device=q.device)
    for i in range(0, q.shape[1], 1024):
        y += q[:, i:i + 1024] @ w[:, i:i + 1024].t()
    y = y.float() * (scale[:, None] * s["scales"])
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(s["x"].dtype)


_OWN = {"embed": _own_embed, "dropout": _own_dropout, "logp": _own_logp, "int8": _own_int8}
_PLAIN = {"embed": _plain_embed, "dropout": _plain_dropout, "logp": _plain_logp, "int8": _plain_int8}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# --- the definitions in 64 bits ---------------------------------------------

def _exact_embed(s):
    v, d = s["table"].shape
    rows = torch.cat([s["table"].double(), torch.zeros((1, d), dtype=torch.float64, device=s["table"].device)])
    at = torch.where((s["index"] < 0) | (s["index"] >= v), v, s["index"])
    y = rows[at] * s["scale"]
    if not s["train"]:
        return y
    order = torch.argsort(at, stable=True)
    ends = torch.searchsorted(at[order], torch.arange(v + 1, device=at.device))
    total = torch.zeros_like(rows)
    for i in range(0, d, 256):        # sums of runs, columns by columns
        part = s["dy"][:, i:i + 256].double()
        total[:, i:i + 256].index_add_(0, at[order], part[order])
    total = torch.where((ends[1:] > ends[:-1])[:, None], total[:v], 0.0)
    return y, total * s["scale"]


def _mul32(a, b):
    """High and low words of a b, by 16-bit halves."""
    al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    low, mid = al * bl, ah * bl
    mid = mid + (low >> 16)
    cross = al * bh + (mid & 0xFFFF)
    return ah * bh + (mid >> 16) + (cross >> 16), ((cross & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_dropout(s):
    x = s["x"]
    n = x.numel()
    i = torch.arange((n + 3) // 4, device=x.device)
    state = [i % (1 << 32), i // (1 << 32), torch.zeros_like(i) + s["offset"] % (1 << 32),
             torch.zeros_like(i) + s["offset"] // (1 << 32)]
    key = [s["seed"] % (1 << 32), s["seed"] // (1 << 32)]
    for _ in range(10):
        hi0, lo0 = _mul32(state[0], 0xD2511F53)
        hi1, lo1 = _mul32(state[2], 0xCD9E8D57)
        state = [hi1 ^ state[1] ^ key[0], lo1, hi0 ^ state[3] ^ key[1], lo0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    uniform = torch.stack(state, 1).flatten()[:n].double() / 2.0 ** 32
    keep = (uniform >= round(s["p"] * 2.0 ** 32) / 2.0 ** 32).reshape(x.shape).double()
    y = x.double() * keep / (1.0 - s["p"])
    if s["residual"]:
        y = y + s["passed"].double()
    if not s["train"]:
        return y
    dx = s["dy"].double() * keep / (1.0 - s["p"])
    return (y, dx, s["dy"].double()) if s["residual"] else (y, dx)


def _exact_logp(s):
    n, v = s["scores"].shape
    k, train = s["top_k"], s["train"]
    parts = []
    step = max(1, (1 << 27) // v)
    for i in range(0, n, step):
        x, t = s["scores"][i:i + step].double(), s["index"][i:i + step]
        r = torch.arange(x.shape[0], device=x.device)
        there = x > -math.inf
        none = ~there.any(1)
        x = torch.where(there, x, -math.inf)
        logs = torch.where(none[:, None], -math.inf, torch.log_softmax(x, 1))
        p = torch.exp(logs)
        plogp = torch.xlogy(p, p)
        h = -plogp.sum(1)
        counts = (t >= 0) & (t < v)
        at = torch.where(counts, t, 0)
        chosen = torch.where(counts, logs[r, at], 0.0)
        left, best, where = logs.clone() if k else None, [], []
        for _ in range(k):
            j = left.argmax(1)      # (a tie's value is the same whichever of them is taken)
            best.append(left[r, j])
            where.append(j)
            left[r, j] = -math.inf
        top = torch.stack(best, 1) if k else x.new_zeros((x.shape[0], 0))
        out = [chosen, h, top]
        if train:
            dc = torch.where(counts & ~none, s["dchosen"][i:i + step].double(), 0.0)
            dh = s["dentropy"][i:i + step].double()
            ds = -dh[:, None] * (plogp + p * h[:, None]) - dc[:, None] * p
            ds[r, at] += torch.where(there[r, at], dc, 0.0)
            if k:
                place = torch.argsort(-x, dim=1, stable=True)[:, :k]
                dt = torch.where(there.gather(1, place), s["dtop"][i:i + step].double(), 0.0)
                ds -= dt.sum(1, keepdim=True) * p
                ds.scatter_add_(1, place, dt)
            out.append(ds)
        parts.append(out)
    out = [torch.cat(c) for c in zip(*parts)]
    return (*out[:3], None, *out[3:])


def _exact_int8(s):
    # The 8-bit values are those of fp32 arithmetic by definition; everything after them is exact.
    x = s["x"].double()
    most = x.abs().max(1).values
    by = torch.where(most > 0, 127.0 / most, 0.0).float().double()
    q = torch.round((x * by[:, None]).float()).double()
    y = (q @ s["values"].double().t()) * (most / 127.0)[:, None] * s["scales"].double()
    return y if s["b"] is None else y + s["b"].double()


def exact(case, seed):
    return {"embed": _exact_embed, "dropout": _exact_dropout, "logp": _exact_logp,
            "int8": _exact_int8}[case["op"]](prepare(case, seed))


# --- what a pass cannot do without ------------------------------------------

def _distinct(case):
    """How many different tokens N draws are expected to give."""
    n, v = case["N"], case["V"]
    if case["skewed"]:
        t = torch.arange(v, dtype=torch.float64)
        p = torch.log((t + 2.0) / (t + 1.0)) / math.log(v + 1.0)
    else:
        p = torch.full((v,), 1.0 / v, dtype=torch.float64)
    return int((1.0 - torch.exp(n * torch.log1p(-p.clamp(max=1.0 - 1e-12)))).sum())


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    n, train = case["N"], case["train"]
    if case["op"] == "embed":
        v, d = case["V"], case["D"]
        floats = d * (max(_distinct(case), 1) + n)
        if train:
            floats += d * (n + v)
        return {"bytes": size * floats + 8 * n, "flops": n * d * (2 if train else 1)}
    if case["op"] == "dropout":
        nd = n * case["D"]
        return {"bytes": size * nd * (2 + case["residual"] + (2 if train else 0)),
                "flops": nd * (2 + case["residual"] + (2 if train else 0))}
    if case["op"] == "logp":
        v, k = case["V"], case["top_k"]
        return {"bytes": size * n * v * (2 if train else 1) + n * (16 + 8 * k + (8 + 4 * k if train else 0)),
                "flops": n * v * (10 if train else 5)}
    d, f = case["D"], case["F"]
    return {"bytes": size * n * (d + f) + f * d + 4 * f + (size * f if case["bias"] else 0), "flops": 2 * n * d * f}
