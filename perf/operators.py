"""Cases, plain forms and 64-bit oracles of the training operators in ``oap_mllib_amd.ops``:
``softmax_cross_entropy`` (loss of a softmax over a catalogue of items or classes, with its
gradients), ``dropout`` (mask from a counter-based generator) and ``route`` (top-k gate of a
mixture of experts).

``run`` computes the plain form (elementary torch operations) while ``own`` is false and calls
the framework's operators when it is true; both return the same outputs.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _ce(name, n, classes, dim, dtype, train, bias=False, ignored=0.0, weighted=False):
    return {"name": name, "op": "ce", "n": n, "classes": classes, "dim": dim, "dtype": dtype,
            "train": train, "bias": bias, "ignored": ignored, "weighted": weighted}


def _dropout(name, rows, cols, dtype, p, offset=0, residual=False, train=True):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p,
            "offset": offset, "residual": residual, "train": train}


def _route(name, tokens, experts, k, dtype, score, train, bias=False, groups=1, top_groups=1,
           renormalize=True, scale=1.0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k,
            "dtype": dtype, "score": score, "train": train, "bias": bias, "groups": groups,
            "top_groups": top_groups, "renormalize": renormalize, "scale": scale}


def listed():
    return [
        # log-likelihood of one user's held-out item under the whole catalogue of the ALS
        # benchmark (2M items, rank 100): a serving call, one pass over the item factors
        _ce("ce_one_row_2M_items", 1, 2_000_000, 100, "f32", train=False),
        # a classifier's small training step: the class count of the k = 1000 clustering
        # benchmark, its class prior as bias, padded rows left out, odd row count
        _ce("ce_small_classifier", 257, 1000, 100, "f32", train=True, bias=True, ignored=0.2),
        # one step of an item softmax over the ALS benchmark's catalogue
        _ce("ce_items_2M", 1024, 2_000_000, 100, "f32", train=True, bias=True),
        # perplexity of a ragged batch: odd classes and a feature count that no tile divides
        _ce("ce_eval_ragged", 300, 50_001, 1000, "bf16", train=False, ignored=0.1),
        # weighted rows (importance weights as upstream gradient) on the wide-row sizes of the
        # K-Means d = 784 benchmark
        _ce("ce_weighted_784", 3000, 20_000, 784, "bf16", train=True, weighted=True),
        # a large vocabulary at a training batch of 8192 tokens
        _ce("ce_vocabulary", 8192, 131_072, 2048, "bf16", train=True, ignored=0.05),
        # one small batch of rank-100 user vectors
        _dropout("dropout_small", 64, 100, "f32", 0.1),
        # odd sizes with the residual's addition, a shard that starts far inside a long table
        _dropout("dropout_residual_ragged", 4095, 1001, "bf16", 0.25, offset=(5 << 32) + 4,
                 residual=True),
        # 1M rows of a table of 100 features
        _dropout("dropout_table", 1_000_000, 100, "f32", 0.5),
        # the gate of one token in serving
        _route("route_one_token", 1, 64, 2, "f32", "softmax", train=False, renormalize=False),
        # a training batch with balance bias and group-limited choice
        _route("route_grouped_bias", 8192, 256, 8, "bf16", "sigmoid", train=True, bias=True,
               groups=8, top_groups=4, scale=2.5),
        # the largest batch, plain softmax gate
        _route("route_large_softmax", 262_144, 128, 8, "f32", "softmax", train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng: random.Random):
    op = rng.choice(["ce", "ce", "dropout", "route"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "ce":
        while True:
            n, classes, dim = _log(rng, 1, 8192), _log(rng, 2, 2_000_000), _log(rng, 1, 2048)
            if (n * classes <= 2 ** 30 and classes * dim <= 200_000_000
                    and n * classes * dim <= 2 ** 40):
                break
        train = rng.random() < 0.7
        c = _ce(None, n, classes, dim, dtype, train, bias=rng.random() < 0.5,
                ignored=rng.choice([0.0, 0.0, 0.1, 0.5]),
                weighted=train and rng.random() < 0.3)
    elif op == "dropout":
        while True:
            rows, cols = _log(rng, 1, 1_000_000), _log(rng, 1, 4096)
            if rows * cols <= 100_000_000:
                break
        c = _dropout(None, rows, cols, dtype, rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]),
                     offset=rng.choice([0, 0, 4 * rng.randrange(1 << 34), rng.randrange(1 << 36)]),
                     residual=rng.random() < 0.4, train=rng.random() < 0.8)
    else:
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, 2 if groups == 1 else 1, 512 // groups)
        experts = groups * per
        while True:
            tokens = _log(rng, 1, 262_144)
            if tokens * experts <= 262_144 * 128:
                break
        top_groups = rng.randint(1, groups)
        c = _route(None, tokens, experts, rng.randint(1, min(16, top_groups * per)), dtype, score,
                   train=rng.random() < 0.6, bias=rng.random() < 0.5, groups=groups,
                   top_groups=top_groups, renormalize=rng.random() < 0.6,
                   scale=rng.choice([1.0, 2.5]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev, dt = "cuda", _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).to(dt)

    s = {"case": case}
    if case["op"] == "ce":
        n, v, d = case["n"], case["classes"], case["dim"]
        # unit-scale features and weights whose logits have a standard deviation of about 2
        s["x"] = randn(n, d).requires_grad_(case["train"])
        s["weight"] = randn(v, d, scale=2.0 / math.sqrt(d)).requires_grad_(case["train"])
        t = torch.randint(0, v, (n,), generator=g, device=dev)
        drop = torch.rand(n, generator=g, device=dev) < case["ignored"]
        s["target"] = torch.where(drop, torch.full_like(t, -100), t)
        s["bias"] = None
        if case["bias"]:  # a log prior
            b = torch.rand(v, generator=g, device=dev).add_(0.05).log_()
            s["bias"] = b.requires_grad_(case["train"])
        if case["weighted"]:
            s["row_weight"] = torch.rand(n, generator=g, device=dev).add_(0.5)
    elif case["op"] == "dropout":
        r, c = case["rows"], case["cols"]
        s["x"] = randn(r, c).requires_grad_(case["train"])
        s["residual"] = randn(r, c).requires_grad_(case["train"]) if case["residual"] else None
        s["grad"] = randn(r, c) if case["train"] else None
        s["seed"] = (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63)
    else:
        t, e = case["tokens"], case["experts"]
        s["logits"] = randn(t, e).requires_grad_(case["train"])
        s["bias"] = None
        if case["bias"]:
            s["bias"] = torch.randn(e, generator=g, device=dev).mul_(0.05)
        s["grad"] = torch.randn(t, case["k"], generator=g, device=dev) if case["train"] else None
    return s


# -------------------------------------------------------------------------------- the run itself
def run(state):
    op = state["case"]["op"]
    if own:
        return {"ce": _own_ce, "dropout": _own_dropout, "route": _own_route}[op](state)
    with torch.no_grad():
        return {"ce": _plain_ce, "dropout": _plain_dropout, "route": _plain_route}[op](state)


def _own_ce(s):
    from oap_mllib_amd import ops

    c = s["case"]
    mean = c["train"] and not c["weighted"]  # an evaluation keeps every row's loss
    loss = ops.softmax_cross_entropy(s["x"], s["weight"], s["target"], bias=s["bias"],
                                     reduction="mean" if mean else "none")
    if not c["train"]:
        return [loss]
    leaves = [s["x"], s["weight"]] + ([s["bias"]] if c["bias"] else [])
    grads = torch.autograd.grad(loss, leaves, s["row_weight"] if c["weighted"] else None)
    return [loss.detach(), *grads]


def _own_dropout(s):
    from oap_mllib_amd import ops

    c = s["case"]
    y = ops.dropout(s["x"], c["p"], s["seed"], offset=c["offset"], residual=s["residual"])
    if not c["train"]:
        return [y]
    leaves = [s["x"]] + ([s["residual"]] if c["residual"] else [])
    return [y.detach(), *torch.autograd.grad(y, leaves, s["grad"])]


def _own_route(s):
    from oap_mllib_amd import ops

    c = s["case"]
    w, idx, counts = ops.route(s["logits"], c["k"], score=c["score"], bias=s["bias"],
                               groups=c["groups"], top_groups=c["top_groups"],
                               renormalize=c["renormalize"], scale=c["scale"])
    if not c["train"]:
        return [w, idx, counts]
    return [w.detach(), idx, counts, *torch.autograd.grad(w, [s["logits"]], s["grad"])]


# ----------------------------------------------------------------------------------- plain forms
def _plain_ce(s):
    c = s["case"]
    x, w, t = s["x"].float(), s["weight"].float(), s["target"]
    z = x @ w.t()
    if c["bias"]:
        z += s["bias"]
    kept = t != -100
    row = torch.arange(len(t), device=t.device)
    col = torch.where(kept, t, torch.zeros_like(t))
    zt = z[row, col]
    m = z.amax(dim=1, keepdim=True)
    z -= m
    e = z.exp_()
    total = e.sum(dim=1, keepdim=True)
    loss = torch.where(kept, total.log()[:, 0] + m[:, 0] - zt, torch.zeros_like(zt))
    if not c["train"]:
        return [loss]
    number = kept.sum().clamp(min=1)
    if not c["weighted"]:
        loss = loss.sum() / number
    up = s["row_weight"] if c["weighted"] else torch.ones_like(zt) / number
    up = torch.where(kept, up, torch.zeros_like(up))
    dz = e.mul_((up / total[:, 0])[:, None])
    dz[row, col] -= up
    gx = torch.zeros_like(x, dtype=torch.float64)
    for a in range(0, len(w), 1 << 15):  # a sum over 2M classes loses too much in one fp32 run
        gx += dz[:, a:a + (1 << 15)] @ w[a:a + (1 << 15)]
    out = [loss, gx.to(s["x"].dtype), (dz.t() @ x).to(s["weight"].dtype)]
    if c["bias"]:
        out.append(dz.sum(dim=0))
    return out


_LOW = 0xFFFFFFFF


def _plain_words(count, offset, seed, device):
    """The 32 random bits of elements offset .. offset + count - 1 (Philox4x32 with ten rounds,
    one block of four words for four consecutive elements), as int64."""
    first = offset // 4
    blocks = (offset + count + 3) // 4 - first
    n = torch.arange(first, first + blocks, device=device, dtype=torch.int64)
    a, b = n & _LOW, (n >> 32) & _LOW
    c, d = torch.zeros_like(a), torch.zeros_like(a)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (((q >> 32) & _LOW) ^ b ^ k0, q & _LOW, ((p >> 32) & _LOW) ^ d ^ k1, p & _LOW)
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([a, b, c, d], dim=1).reshape(-1)
    return words[offset - 4 * first:offset - 4 * first + count]


def _plain_dropout(s):
    c = s["case"]
    x = s["x"]
    words = _plain_words(x.numel(), c["offset"], s["seed"], x.device)
    keep = (words >= round(c["p"] * 2 ** 32)).view(x.shape)
    scale = 1.0 / (1.0 - c["p"])
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    if c["residual"]:
        y = y + s["residual"].float()
    out = [y.to(x.dtype)]
    if c["train"]:
        out.append(torch.where(keep, s["grad"].float() * scale, zero).to(x.dtype))
        if c["residual"]:
            out.append(s["grad"].clone())
    return out


def _plain_route(s):
    c = s["case"]
    z32 = s["logits"].float()
    z = z32.double()  # the choice is made in 64 bits: scores lie close to each other
    t, e = z.shape
    k = c["k"]
    if c["score"] == "softmax":
        sc = (z - z.amax(dim=1, keepdim=True)).exp()
        sc = sc / sc.sum(dim=1, keepdim=True)
    else:
        sc = 1.0 / (1.0 + (-z).exp())
    choice = sc if s["bias"] is None else sc + s["bias"].double()
    order = z if s["bias"] is None else choice
    per = e // c["groups"]
    if c["top_groups"] < c["groups"]:
        best = choice.view(t, c["groups"], per).sort(dim=2, descending=True).values
        best = best[:, :, :2].sum(dim=2)
        chosen = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, chosen, True)
        order = torch.where(mask.repeat_interleave(per, dim=1), order,
                            torch.full_like(order, -math.inf))
    idx = order.sort(dim=1, descending=True, stable=True).indices[:, :k]
    counts = torch.zeros(e, device=z.device, dtype=torch.int64)
    counts.scatter_add_(0, idx.reshape(-1), torch.ones_like(idx.reshape(-1)))
    if c["score"] == "softmax":
        s32 = (z32 - z32.amax(dim=1, keepdim=True)).exp()
        s32 = s32 / s32.sum(dim=1, keepdim=True)
    else:
        s32 = 1.0 / (1.0 + (-z32).exp())
    top = s32.gather(1, idx)
    w = top / top.sum(dim=1, keepdim=True) if c["renormalize"] else top
    out = [w * c["scale"], idx.int(), counts.int()]
    if c["train"]:
        g = s["grad"] * c["scale"]
        if c["renormalize"]:
            gs = (g - (g * w).sum(dim=1, keepdim=True)) / top.sum(dim=1, keepdim=True)
        else:
            gs = g
        dense = torch.zeros_like(s32).scatter_(1, idx, gs)
        if c["score"] == "softmax":
            dz = s32 * (dense - (dense * s32).sum(dim=1, keepdim=True))
        else:
            dz = dense * s32 * (1.0 - s32)
        out.append(dz.to(s["logits"].dtype))
    return out


# ---------------------------------------------------------------------------------- what is needed
def work(case):
    b = _SIZES[case["dtype"]]
    if case["op"] == "ce":
        n, v, d = case["n"], case["classes"], case["dim"]
        nbytes = (n + v) * d * b + 8 * n + (4 * v if case["bias"] else 0)
        nbytes += 4 if case["train"] and not case["weighted"] else 4 * n
        flops = 2 * n * v * d
        if case["train"]:
            nbytes += (n + v) * d * b + (4 * v if case["bias"] else 0)
            nbytes += 4 * n if case["weighted"] else 0
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        tensors = 2 + case["residual"]
        if case["train"]:
            tensors += 2 + case["residual"]  # (the residual's gradient is the upstream one)
        return {"bytes": tensors * n * b, "flops": (2 if case["train"] else 1) * n}
    t, e, k = case["tokens"], case["experts"], case["k"]
    nbytes = t * e * b + 8 * t * k + 4 * e + (4 * e if case["bias"] else 0)
    if case["train"]:
        nbytes += 4 * t * k + t * e * b
    return {"bytes": nbytes, "flops": 4 * t * e * (2 if case["train"] else 1)}


# ------------------------------------------------------------------------------- 64-bit oracles
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"ce": _exact_ce, "dropout": _exact_dropout, "route": _exact_route}[case["op"]](s)


def _exact_ce(s):
    c = s["case"]
    x, w, t = s["x"].double(), s["weight"].double(), s["target"]
    b = s["bias"].double() if c["bias"] else torch.zeros(len(w), device=x.device).double()
    n_kept = max(1, int((t >= 0).sum()))
    up = s["row_weight"].double() if c["weighted"] else torch.full_like(x[:, 0], 1.0 / n_kept)
    losses = torch.zeros(len(x), device=x.device, dtype=torch.float64)
    gx, gw, gb = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, (1 << 28) // len(w))
    for r in range(0, len(x), step):  # blocks of rows; ignored rows add nothing
        rows = (r + torch.nonzero(t[r:r + step] >= 0)[:, 0])
        if not len(rows):
            continue
        logp = torch.log_softmax(torch.addmm(b, x[rows], w.t()), dim=1)
        pick = t[rows][:, None]
        losses[rows] = -logp.gather(1, pick)[:, 0]
        if c["train"]:
            p = logp.exp_()
            p.scatter_add_(1, pick, -torch.ones_like(pick, dtype=torch.float64))
            p.mul_(up[rows][:, None])
            gx[rows] = p @ w
            gw.addmm_(p.t(), x[rows])
            gb += p.sum(dim=0)
    if not c["train"]:
        return [losses]
    out = [losses if c["weighted"] else losses.sum() / n_kept]
    return out + [gx, gw] + ([gb] if c["bias"] else [])


def _exact_keep(count, offset, seed, p):
    low = np.uint64(_LOW)
    half = np.uint64(32)
    blk = np.arange(offset // 4, (offset + count - 1) // 4 + 1, dtype=np.uint64)
    ctr = [blk & low, blk >> half, np.zeros_like(blk), np.zeros_like(blk)]
    for r in range(10):
        key = [np.uint64((seed + r * 0x9E3779B9) & _LOW),
               np.uint64(((seed >> 32) + r * 0xBB67AE85) & _LOW)]
        m0 = ctr[0] * np.uint64(0xD2511F53)
        m1 = ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(m1 >> half) ^ ctr[1] ^ key[0], m1 & low, (m0 >> half) ^ ctr[3] ^ key[1], m0 & low]
    bits = np.empty((len(blk), 4), dtype=np.uint32)
    for j in range(4):
        bits[:, j] = ctr[j]
    return bits.reshape(-1)[offset % 4:offset % 4 + count].astype(np.float64) / 2.0 ** 32 >= \
        round(p * 2 ** 32) / 2.0 ** 32


def _exact_dropout(s):
    c = s["case"]
    x = s["x"].double()
    keep = torch.from_numpy(_exact_keep(x.numel(), c["offset"], s["seed"], c["p"]))
    factor = keep.to(x.device).view(x.shape).double() / (1.0 - c["p"])
    out = [x * factor + (s["residual"].double() if c["residual"] else 0.0)]
    if c["train"]:
        out.append(s["grad"].double() * factor)
        if c["residual"]:
            out.append(s["grad"].double())
    return out


def _exact_route(s):
    c = s["case"]
    z = s["logits"].double()
    t, e = z.shape
    score = torch.softmax(z, dim=1) if c["score"] == "softmax" else torch.sigmoid(z)
    value = score + s["bias"].double() if c["bias"] else score
    rank = value.clone() if c["bias"] else z.clone()
    number = torch.arange(e, device=z.device)
    per = e // c["groups"]
    if c["top_groups"] < c["groups"]:
        parts = value.view(t, c["groups"], per)
        total = parts.topk(min(2, per), dim=2).values.sum(dim=2)
        open_groups = torch.zeros_like(total, dtype=torch.bool)
        for _ in range(c["top_groups"]):  # the best group left, the lowest number among equals
            hit = total == total.amax(dim=1, keepdim=True)
            first = torch.where(hit, number[:c["groups"]], e).amin(dim=1, keepdim=True)
            open_groups.scatter_(1, first, True)
            total.scatter_(1, first, -math.inf)
        rank.masked_fill_(~open_groups[:, number // per], -math.inf)
    picks = []
    for _ in range(c["k"]):
        hit = rank == rank.amax(dim=1, keepdim=True)
        first = torch.where(hit, number, e).amin(dim=1, keepdim=True)
        picks.append(first)
        rank.scatter_(1, first, -math.inf)
    idx = torch.cat(picks, dim=1)
    chosen = score.gather(1, idx)
    norm = chosen.sum(dim=1, keepdim=True) if c["renormalize"] else torch.ones_like(chosen[:, :1])
    w = chosen / norm * c["scale"]
    counts = torch.zeros(e, device=z.device, dtype=torch.int64)
    counts.index_add_(0, idx.reshape(-1), torch.ones_like(idx.reshape(-1)))
    out = [w, idx.int(), counts.int()]
    if c["train"]:
        g = s["grad"].double()
        into = c["scale"] * g / norm  # d / d score of the chosen
        if c["renormalize"]:
            into = into - (g * w).sum(dim=1, keepdim=True) / norm
        if c["score"] == "softmax":
            dz = -score * (into * chosen).sum(dim=1, keepdim=True)
            dz.scatter_add_(1, idx, into * chosen)
        else:
            dz = torch.zeros_like(z).scatter_(1, idx, into * chosen * (1.0 - chosen))
        out.append(dz)
    return out
