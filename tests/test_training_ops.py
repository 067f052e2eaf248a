"""oap_mllib_amd.ops training ops (softmax_cross_entropy, dropout, route) against plain 64-bit
implementations: every case runs on the host engine and, marked gpu, on the kernels.

Tolerances follow the arithmetic: u is half a step of the element type (relative), fp32 sums of n
terms are off by at most n 2^-23 of the sum of the terms' magnitudes (the matrix units may
truncate), and a result is rounded once to its type."""
import math

import numpy as np
import pytest
import torch

from oap_mllib_amd import _loader, ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -23
INF = math.inf


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rand(shape, seed, dtype=torch.float32, device="cpu", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def cpu64(t):
    return t.detach().cpu().double()


def check(got, ref, tol, what):
    got = cpu64(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~same & ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4],
                           torch.as_tensor(tol).expand_as(ref)[bad][:4])


# --------------------------------------------------------------------- softmax cross entropy
def ce_oracle(x, w, t, b, up, ignore=-100):
    """64-bit losses, gradients (for the upstream row gradients `up`) and the bounds of their
    errors per unit of relative error of dz."""
    x, w, t = cpu64(x), cpu64(w), t.cpu().long()
    n, v = len(x), len(w)
    out = torch.zeros(v, dtype=torch.bool) if b is None else cpu64(b) == -INF
    x = torch.where((t == ignore)[:, None], torch.zeros_like(x), x)
    w = torch.where(out[:, None], torch.zeros_like(w), w)
    bias = torch.zeros(v).double() if b is None else cpu64(b)
    z = x @ w.t() + bias
    lse = torch.logsumexp(z, dim=1)
    p = torch.where(out, torch.zeros_like(z), (z - lse[:, None]).exp())
    valid = (t >= 0) & (t < v) & (t != ignore)
    tt = torch.where(valid, t, torch.zeros_like(t))
    zt = z.gather(1, tt[:, None])[:, 0]
    loss = torch.where(zt == -INF, torch.full_like(zt, INF), lse - zt)
    loss = torch.where(t == ignore, torch.zeros_like(loss),
                       torch.where(valid, loss, torch.full_like(loss, math.nan)))
    hot = torch.zeros_like(p)
    hot[torch.arange(n), tt] = (valid & ~out[tt]).double()
    u = torch.where(valid, cpu64(up).expand(n), torch.zeros(n).double())
    dz = u[:, None] * (p - hot)
    mag = u.abs()[:, None] * (p + hot)
    # largest error of a logit, and of the sums
    absz = (x.abs() @ w.abs().t()).max().item() if n and v else 0.0
    fin = bias[bias > -INF]
    bmax = fin.abs().max().item() if len(fin) else 0.0
    zerr = (x.shape[1] + 8) * E32 * absz + 2 * E32 * (absz + bmax)
    return {"loss": loss, "dx": dz @ w, "dw": dz.t() @ x, "db": dz.sum(0), "zerr": zerr,
            "mdx": mag @ w.abs(), "mdw": mag.t() @ x.abs(), "mdb": mag.sum(0), "lse": lse}


def ce_check(x, w, t, b, reduction="mean", up=None, ignore=-100, want=(True, True, True)):
    leaves = [None if o is None else o.detach().requires_grad_(q)  # (the strides of a view)
              for o, q in zip((x, w, b), want)]
    n = len(x)
    count = max(1, int((t != ignore).sum()))
    loss = ops.softmax_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2],
                                     ignore_index=ignore, reduction=reduction)
    if reduction == "none":
        rows = up if up is not None else torch.ones(n, device=x.device)
    else:
        rows = torch.full((n,), 1.0 / count if reduction == "mean" else 1.0)
    ref = ce_oracle(x, w, t, b, rows, ignore)
    u = half_step(x.dtype)
    # (inf - inf of an excluded or infinite row compares equal in check)
    ltol = 2 * ref["zerr"] + 4 * E32 * (ref["lse"].nan_to_num(0, 0, 0).abs() + 1)
    if reduction == "none":
        check(loss, ref["loss"], ltol, "loss")
    else:
        kept = ref["loss"][t.cpu() != ignore]
        total = kept.sum() / (count if reduction == "mean" else 1)
        scale = kept.nan_to_num(0, 0, 0).abs().sum() / (count if reduction == "mean" else 1)
        tol = ltol.max() * (1 if reduction == "mean" else n) + 2 * E32 * scale
        check(loss, total, tol, "total")
    assert loss.dtype == torch.float32
    use = [(k, v) for k, v in zip(("dx", "dw", "db"), leaves) if v is not None and v.requires_grad]
    if not use:
        return
    grads = torch.autograd.grad(loss, [v for _, v in use],
                                rows.to(loss.device) if reduction == "none" else None)
    top = rows.abs().max().item() if n else 0.0
    for (name, leaf), g in zip(use, grads):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        terms = {"dx": len(w), "dw": n, "db": n}[name]
        # dz: logits, lse and exp in fp32; rounded to the operand type unless summed for db
        rel = 2 * ref["zerr"] + 16 * E32 + (0 if name == "db" else u) + (terms + 8) * E32
        uo = half_step(leaf.dtype)
        # fp16: dz below 2^-28 of the largest upstream gradient and results below the normal
        # range lose bits
        small = 2.0 ** -38 * top * (terms * float(cpu64(w if name == "dx" else x)
                                                  .nan_to_num(0, 0, 0).abs().amax())
                                    if terms and x.numel() and w.numel() else 1.0)
        tiny = (small + 2.0 ** -24 if leaf.dtype == torch.float16 else 1e-37)
        check(g, ref[name], ref["m" + name] * (rel + uo) + uo * ref[name].abs() + tiny, name)


CE_SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 8), (5, 7, 13), (2, 300, 64), (64, 255, 64),
            (65, 257, 100), (130, 1000, 128), (257, 513, 200), (70, 2050, 65), (33, 40, 513)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", CE_SIZES)
def test_ce_sizes(device, dtype, n, v, d):
    x = rand((n, d), 1, dtype, device)
    w = rand((v, d), 2, dtype, device, 2 / math.sqrt(d))
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).to(device)
    t[::4] = -100
    b = rand((v,), 4, torch.float32, device)
    ce_check(x, w, t, b)
    ce_check(x, w, t, None, "sum")
    up = rand((n,), 5, torch.float32, device)
    ce_check(x, w, t, b, "none", up)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_ce_left_out_rows_and_classes(device, dtype):
    """Ignored rows and classes with bias -inf may hold anything; an excluded or invalid target
    gives inf or NaN and touches no other row."""
    n, v, d = 70, 300, 64
    x, w = rand((n, d), 1, dtype, device), rand((v, d), 2, dtype, device, 0.3)
    t = torch.arange(n, device=device) % v
    t[5:20] = -100
    x[6], x[7, 3], x[8, 0] = math.nan, INF, -INF
    b = rand((v,), 3, torch.float32, device)
    b[100:200:3] = -INF
    w[100], w[103, 1], w[106, 2] = math.nan, INF, -INF
    ce_check(x, w, t, b)
    t[30], t[31], t[32] = 100, v, -7  # excluded target; two that are no class
    ones = torch.ones(n, device=device)
    ce_check(x, w, t, b, "none", ones)
    loss = ops.softmax_cross_entropy(x, w, t, b, reduction="none").cpu()
    assert loss[30] == INF and loss[31].isnan() and loss[32].isnan()
    assert loss.isfinite().sum() == n - 3
    assert ops.softmax_cross_entropy(x, w, t, b).isnan()


@pytest.mark.parametrize("device", DEVICES)
def test_ce_nothing_left(device):
    n, v, d = 10, 20, 16
    for dtype in DTYPES:
        x = rand((n, d), 1, dtype, device).requires_grad_()
        w = rand((v, d), 2, dtype, device).requires_grad_()
        t = torch.full((n,), -100, device=device)
        loss = ops.softmax_cross_entropy(x, w, t)
        gx, gw = torch.autograd.grad(loss, [x, w])
        assert loss.item() == 0 and not gx.any() and not gw.any()
        # every class left out
        b = torch.full((v,), -INF, device=device)
        t = torch.arange(n, device=device)
        loss = ops.softmax_cross_entropy(x, w, t, b, reduction="none")
        gx, gw = torch.autograd.grad(loss, [x, w], torch.ones_like(loss))
        assert (loss == INF).all() and not gx.any() and not gw.any()
        # the type's lowest value is a bias like any other: the softmax is flat
        b = torch.full((v,), torch.finfo(torch.float32).min, device=device)
        loss = ops.softmax_cross_entropy(x, w, t, b, reduction="none")
        check(loss, torch.full((n,), math.log(v)).double(), 64 * E32 * math.log(v) + 1e-5,
              "lowest")
        # no row
        loss = ops.softmax_cross_entropy(x[:0], w, t[:0])
        gw, = torch.autograd.grad(loss, [w])
        assert loss.item() == 0 and not gw.any() and gw.shape == w.shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_ce_strides_and_types(device, dtype):
    n, v, d = 40, 130, 64
    wide = rand((n, d + 9), 1, dtype, device)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).to(device)
    w = rand((v, d), 2, dtype, device, 0.3)
    for x in (wide[:, 1:d + 1], wide[:, 8:d + 8], rand((d, n), 4, dtype, device).t(),
              rand((1, d), 5, dtype, device).expand(n, d), rand((2 * n, d), 6, dtype, device)[::2]):
        ce_check(x, w, t, None)
    ce_check(wide[:, :d], rand((d, v), 7, dtype, device).t(), t.int(),
             rand((v,), 8, torch.bfloat16, device))
    tt = torch.stack([t, t], 1)[:, 0]  # a strided target
    ce_check(wide[:, :d], w, tt, None, "sum", want=(True, False, False))
    ce_check(wide[:, :d], w, tt, None, "sum", want=(False, True, False))
    ce_check(wide[:, :d], w, tt, rand((v,), 9, torch.float32, device), want=(False, False, True))
    t0 = torch.where(t % 3 == 0, torch.zeros_like(t), t)
    ce_check(wide[:, :d], w, t0, None, ignore=0)


@pytest.mark.parametrize("device", DEVICES)
def test_ce_gradient_against_differences(device):
    n, v, d = 6, 50, 20
    x, w, b = rand((n, d), 1), rand((v, d), 2), rand((v,), 3)
    t = torch.tensor([3, 3, -100, 49, 0, 7])
    up = torch.rand(n, generator=torch.Generator().manual_seed(4)) + 0.5
    leaves = [q.to(device).requires_grad_() for q in (x, w, b)]
    loss = ops.softmax_cross_entropy(*leaves[:2], t.to(device), leaves[2], reduction="none")
    grads = torch.autograd.grad(loss, leaves, up.to(device))

    def f(h, dirs):
        xs = [q.double() + h * r for q, r in zip((x, w, b), dirs)]
        z = xs[0] @ xs[1].t() + xs[2]
        rows = torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0]
        return (rows * up.double() * (t != -100)).sum()

    for seed in range(5):
        dirs = [rand(q.shape, 10 + seed).double() for q in (x, w, b)]
        h = 1e-4
        diff = (f(h, dirs) - f(-h, dirs)) / (2 * h)
        got = sum((cpu64(g) * r).sum() for g, r in zip(grads, dirs))
        size = sum((cpu64(g).abs() * r.abs()).sum() for g, r in zip(grads, dirs))
        # h^2 / 6 of a third derivative of at most a few |z'|^3 (|z'| below 60 here): below
        # 1e-8 / 6 * 2 * 60^3 * n; the gradients' own error: (d + v + 30) 2^-23
        assert abs(diff - got) <= 1e-8 / 6 * 2 * 60 ** 3 * n + (d + v + 30) * E32 * size


def test_ce_refusals():
    x, w, t = rand((4, 8), 1), rand((9, 8), 2), torch.zeros(4, dtype=torch.int64)
    f = ops.softmax_cross_entropy
    for bad in [lambda: f(x[0], w, t), lambda: f(x, w[0], t), lambda: f(x, w[:, :5], t),
                lambda: f(x, w.half(), t), lambda: f(x.double(), w.double(), t),
                lambda: f(x, w, t[:3]), lambda: f(x, w, t.float()), lambda: f(x, w, t, x[:, 0]),
                lambda: f(x, w, t, torch.zeros(9, dtype=torch.int64)),
                lambda: f(x, w, t, reduction="avg"), lambda: f(x[:, :0], w[:, :0], t),
                lambda: f(x, w[:0], t), lambda: f([1], w, t), lambda: f(x, w, [0] * 4),
                lambda: f(x, w.to("meta"), t), lambda: f(x.to("meta"), w, t)]:
        with pytest.raises(ValueError):
            bad()
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(f(leaf, w, t), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [leaf])


@pytest.mark.gpu
def test_ce_pieces_gpu():
    """Classes in more than one piece, and a row count whose tiles span several workgroups."""
    for dtype, n, v, d, bias in [(torch.bfloat16, 8190, 40_001, 64, False),
                                 (torch.float32, 2000, 50_003, 5, True)]:
        g = torch.Generator(device="cuda").manual_seed(1)
        x = torch.randn(n, d, generator=g, device="cuda").to(dtype).requires_grad_()
        w = (torch.randn(v, d, generator=g, device="cuda") * 0.3).to(dtype).requires_grad_()
        b = torch.randn(v, generator=g, device="cuda").requires_grad_() if bias else None
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        leaves = [x, w] + ([b] if bias else [])
        loss = ops.softmax_cross_entropy(x, w, t, b)
        grads = torch.autograd.grad(loss, leaves)
        xd, wd = x.detach().double(), w.detach().double()
        z = xd @ wd.t() + (b.detach().double() if bias else 0)
        p = torch.softmax(z, 1)
        ref = -p.gather(1, t[:, None]).log().mean()
        p.scatter_add_(1, t[:, None], -torch.ones_like(p[:, :1]))
        p /= n
        u = half_step(dtype)
        assert abs(loss.item() - ref.item()) <= 1e-5 * abs(ref.item())
        for got, want, mag in [(grads[0], p @ wd, p.abs() @ wd.abs()),
                               (grads[1], p.t() @ xd, p.abs().t() @ xd.abs())] + \
                ([(grads[2], p.sum(0), p.abs().sum(0))] if bias else []):
            # sums over blocks: at most 2^16 terms in one fp32 run
            tol = mag * (u + 2e-5 + 256 * E32) + u * want.abs() + 1e-30
            err = (got.double() - want).abs()
            assert (err <= tol).all(), (dtype, (err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 1e-18, 1e18])
def test_ce_large_fp32_gpu(scale):
    """fp32 problems large enough for the split operands: sizes off every tile, rows and classes
    that are left out, magnitudes far from one (x and weight scaled against each other).  What the
    split leaves out, 2^-40 of an operand's largest entry and 2^-39 of the largest coefficient, is
    below 2^-23 of the sums of magnitudes here: every row of x and weight holds an entry within
    2^-3 of the largest, and the smallest dz is above 2^-15 of the largest."""
    n, v, d = 333, 15_013, 301
    x, w = rand((n, d), 1, device="cuda"), rand((v, d), 2, device="cuda", scale=0.5 / math.sqrt(d))
    x, w = x * scale, w / scale
    b = rand((v,), 3, device="cuda", scale=0.3)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(4)).cuda()
    ce_check(x, w, t, None)
    t[7:200:5] = -100
    x[7], x[12, 3] = math.nan, INF
    b[100:9000:7] = -INF
    w[100], w[107, 5] = math.nan, -INF
    ce_check(x, w, t, b)
    ce_check(x, w, t, b, "none", torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda()
             + 0.5)
    z = torch.zeros_like(x)
    loss = ops.softmax_cross_entropy(z, torch.zeros_like(w), t)
    check(loss, torch.tensor(math.log(v)).double(), 8 * E32 * math.log(v), "zeros")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [False, True])
def test_ce_many_tiles_gpu(dtype, bias):
    """Enough rows and classes for the wider tiles of 16-bit logits."""
    n, v, d = 1100, 30001, 40
    x, w = rand((n, d), 1, dtype, "cuda", 0.5), rand((v, d), 2, dtype, "cuda", 0.5)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    t[::7] = -100
    b = None
    if bias:
        b = rand((v,), 4)
        b[5::11] = -INF
        b[t[t >= 0]] = 0.25
        b = b.cuda()
    ce_check(x, w, t.cuda(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(50, 30_001, 72), (33, 26_000, 1100), (700, 20_003, 1100),
                                   (257, 15_000, 1032), (300, 9000, 100)])
def test_ce_each_tile_gpu(dtype, n, v, d):
    """Few rows of many classes, the largest tiles (long rows), and middling problems; rows with
    a stride, left-out rows and classes."""
    x = rand((n, d + 8), 1, dtype, "cuda", 0.3)[:, :d]
    w = rand((v, d), 2, dtype, "cuda", 0.3)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    b = rand((v,), 4)
    b[3::17] = -INF
    b[t] = 0.5
    t[::9] = -100
    ce_check(x, w, t.cuda(), b.cuda(), reduction="sum")
    ce_check(x, w, t.cuda(), None, want=(True, False, False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(5, 5000, 100), (6, 3000, 1032), (7, 33, 40), (8, 999, 1024),
                                   (8, 30_000, 64), (5, 7, 8), (2, 2000, 200), (8, 1, 4),
                                   (9, 40_000, 8), (20, 30_001, 100), (32, 26_000, 300)])
def test_ce_small_batches_gpu(dtype, n, v, d):
    """Up to eight rows at once from registers, up to 32 in narrow tiles."""
    x, w = rand((n, d), 1, dtype, "cuda", 0.5), rand((v, d), 2, dtype, "cuda", 0.5)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    b = rand((v,), 4)
    b[1::7] = -INF
    b[t] = 0.5
    for bias in (None, b.cuda()):
        ce_check(x, w, t.cuda(), bias, reduction="none")
    t[n // 2] = -100
    x[n // 2] = math.nan
    w[b.cuda() == -INF] = math.nan
    ce_check(x, w, t.cuda(), b.cuda(), want=(True, True, True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(40, 700, 24), (300, 9000, 100), (600, 12_000, 1100)])
def test_ce_each_gradient_alone_gpu(dtype, n, v, d):
    x, w = rand((n, d), 1, dtype, "cuda", 0.3), rand((v, d), 2, dtype, "cuda", 0.3)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    b = rand((v,), 4, device="cuda")
    for want in ((True, False, False), (False, True, False), (False, False, True),
                 (False, True, True)):
        ce_check(x, w, t, b, want=want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 8])
@pytest.mark.parametrize("d,shift", [(101, 0), (100, 0), (100, 4), (102, 2), (96, 3), (520, 1)])
def test_ce_few_rows_of_any_alignment_gpu(dtype, n, d, shift):
    v = 2500
    x = rand((n, d + shift), 1, dtype, "cuda", 0.5)[:, shift:]
    w = rand((v, d + shift), 2, dtype, "cuda", 0.5)[:, shift:]
    b = rand((v,), 4, device="cuda")
    b[1::7] = -INF
    t = torch.arange(n, device="cuda") * 7 + 3
    ce_check(x, w, t, None, want=(False, False, False))
    w[b == -INF] = math.nan
    ce_check(x, w, t, b, "none")


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["rows", "classes", "targets", "weights"])
def test_ce_large_numbers_left_out_gpu(what):
    """Finite numbers of any size in rows and classes that are left out change nothing else (fp32
    problems whose operands are scaled by their largest number)."""
    n, v, d = 300, 50_000, 128
    x, w = rand((n, d), 1, torch.float32, "cuda"), rand((v, d), 2, torch.float32, "cuda", 0.2)
    t = torch.randint(0, v // 2, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    b = None
    if what == "classes":
        b = torch.zeros(v, device="cuda")
        b[v // 2:] = -INF
        w[v // 2:] = 1e30
        ce_check(x, w, t, b)
        return
    up = torch.ones(n, device="cuda")
    if what == "weights":
        up[::3] = 0  # (rows with a loss of their own)
    else:
        t[::3] = -100 if what == "rows" else v + 5
    clean = [q.clone().requires_grad_() for q in (x, w)]
    x[::3] = 1e30
    dirty = [q.requires_grad_() for q in (x, w)]
    loss = []
    for leaves in (clean, dirty):
        rows = ops.softmax_cross_entropy(*leaves, t, reduction="none")
        loss.append((rows.detach()[up > 0], *torch.autograd.grad(rows, leaves, up)))
    if what == "rows":
        ce_check(clean[0].detach(), clean[1].detach(), t, None)
    for a, c in zip(*loss):
        assert torch.equal(a.nan_to_num(7.0), c.nan_to_num(7.0))


@pytest.mark.gpu
def test_ce_rows_of_any_size_gpu():
    """A row's loss and its gradient of x do not depend on what the other rows hold."""
    n, v, d = 300, 50_000, 128
    x, w = rand((n, d), 1, torch.float32, "cuda"), rand((v, d), 2, torch.float32, "cuda", 0.2)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    x[1::3] *= 1e-12
    got = []
    for big in (1.0, 1e12):
        leaf = torch.cat([x[:150], x[150:] * big]).requires_grad_()
        rows = ops.softmax_cross_entropy(leaf, w, t, reduction="none")
        got.append((rows.detach()[:150], torch.autograd.grad(rows.sum(), leaf)[0][:150]))
    for a, c in zip(*got):
        assert torch.equal(a, c)
    ce_check(x, w, t, None, reduction="none")


@pytest.mark.parametrize("device", DEVICES)
def test_ce_rows_without_upstream_gradient(device):
    x, w = rand((6, 9), 1, device=device), rand((11, 9), 2, device=device).requires_grad_()
    t = torch.tensor([0, 3, 10, 5, 5, 1], device=device)
    up = torch.tensor([1.0, 0.0, -2.0, 0.0, 0.5, 1.0], device=device)
    got = []
    for bad in (0.0, math.nan):
        leaf = x.clone()
        leaf[1], leaf[3] = bad, -bad
        leaf.requires_grad_()
        rows = ops.softmax_cross_entropy(leaf, w, t, reduction="none")
        got.append(torch.autograd.grad(rows, [leaf, w], up))
    for a, c in zip(*got):
        assert torch.equal(a, c) and not a.isnan().any()


@pytest.mark.gpu
def test_ce_rows_in_turns_gpu():
    """More rows than one turn of the forward pass keeps statistics for: every row's loss is that
    of a call on its own part of the rows, but for the order in which 15625 tiles' sums are joined
    (up to 31 additions and powers in a row of threads, 10 levels above them)."""
    n, v, d = 9000, 2_000_000, 4
    x, w = rand((n, d), 1, torch.bfloat16, "cuda"), rand((v, d), 2, torch.bfloat16, "cuda")
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    t[::7] = -100
    whole = ops.softmax_cross_entropy(x, w, t, reduction="none")
    parts = [ops.softmax_cross_entropy(x[a:a + 3000], w, t[a:a + 3000], reduction="none")
             for a in range(0, n, 3000)]
    parts = torch.cat(parts)
    assert ((whole - parts).abs() <= 2 * 41 * 3 * E32 + 4 * E32 * parts.abs()).all()
    mean = ops.softmax_cross_entropy(x, w, t)
    ref = whole.double().sum() / (t != -100).sum()
    assert abs(mean.item() - ref.item()) <= E32 * abs(ref.item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(1, 5000, 100), (3, 1000, 1024), (4, 999, 40), (4, 33, 2048),
                                   (2, 70, 4096), (1, 1, 8), (5, 3000, 128)])
def test_ce_few_rows_gpu(dtype, n, v, d):
    """One row and a few: losses alone and with gradients, odd counts, every lane layout."""
    x, w = rand((n, d), 1, dtype, "cuda"), rand((v, d), 2, dtype, "cuda", 2 / math.sqrt(d))
    t = torch.arange(n, device="cuda") * 13 % v
    b = rand((v,), 3, device="cuda")
    b[v // 2 + 1::3] = -INF
    for bias in (None, b):
        ce_check(x, w, t, bias, "none", want=(False, False, False))
        ce_check(x, w, t, bias)


# ----------------------------------------------------------------------------------- dropout
def philox_words(count, offset, seed):
    """Words of elements offset .. offset + count - 1, in plain integers."""
    out = []
    for i in range(offset, offset + count):
        c = [(i >> 2) & 0xFFFFFFFF, i >> 34, 0, 0]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out.append(c[i & 3])
    return out


def test_philox_known_answer():
    # the generator's published answers for a counter and key of zeros
    assert philox_words(4, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = torch.ones(4)
    for i, w in enumerate(philox_words(4, 0, 0)):
        p = w / 2 ** 32  # kept at the threshold itself, dropped just above
        assert ops.dropout(ones, p, 0)[i] != 0
        assert ops.dropout(ones, (w + 1) / 2 ** 32, 0)[i] == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,offset", [(1, 0), (3, 5), (8, 4), (9, 8), (1001, 3), (1001, 1 << 35),
                                      (4111, (1 << 40) + 2), (70, (1 << 64) - 70)])
def test_dropout(device, dtype, n, offset):
    seed = 0xFEDCBA9876543210 + n
    x, res, g = (rand((n,), i, dtype, device) for i in range(3))
    words = torch.tensor(philox_words(n, offset, seed))
    u = half_step(dtype)
    for p in (0.0, 0.3, 0.875, 1.0):
        keep = (words >= round(p * 2 ** 32)).double()
        f = keep / (1 - p) if p < 1 else keep * 0
        for r in (None, res):
            xl, rl = x.clone().requires_grad_(), res.clone().requires_grad_()
            y = ops.dropout(xl, p, seed, offset=offset, residual=rl if r is not None else None)
            ref = cpu64(x) * f + (cpu64(res) if r is not None else 0)
            tol = 2 * E32 * (cpu64(x) * f).abs() + (u + E32) * ref.abs() + 2.0 ** -25
            check(y, ref, tol if dtype == torch.float16 else tol - 2.0 ** -25 + 1e-38, "y")
            assert ((y.cpu() == 0) | (keep > 0)).all() or r is not None
            grads = torch.autograd.grad(y, [xl] + ([rl] if r is not None else []), g)
            check(grads[0], cpu64(g) * f, (2 * E32 + u) * (cpu64(g) * f).abs() + 2.0 ** -25, "dx")
            if r is not None:
                assert torch.equal(grads[1], g)


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_places_and_shapes(device):
    x = rand((6, 50, 7), 1, torch.float32, device)
    x[0, :10] = math.nan
    x[1, :10] = INF
    y = ops.dropout(x, 0.5, 7)
    keep = (torch.tensor(philox_words(x.numel(), 0, 7)) >= 1 << 31).view(x.shape)
    assert not y.cpu()[~keep].any() and y.cpu()[0, :10][keep[0, :10]].isnan().all()
    assert not ops.dropout(x, 1.0, 7).any()
    # a shard draws what the whole table draws; so do views, an unaligned one among them
    assert torch.equal(ops.dropout(x[2:], 0.5, 7, offset=2 * 350), y[2:])
    flat = rand((2001,), 2, torch.bfloat16, device)
    assert torch.equal(ops.dropout(flat[1:], 0.5, 9), ops.dropout(flat[1:].clone(), 0.5, 9))
    z = rand((30, 40), 3, torch.float32, device)
    assert torch.equal(ops.dropout(z.t(), 0.5, 9), ops.dropout(z.t().contiguous(), 0.5, 9))
    zl = z.clone().requires_grad_()
    g, = torch.autograd.grad(ops.dropout(zl, 0.25, 9).sum(), [zl])  # (an expanded gradient)
    assert torch.equal(g, ops.dropout(torch.ones_like(z), 0.25, 9))
    seed = torch.tensor([9], device=device)
    assert torch.equal(ops.dropout(z, 0.25, seed), ops.dropout(z, 0.25, 9))
    assert torch.equal(ops.dropout(z, 0.25, -1), ops.dropout(z, 0.25, (1 << 64) - 1))
    y = ops.dropout(zl, 0.25, seed)
    seed += 1
    with pytest.raises(RuntimeError):  # (the mask of the gradient would be another)
        torch.autograd.grad(y.sum(), [zl])
    assert ops.dropout(z[:0], 0.25, 9).shape == (0, 40)
    many = ops.dropout(torch.ones(1 << 20, device=device), 0.1, 5)
    # binomial: six standard deviations of 2^20 draws
    assert abs((many == 0).double().mean().item() - 0.1) < 6 * math.sqrt(0.09 / 2 ** 20)


def test_dropout_refusals():
    x = torch.ones(8)
    for bad in [lambda: ops.dropout(x, -0.1, 1), lambda: ops.dropout(x, 1.1, 1),
                lambda: ops.dropout(x, math.nan, 1), lambda: ops.dropout(x.double(), 0.1, 1),
                lambda: ops.dropout(x.long(), 0.1, 1), lambda: ops.dropout(x, 0.1, 1 << 64),
                lambda: ops.dropout(x, 0.1, 1, offset=-4),
                lambda: ops.dropout(x, 0.1, 1, offset=(1 << 64) - 7),
                lambda: ops.dropout(x, 0.1, 1, residual=x[:4]),
                lambda: ops.dropout(x, 0.1, 1, residual=x.half()),
                lambda: ops.dropout(x, 0.1, torch.tensor([1, 2])),
                lambda: ops.dropout(x, 0.1, torch.tensor([1.0])),
                lambda: ops.dropout(x, 0.1, torch.ones(1, dtype=torch.int64, device="meta")),
                lambda: ops.dropout([1.0], 0.1, 1)]:
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------- route
def route_oracle(z, k, score, bias, groups, top, renorm, scale, g):
    """Plain 64-bit gate: weights, indices, counts and the logits' gradient."""
    z = cpu64(z).numpy()
    t, e = z.shape
    w, idx = np.zeros((t, k)), np.full((t, k), -1)
    dz = np.zeros((t, e))
    per = e // groups
    b = np.zeros(e) if bias is None else cpu64(bias).numpy()
    for i in range(t):
        zi = np.where(np.isnan(z[i]), -INF, z[i])
        m = zi.max()
        if score == "softmax":
            s = np.where(zi > -INF, np.exp(zi - (m if m > -INF else 0)), 0.0)
            s = s / s.sum() if s.sum() > 0 else s
        else:
            s = np.where(zi > -INF, 1 / (1 + np.exp(-np.maximum(zi, -700))), 0.0)
        c = s + b
        ok = (zi > -INF) & (c > -INF)
        if top < groups:
            gv = []
            for j in range(groups):
                best = np.sort(c[j * per:(j + 1) * per][ok[j * per:(j + 1) * per]])[::-1][:2]
                gv.append(best.sum() if len(best) else -INF)
            order = sorted(range(groups), key=lambda j: (-gv[j], j))
            for j in order[top:]:
                ok[j * per:(j + 1) * per] = False
        by = zi if bias is None else c
        order = sorted((j for j in range(e) if ok[j]), key=lambda j: (-by[j], j))[:k]
        r = len(order)
        idx[i, :r] = order
        so = s[order]
        if renorm and r:  # ratios of scores, from their logarithms
            ls = zi[order] if score == "softmax" else -np.logaddexp(0, -zi[order])
            so = np.exp(ls - ls.max())
            so = so / so.sum()
        w[i, :r] = so * scale
        gi = g[i, :r]
        if renorm:
            d = w[i, :r] * (gi - (gi * w[i, :r]).sum() / scale)
        else:
            d = w[i, :r] * gi
        if score == "sigmoid":
            d = d * (1 - s[order])
        dz[i, order] = d
        if score == "softmax" and not renorm:
            dz[i] -= s * (gi * w[i, :r]).sum()
    counts = np.bincount(idx[idx >= 0], minlength=e)
    return (torch.from_numpy(w), torch.from_numpy(idx), torch.from_numpy(counts),
            torch.from_numpy(dz))


def route_check(z, k, score="softmax", bias=None, groups=1, top=None, renorm=True, scale=1.0):
    zl = z.detach().requires_grad_()
    w, idx, counts = ops.route(zl, k, score=score, bias=bias, groups=groups, top_groups=top,
                               renormalize=renorm, scale=scale)
    g = rand(w.shape, 77)
    dz, = torch.autograd.grad(w, [zl], g.to(w.device))
    rw, ri, rc, rd = route_oracle(z, k, score, bias, groups, groups if top is None else top,
                                  renorm, scale, g.double().numpy())
    assert idx.dtype == torch.int32 and counts.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(idx.cpu().long(), ri) and torch.equal(counts.cpu().long(), rc)
    # exponentials of differences of logits |z| <= zm (relative 2 E32 (zm + 1) each) and sums of
    # up to E terms
    e = z.shape[1]
    fin = z[z.isfinite()].abs()
    zm = fin.max().item() if fin.numel() else 0.0
    rel = (e + 16 + 8 * zm) * E32
    check(w, rw, rel * rw + 1e-37, "weights")
    gm = g.abs().amax(dim=1, keepdim=True).double() if g.numel() else 0
    u = half_step(z.dtype)
    wsum = rw.abs().sum(dim=1, keepdim=True)
    small = 2.0 ** -24 if z.dtype == torch.float16 else 1e-37
    check(dz, rd, 4 * rel * gm * torch.maximum(wsum, rd.abs()) + u * rd.abs() + small, "dz")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 64, 2), (5, 3, 3), (17, 16, 4), (33, 17, 5),
                                   (9, 60, 32), (40, 64, 8), (50, 128, 8), (130, 200, 6),
                                   (20, 256, 16), (7, 500, 10), (5, 1024, 32), (600, 8, 2)])
def test_route(device, dtype, t, e, k):
    z = rand((t, e), t + e, dtype, device, 1.5)
    bias = rand((e,), 5, torch.float32, device, 0.1)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            route_check(z, k, score, renorm=renorm, scale=2.5)
            route_check(z, k, score, bias, renorm=renorm)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("e,groups,top,k", [(8, 8, 3, 3), (16, 4, 2, 5), (64, 8, 3, 6),
                                            (128, 2, 1, 8), (256, 8, 4, 8), (192, 64, 5, 15),
                                            (1000, 10, 7, 20), (12, 3, 3, 4)])
def test_route_groups(device, e, groups, top, k):
    for dtype in DTYPES:
        z = rand((37, e), e, dtype, device)
        bias = rand((e,), 6, torch.float32, device, 0.05)
        for score in ("softmax", "sigmoid"):
            route_check(z, k, score, bias, groups, top, scale=2.5)
            route_check(z, k, score, None, groups, top, renorm=False)


@pytest.mark.parametrize("device", DEVICES)
def test_route_ties_and_left_out(device):
    z = torch.zeros((9, 70), device=device)
    z[1, 5:] = 1.0
    z[2, ::7] = -1.0
    z[3, 3:] = -INF      # three are left
    z[4] = -INF          # none
    z[5, 1::2] = math.nan
    z[6] = 200.0         # scores that round to 1, and to 0
    z[7] = -200.0
    z[7, 9] = -199.0
    z[8, 60:] = 3e38
    route_check(z, 5)
    route_check(z[:6], 5, renorm=False)
    for groups, top in ((1, 1), (7, 3), (10, 2)):
        route_check(z, 5, "sigmoid", None, groups, top)
        route_check(z[:6], 5, "sigmoid", None, groups, top, renorm=False)
        bias = torch.zeros(70, device=device)
        bias[10:13] = -INF
        bias[20], bias[33] = math.nan, torch.finfo(torch.float32).min
        route_check(z[:6], 5, "sigmoid", bias, groups, top)
        route_check(z[:6], 5, "softmax", bias, groups, top, renorm=False)
    # near ties: choice values that differ by less than a step of fp32
    z = torch.zeros((4, 40), device=device)
    bias = torch.full((40,), 0.25, device=device)
    z[:, 30] = 2.0 ** -24
    w, idx, _ = ops.route(z, 3, score="sigmoid", bias=bias)
    assert idx.cpu().tolist() == [[30, 0, 1]] * 4
    w, idx, counts = ops.route(z[:0], 3)
    assert w.shape == (0, 3) and not counts.any() and counts.shape == (40,)


@pytest.mark.parametrize("device", DEVICES)
def test_route_strides(device):
    wide = rand((50, 77), 1, torch.float32, device)
    for z in (wide[:, 1:65], wide[:, :64], wide[::2, 4:68], rand((64, 30), 2, device=device).t(),
              rand((1, 64), 3, device=device).expand(20, 64)):
        route_check(z, 4)


def test_route_refusals():
    z = torch.zeros((3, 16))
    b = torch.zeros(16)
    for bad in [lambda: ops.route(z[0], 2), lambda: ops.route(z, 0), lambda: ops.route(z, 17),
                lambda: ops.route(z, 2, groups=3), lambda: ops.route(z, 2, groups=0),
                lambda: ops.route(z, 2, groups=4, top_groups=5),
                lambda: ops.route(z, 2, groups=4, top_groups=0),
                lambda: ops.route(z, 9, groups=4, top_groups=2),
                lambda: ops.route(torch.zeros((3, 1025)), 2),
                lambda: ops.route(torch.zeros((3, 64)), 33), lambda: ops.route(z[:, :0], 1),
                lambda: ops.route(torch.zeros((3, 130)), 2, groups=65),
                lambda: ops.route(z, 2, score="relu"), lambda: ops.route(z, 2, scale=0.0),
                lambda: ops.route(z, 2, scale=math.nan), lambda: ops.route(z, 2, bias=b[:3]),
                lambda: ops.route(z, 2, bias=b.half()), lambda: ops.route(z.double(), 2),
                lambda: ops.route(z.long(), 2), lambda: ops.route([[1.0]], 1)]:
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------ together, as in use
def step(x, gate, experts, items, bias, target, seed, p=0.2, k=2):
    """Denoising features -> gate -> mixture of projections -> softmax over the catalogue."""
    h = ops.dropout(x, p, seed)
    w, idx, counts = ops.route(h.float() @ gate, k)
    dense = (w[:, :, None] * (idx[:, :, None] == torch.arange(len(experts), device=x.device))) \
        .sum(1)
    user = sum(dense[:, e:e + 1] * (h.float() @ experts[e]) for e in range(len(experts)))
    user = user.to(x.dtype)
    return ops.softmax_cross_entropy(user, items, target, bias), counts


def step_inputs(device, dtype, n=37, d=24, e=6, v=211):
    x = rand((n, d), 1, dtype, device)
    leaves = [rand((d, e), 2, torch.float32, device, 0.5),
              rand((e, d, d), 3, torch.float32, device, 0.3), rand((v, d), 4, dtype, device, 0.4),
              rand((v,), 5, torch.float32, device)]
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(6)).to(device)
    t[3::5] = -100
    return x, [q.requires_grad_() for q in leaves], t


@pytest.mark.parametrize("device", DEVICES)
def test_training_step_together(device):
    x, leaves, t = step_inputs(device, torch.float32)
    x.requires_grad_()
    loss, counts = step(x, *leaves, t, 11)
    grads = torch.autograd.grad(loss, [x] + leaves)
    # the same in 64 bits from elementary operations
    p64 = [cpu64(q).requires_grad_() for q in [x] + leaves]
    words = torch.tensor(philox_words(x.numel(), 0, 11)).view(x.shape)
    h = p64[0] * (words >= round(0.2 * 2 ** 32)).double() / 0.8
    z = h @ p64[1]
    top, idx = z.topk(2, dim=1)
    w = torch.softmax(top, 1)
    mixed = torch.stack([(h[:, :, None] * p64[2][idx[:, j]]).sum(1) for j in range(2)], 1)
    user = (w[:, :, None] * mixed).sum(1)
    ref = torch.nn.functional.cross_entropy(user @ p64[3].t() + p64[4], t.cpu())
    want = torch.autograd.grad(ref, p64)
    assert torch.equal(counts.cpu().long(), torch.bincount(idx.reshape(-1), minlength=6))
    # five fp32 stages of at most a few hundred terms: 2^-23 times 2000 of the largest entry
    check(loss, ref.detach(), 2000 * E32 * ref.item(), "loss")
    for i, (g, r) in enumerate(zip(grads, want)):
        check(g, r, 2000 * E32 * r.abs().max().item(), f"grad {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_training_step_captured(dtype):
    """One captured training step, replayed with new inputs and seeds, against the eager step."""
    x, leaves, t = step_inputs("cuda", dtype, n=70, v=600)
    seed = torch.tensor([1], device="cuda")

    def run():
        loss, counts = step(x, *leaves, t, seed)
        return [loss.detach(), counts, *torch.autograd.grad(loss, leaves)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn: neither may use the other's workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for i in range(4):
        x.copy_(rand(x.shape, 50 + i, dtype))
        seed.fill_(100 + i)
        eager = run()
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_other_stream_gives_the_same():
    x, leaves, t = step_inputs("cuda", torch.bfloat16, n=300, v=3000)
    want = step(x, *leaves, t, 5)[0]
    want = [want.detach(), *torch.autograd.grad(want, leaves)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = step(x, *leaves, t, 5)[0]
        got = [got.detach(), *torch.autograd.grad(got, leaves)]
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)  # (fixed order of every sum)


@pytest.mark.gpu
def test_threads_at_once():
    """Calls from several threads, each on a stream of its own."""
    from concurrent.futures import ThreadPoolExecutor
    x, leaves, t = step_inputs("cuda", torch.bfloat16, n=300, v=3000)

    def run(seed):
        loss, counts = step(x, *leaves, t, seed)
        return [loss.detach(), counts, *torch.autograd.grad(loss, leaves)]

    want = [run(s) for s in range(4)]
    torch.cuda.synchronize()

    def worker(seed):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [run(seed) for _ in range(5)]
        stream.synchronize()
        return all(torch.equal(a, b) for g in got for a, b in zip(g, want[seed]))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(worker, range(4)))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 70])
def test_ce_offsets_beyond_32_bits(n):
    """Weights of more than 2^31 elements and 2^32 bytes.  All classes but the last 300 have zero
    weights, so each adds exp(0) to a row's sum."""
    v, d, tail = 1_200_000, 2000, 300
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    w[-tail:] = rand((tail, d), 1, torch.bfloat16, "cuda")
    x = rand((n, d), 2, torch.bfloat16, "cuda", 0.2)
    t = torch.randint(v - tail, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.softmax_cross_entropy(*leaves, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, leaves)
    x64, w64, k = cpu64(x), cpu64(w[-tail:]), t.cpu() - (v - tail)
    z = x64 @ w64.t()
    lse = torch.logsumexp(torch.cat([z, torch.full((n, 1), math.log(v - tail))], 1), 1)
    hot = torch.zeros_like(z)
    hot[torch.arange(n), k] = 1
    zerr = 2 * (d + 10) * E32 * (x64.abs() @ w64.abs().t()).max().item()
    u = half_step(torch.bfloat16)
    check(loss, (lse - z.gather(1, k[:, None])[:, 0]).sum(),
          n * (zerr + 4 * E32 * (lse.abs().max() + 1)) * 2, "loss")
    p, p0 = (z - lse[:, None]).exp(), (-lse).exp()
    # (the classes of zero weights add nothing to a sum of dx, exactly)
    rel = 2 * zerr + 16 * E32 + u + (max(tail, n) + 8) * E32
    check(dx, (p - hot) @ w64, ((p + hot) @ w64.abs()) * (rel + u) + 1e-37, "dx")
    check(dw[-tail:], (p - hot).t() @ x64, ((p + hot).t() @ x64.abs()) * (rel + u) + 1e-37,
          "dw of the last")
    head = dw[[0, v // 2, v - tail - 1]]
    check(head, (p0 @ x64).expand(3, d), (p0 @ x64.abs()).expand(3, d) * (rel + u) + 1e-37,
          "dw of the others")


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 3])
def test_dropout_offsets_beyond_32_bits(offset):
    n = (1 << 31) + 1001
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.3, 9, offset=offset)
    for i in (0, 1 << 30, n - 1001):
        part = ops.dropout(x[:1001], 0.3, 9, offset=offset + i)
        assert torch.equal(y[i:i + 1001], part)


@pytest.mark.gpu
def test_route_offsets_beyond_32_bits():
    e, k, turns = 128, 4, 17000
    base = rand((1000, e), 4, torch.bfloat16, "cuda").requires_grad_()
    up = rand((1000, k), 5, torch.float32, "cuda")
    w, i, c = ops.route(base, k)
    g, = torch.autograd.grad(w, base, up)
    big = base.detach().repeat(turns, 1).requires_grad_()
    bw, bi, bc = ops.route(big, k)
    assert torch.equal(bw.view(turns, 1000, k), w.expand(turns, 1000, k))
    assert torch.equal(bi.view(turns, 1000, k), i.expand(turns, 1000, k))
    assert torch.equal(bc, c * turns)
    bg, = torch.autograd.grad(bw, big, up.repeat(turns, 1))
    for t in (0, turns // 2, turns - 1):
        assert torch.equal(bg.view(turns, 1000, e)[t], g)


def test_route_limits():
    z = torch.zeros(1, 4)
    for scale in (1e39, 1e-39, 1e-60):  # not a normal fp32 number
        with pytest.raises(ValueError, match="scale"):
            ops.route(z, 2, scale=scale)
    with pytest.raises(ValueError, match="tokens"):  # (the loads are 32-bit numbers)
        ops.route(z.expand(1 << 31, 4), 2)


def test_host_large_logits():
    """Sums and probabilities refer to the stored maximum: logits of 1e5 keep their differences."""
    x = torch.tensor([[100000.125]], requires_grad=True)
    w = torch.tensor([[1.0], [1.00001], [0.99999]], requires_grad=True)
    t = torch.tensor([0])
    loss = ops.softmax_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    z = cpu64(x) @ cpu64(w).t()
    p = torch.softmax(z, 1)
    p[0, 0] -= 1
    # sums in 64 bits; the sum of exponentials (2^-24) and the results are rounded to fp32
    check(loss, (z.logsumexp(1) - z[:, 0])[0], 1e-6, "loss")
    check(dw, p.t() @ cpu64(x), 4 * 2.0 ** -24 * 1e5, "dw")
    check(dx, p @ cpu64(w), 4 * 2.0 ** -24 * 2, "dx")


def test_host_engine_in_a_forked_child():
    """The child of a fork has none of the host engine's threads."""
    import multiprocessing
    x = torch.ones(4096)
    want = ops.dropout(x, 0.5, 7)
    fork = multiprocessing.get_context("fork")

    def child(out):
        out.put(bool((ops.dropout(x, 0.5, 7).numpy() == want.numpy()).all()))

    out = fork.Queue()
    p = fork.Process(target=child, args=(out,))
    p.start()
    p.join(30)
    alive = p.is_alive()
    if alive:
        p.kill()
        p.join()
    assert not alive and out.get(timeout=5)


def test_second_derivatives_are_refused():
    """A graph of the gradient gives the same gradient, and an error when it is differentiated."""
    x = rand((5, 8), 1).requires_grad_()
    up = rand((5, 2), 2)
    for f in (lambda: (ops.dropout(x, 0.3, 4) ** 2).sum(),
              lambda: (ops.route(x, 2)[0] * up).sum()):
        plain, = torch.autograd.grad(f(), x)
        g, = torch.autograd.grad(f(), x, create_graph=True)
        assert torch.equal(plain, g.detach())
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v,d,copies", [(130, 8, 1), (515, 40, 1), (515, 40, 40), (300, 1100, 50),
                                        (9000, 100, 1)])
def test_ce_target_at_every_place_of_a_tile_gpu(dtype, v, d, copies):
    """Every class is a target: the first and the last of each lane's, of a wave's and of a tile's
    (also beside a class that is left out)."""
    x = rand((v * copies, d), 1, dtype, "cuda", 0.5)
    w = rand((v, d), 2, dtype, "cuda", 0.5)
    t = torch.arange(v).repeat(copies).cuda()
    ce_check(x, w, t, None, "sum")
    b = rand((v,), 4)
    b[3::4], b[64], b[128 % v] = -INF, -INF, -INF
    t[b.cuda()[t] == -INF] = -100
    ce_check(x, w, t, b.cuda())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_signed_zeros(device, dtype):
    """-0 and +0 are equal: among them the lowest index goes first, on either side of the last
    choice."""
    z = rand((40, 48), 1, dtype, device)
    z[::2] = -z[::2].abs()  # (rows in which the zeros come first)
    z[:, 1::3] = 0.0
    z[:, 4::6] = -0.0
    z[5] = -0.0
    z[6, ::2], z[6, 1::2] = -0.0, 0.0
    z[7, ::2], z[7, 1::2] = 0.0, -0.0
    for score in ("softmax", "sigmoid"):
        for k in (1, 2, 3, 7):
            route_check(z, k, score)
            route_check(z, k, score, renorm=False)
            route_check(z, k, score, None, 8, 3)
            route_check(z, k, score, rand((48,), 2, device=device, scale=0.1))
    for k in (1, 2):  # one +0 (two would be a tie that is looked at again)
        w, idx, counts = ops.route(torch.tensor([[-0.0, 0.0, -1.0], [-2.0, -0.0, 0.0]], dtype=dtype,
                                                device=device), k)
        assert idx.tolist() == [[0, 1][:k], [1, 2][:k]]
    w, idx, counts = ops.route(torch.tensor([[-0.0, 0.0, -1.0, 0.0]], dtype=dtype, device=device),
                               2)
    assert idx.tolist() == [[0, 1]] and counts.tolist() == [1, 1, 0, 0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_infinite_logits(device, dtype):
    """A logit of +inf counts as the largest finite fp32 number: it is chosen, whatever the score,
    the bias and the groups, and its token's weights are numbers."""
    z = rand((12, 40), 1, dtype, device)
    z[0, 7] = INF
    z[1, 30], z[1, 3] = INF, INF
    z[2] = INF
    z[3, 5], z[3, 6], z[3, 7] = INF, math.nan, -INF
    z[4, 11], z[4, 12] = INF, torch.finfo(dtype).max
    capped = z.float().clamp(max=torch.finfo(torch.float32).max)
    bias = rand((40,), 2, device=device, scale=0.1)
    g = rand((12, 4), 3, device=device)
    for score in ("softmax", "sigmoid"):
        for b, groups, top in ((None, 1, 1), (bias, 1, 1), (None, 8, 3), (bias, 8, 3)):
            for renorm in (True, False):
                got = []
                for logits in (z, capped):
                    leaf = logits.clone().requires_grad_()
                    out = ops.route(leaf, 4, score=score, bias=b, groups=groups, top_groups=top,
                                    renormalize=renorm)
                    got.append((*out, torch.autograd.grad(out[0], leaf, g)[0]))
                (w, i, c, d), (rw, ri, rc, rd) = got
                assert torch.equal(i, ri) and torch.equal(c, rc) and torch.equal(w, rw)
                assert torch.equal(d, rd.to(dtype))
                assert w.isfinite().all() and d.isfinite().all()
                assert (i[:, 0] >= 0).all()
                if b is None:
                    assert i[0, 0] == 7 and i[1, :2].tolist() == [3, 30]
                    assert i[2].tolist() == [0, 1, 2, 3] and i[4, 0] == 11


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
def test_ce_upstream_gradients_that_are_no_numbers(device, dtype, bad):
    """An upstream gradient that is infinite or NaN reaches its own row's gradient of x only; rows
    and classes that are left out keep the gradient 0."""
    sizes = [(9, 30, 16), (70, 300, 64)]
    if device == "cuda":
        sizes += [(300, 9000, 100), (300, 50_000, 128), (520, 9000, 1100)]
    for n, v, d in sizes:
        x = rand((n, d), 1, dtype, device, 0.3).requires_grad_()
        w = rand((v, d), 2, dtype, device, 0.3).requires_grad_()
        b = rand((v,), 3, device=device)
        b[4::5] = -INF
        b.requires_grad_()
        t = (torch.arange(n, device=device) * 5 + 1) % v // 5 * 5
        t[2::7] = -100
        up = torch.rand(n, generator=torch.Generator().manual_seed(4)).to(device) + 0.5
        up[0] = 2.0  # (the largest that is a number)
        worse = up.clone()
        worse[3], worse[n - 1] = bad, bad
        assert t[3] >= 0 and t[n - 1] >= 0
        up[3], up[n - 1] = 0.0, 0.0
        rows = ops.softmax_cross_entropy(x, w, t, b, reduction="none")
        want, = torch.autograd.grad(rows, [x], up, retain_graph=True)
        dx, dw, db = torch.autograd.grad(rows, [x, w, b], worse)
        others = torch.ones(n, dtype=torch.bool, device=device)
        others[3], others[n - 1] = False, False
        assert torch.equal(dx[others], want[others]), (n, v, d)
        assert not dx[~others].isfinite().any()
        out = b == -INF
        assert not dw[out].any() and not db[out].any()
        assert not dw[~out].isfinite().any() and not db[~out].isfinite().any()
        # one number for all rows
        loss = ops.softmax_cross_entropy(x, w, t, b)
        dx, dw, db = torch.autograd.grad(loss, [x, w, b], torch.tensor(bad, device=device))
        assert not dx[t == -100].any() and not dx[t >= 0].isfinite().any()
        assert not dw[out].any() and not db[out].any()
        loss = ops.softmax_cross_entropy(x, w, torch.full_like(t, -100), b)
        for g in torch.autograd.grad(loss, [x, w, b], torch.tensor(bad, device=device)):
            assert not g.any()


def ce_plan(x, w, b, grad):
    """(rows of a turn, classes of a piece, fp32 operands split) of a call"""
    elem = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[x.dtype]
    return _loader.load().softmax_ce_plan(elem, x.data_ptr(), x.stride(0), w.data_ptr(),
                                          w.stride(0), 0 if b is None else b.data_ptr(),
                                          *x.shape[:1], *w.shape, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,v,d,split", [(torch.bfloat16, 8190, 140_001, 64, False),
                                               (torch.float16, 8000, 131_100, 24, False),
                                               (torch.float32, 2000, 300_001, 16, True),
                                               (torch.float32, 100, 1_100_003, 8, False)])
@pytest.mark.parametrize("bias", [False, True])
def test_ce_several_pieces_gpu(dtype, n, v, d, split, bias):
    """Classes in several pieces, weights, targets and left-out classes in each, and the weights'
    magnitudes different from piece to piece."""
    x = rand((n, d), 1, dtype, "cuda", 0.5)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    w = rand((v, d), 2, torch.float32, "cuda", 1 / math.sqrt(d)) + 0.25 / math.sqrt(d)
    b = None
    if bias:
        b = rand((v,), 4, device="cuda")
        b[5::11] = -INF
        b[t] = 0.25
    t[::9] = -100
    plan = ce_plan(x, w.to(dtype), b, True)
    pieces = range(0, v, plan[1])
    assert len(pieces) > 1 and plan[2] == split
    for i, c in enumerate(pieces):
        w[c:c + plan[1]] *= (1.0, 0.0625, 4.0)[i % 3]
        assert ((t >= c) & (t < c + plan[1])).any()
    w = w.to(dtype)
    leaves = [q.requires_grad_() for q in (x, w, b) if q is not None]
    loss = ops.softmax_cross_entropy(x, w, t, b, reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    with torch.no_grad():
        kept = torch.nonzero(t >= 0)[:, 0]
        xd, wd = x.double()[kept], w.double()
        z = xd @ wd.t()
        if bias:
            z += b.double()
        hot = t[kept][:, None]
        lse = torch.logsumexp(z, 1)
        ref = (lse - z.gather(1, hot)[:, 0]).sum()
        zerr = (d + 8) * E32 * (xd.norm(dim=1).max() * wd.norm(dim=1).max()).item() + \
            4 * E32 * lse.abs().max().item()
        assert abs(loss.double() - ref) <= n * 2 * zerr + 4 * E32 * ref.abs()
        p = z.sub_(lse[:, None]).exp_()
        one = torch.ones_like(hot, dtype=torch.float64)
        mags = [p.scatter_add(1, hot, one)]
        p.scatter_add_(1, hot, -one)
        wants = [torch.zeros(n, d, device="cuda").double().index_copy(0, kept, p @ wd),
                 p.t() @ xd, p.sum(0)]
        mags = [torch.zeros(n, d, device="cuda").double().index_copy(0, kept, mags[0] @ wd.abs()),
                mags[0].t() @ xd.abs(), mags[0].sum(0)]
        u = half_step(dtype)
        # dx: a run of at most 8192 classes, 16 of them (2 in fp32, with as many fewer classes) a
        # step, and the runs' and pieces' sums: below 1024 steps of two roundings
        for name, got, want, mag, steps in zip(("dx", "dw", "db"), grads, wants, mags,
                                               (2048, n + 8, n + 8)):
            uo = u if name != "db" else 0
            rel = 2 * zerr + 16 * E32 + uo + steps * E32
            # fp16: dz keeps 2^-39; results keep half of 2^-24
            tiny = 2.0 ** -25 + 2.0 ** -39 * {"dx": v, "dw": n, "db": 0}[name] * 4 \
                if dtype == torch.float16 and name != "db" else 1e-37
            err = (got.double() - want).abs() - (mag * (rel + uo) + uo * want.abs() + tiny)
            assert not (err > 0).any(), (name, err.max())


@pytest.mark.gpu
def test_ce_rows_in_several_turns_gpu():
    """More rows than one turn of the forward pass keeps statistics for: a row's loss is that of a
    call on its own part of the rows, but for the order in which 7813 tiles' sums are joined (up to
    489 joins in a row by a thread, 4 to 10 levels above them, three roundings each)."""
    n, v, d = 20_000, 2_000_000, 4
    x, w = rand((n, d), 1, torch.bfloat16, "cuda"), rand((v, d), 2, torch.bfloat16, "cuda")
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    t[::7] = -100
    assert ce_plan(x, w, None, False)[0] < n <= 2 * ce_plan(x, w, None, False)[0]
    whole = ops.softmax_cross_entropy(x, w, t, reduction="none")
    parts = torch.cat([ops.softmax_cross_entropy(x[a:a + 5000], w, t[a:a + 5000], reduction="none")
                       for a in range(0, n, 5000)])
    assert ((whole - parts).abs() <= 2 * 499 * 3 * E32 + 4 * E32 * parts.abs()).all()
    mean = ops.softmax_cross_entropy(x, w, t)
    ref = whole.double().sum() / (t != -100).sum()
    assert abs(mean.item() - ref.item()) <= E32 * abs(ref.item())
    # some rows against 64 bits, on both sides of the border
    turn = ce_plan(x, w, None, False)[0]
    some = torch.tensor([1, 2, turn - 1, turn, turn + 1, n - 1], device="cuda")
    z = x[some].double() @ w.double().t()
    ref = torch.logsumexp(z, 1) - z.gather(1, t[some].clamp(min=0)[:, None])[:, 0]
    ref[t[some] == -100] = 0
    zerr = (d + 8) * E32 * (x.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item()
    tol = 2 * zerr + 499 * 3 * E32 + 4 * E32 * (ref.abs() + 20)
    assert ((whole[some] - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_ce_fitted_rows_of_many_classes_gpu():
    """Rows whose loss is 2e-3 to 1e-7 over a million classes: the other classes' probabilities,
    down to 2^-43, keep their relative precision in dW, and their sum reaches dx."""
    n, v, d, k = 130, 1_000_003, 12, 777
    w = rand((v, d), 1, device="cuda", scale=0.3) + 1
    w[:, 0] = 0
    w[k] = 0
    w[k, 0] = 1
    x = rand((n, d), 2, device="cuda", scale=0.3)
    x[:, 0] = torch.linspace(20, 30, n)
    t = torch.full((n,), k, device="cuda")
    for up in (None, 2.0 ** -torch.arange(n).remainder(9).float().cuda()):
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        rows = ops.softmax_cross_entropy(*leaves, t, reduction="none")
        rows = rows if up is None else rows * up
        dx, dw = torch.autograd.grad(rows.sum(), leaves)
        x64, w64 = x.double(), w.double()
        z = x64 @ w64.t()
        lse = torch.logsumexp(z, 1)
        zerr = (d + 8) * E32 * (x64.abs() @ w64.abs().t()).max().item() + 4 * E32 * lse.max().item()
        p = (z - lse[:, None]).exp()
        p[:, k] = 0  # the target's dz is minus the sum of the others
        miss = p.sum(1)
        if up is not None:
            p *= up[:, None].double()
        rel = 2 * zerr + 16 * E32
        others = torch.arange(v, device="cuda") != k
        want, mag = p.t() @ x64, p.t() @ x64.abs()
        err = (dw.double() - want).abs()[others] / mag[others]
        assert err.max() <= rel + (n + 8) * E32, err.max()
        # dx beyond the first feature: the target's weights are 0 there
        want, mag = p @ w64, p @ w64.abs()
        err = (dx.double() - want).abs()[:, 1:] / mag[:, 1:]
        assert err.max() <= rel + v * E32, err.max()
        # ... and in the first, the target's alone: p - 1 in fp32
        scale = 1.0 if up is None else up.double()
        assert ((dx[:, 0].double() + miss * scale).abs()
                <= scale * (miss * rel + 2 * zerr + 8 * E32)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
def test_ce_unlikely_classes_gpu(bias):
    """Untrained rows over 300 thousand classes whose probabilities range over 2^-10 to 2^-50: each
    class's row of dW has the relative precision of fp32 sums."""
    n, v, d = 200, 300_007, 28
    x, w = rand((n, d), 1, device="cuda"), rand((v, d), 2, device="cuda", scale=0.5)
    t = torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    b = None
    if bias:
        b = rand((v,), 4, device="cuda", scale=3.0)
        b[t] = 1.0
    ce_check(x, w, t, b, "sum")
    ce_check(x, w, t, b, "none", torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda()
             + 0.5)


def test_host_engine_lets_a_forked_child_end():
    """A child of a fork that ends normally (not by os._exit) takes down none of the parent's
    threads."""
    import subprocess
    import sys
    from pathlib import Path
    code = ("import os, sys, torch\n"
            "from oap_mllib_amd import ops\n"
            "x = torch.ones(4096)\n"
            "ops.dropout(x, 0.5, 7)\n"
            "pid = os.fork()\n"
            "if pid == 0:\n"
            "    ops.dropout(x, 0.5, 7)\n"
            "    sys.exit(0)\n"
            "sys.exit(os.waitpid(pid, 0)[1])\n")
    root = Path(__file__).resolve().parent.parent
    assert subprocess.run([sys.executable, "-c", code], timeout=60, cwd=root).returncode == 0


def test_numbers_beyond_64_bits_and_row_lengths_are_refused():
    x, w, t = rand((4, 8), 1), rand((9, 8), 2), torch.zeros(4, dtype=torch.int64)
    for bad in (1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            ops.softmax_cross_entropy(x, w, t, ignore_index=bad)
    for fine in ((1 << 63) - 1, -(1 << 63)):
        assert ops.softmax_cross_entropy(x, w, t, ignore_index=fine).isfinite()
    long = torch.zeros(1, 1).expand(2, (1 << 20) + 1)
    with pytest.raises(ValueError, match="features"):
        ops.softmax_cross_entropy(long, long, t[:2])
    for offset in (1 << 64, 1 << 70):  # (no element at all, but an index that is none)
        with pytest.raises(ValueError, match="offset"):
            ops.dropout(x[:0], 0.1, 1, offset=offset)
    assert ops.dropout(x[:0], 0.1, 1, offset=(1 << 64) - 1).numel() == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_ce_loss_of_rows_that_their_target_decides(device, dtype):
    """Where all other logits lie at least 60 below the target's, the loss is 0 but for e^-60 per
    class: never negative, and no larger for large logits (whose products are exact here: x and
    weight hold small integers)."""
    sizes = [(1, 1, 3), (4, 60, 24), (70, 300, 64)]
    if device == "cuda":
        sizes += [(7, 3000, 40), (20, 30_000, 24), (50, 30_000, 24), (300, 9000, 100),
                  (160, 200_000, 48), (1100, 30_001, 40), (520, 9000, 1100)]
    for n, v, d in sizes:
        w = rand((v, d), 1).sign()
        t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
        own = torch.arange(n) % 7 + 2  # the target's logit is own * d, the others' own * |sum| < it
        x = w[t] * own[:, None]
        z = x @ w.t()
        gap = z.gather(1, t[:, None]) - z.scatter(1, t[:, None], -INF).amax(1, keepdim=True)
        x = x * torch.ceil(60 / gap.clamp(min=1))
        keep = gap[:, 0] >= 1  # (another class may have the same weights)
        assert keep.any() and x.abs().max() < 1024
        args = [q.to(dtype).to(device) for q in (x[keep], w)] + [t[keep].to(device)]
        for b in (None, torch.zeros(v, device=device)):
            loss = ops.softmax_cross_entropy(*args, b, reduction="none")
            assert (loss >= 0).all() and (loss <= 2 * E32).all(), (n, v, d, loss.min(), loss.max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [10.0, 1000.0])
def test_ce_gradients_of_large_logits(device, dtype, scale):
    """Logits of 1e4 to 1e8, whose fp32 sums are off by much more than one: another class lies far
    above the target, so its probability is 1 and its dz the upstream gradient, the target's is
    minus that and all others' are 0.  The pass that forms the maxima has to see the same logits
    as the one that forms the gradients."""
    sizes = [(1, 50, 100), (1, 50, 1000), (4, 60, 101), (7, 90, 100), (70, 300, 64)]
    if device == "cuda":
        sizes += [(8, 30_000, 100), (20, 30_000, 100), (300, 15_000, 400), (520, 9000, 1100)]
    for n, v, d in sizes:
        x, w = rand((20 * n, d), 1, dtype, device, scale), rand((v, d), 2, dtype, device, scale)
        z = x.double() @ w.double().t()
        top2 = z.topk(2, dim=1)
        # (sums of d products in any order: d 2^-23 of the sum of their magnitudes)
        error = d * E32 * (x.double().abs() @ w.double().abs().t()).amax(1)
        gap = top2.values[:, 0] - top2.values[:, 1]
        rows = (gap > 2 * error + 100).nonzero()[:n, 0]
        assert len(rows) == n
        x, best, t = x[rows], top2.indices[rows, 0], z[rows].argmin(1)
        for b in (None, torch.zeros(v, device=device, requires_grad=True)):
            leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
            leaves += [b] if b is not None else []
            loss = ops.softmax_cross_entropy(leaves[0], leaves[1], t, b, reduction="none")
            grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
            xr, u = x.double(), half_step(dtype)
            want = [w.double()[best] - w.double()[t],
                    torch.zeros(v, d, device=device).double()
                    .index_add_(0, best, xr).index_add_(0, t, -xr)]
            mags = [w.double()[best].abs() + w.double()[t].abs(),
                    torch.zeros(v, d, device=device).double()
                    .index_add_(0, best, xr.abs()).index_add_(0, t, xr.abs())]
            for got, ref, mag in zip(grads, want, mags):
                err = (got.double() - ref).abs() - (n + 8) * E32 * mag \
                    - u * ref.abs() - 1e-37  # (the others' e^-100)
                assert (err <= 0).all(), (n, v, d, err.max())
            if b is not None:
                count = torch.zeros(v, device=device).double()
                one = torch.ones(n, device=device).double()
                count.index_add_(0, best, one).index_add_(0, t, -one)
                assert ((grads[2].double() - count).abs() <= (n + 8) * E32 * n).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e5, 1e9, 1e15])
def test_ce_gradients_of_huge_logits(device, dtype, scale):
    """The same at logits of 1e11 to 1e31, where the rounding of a maximum alone passes the range
    of a power."""
    test_ce_gradients_of_large_logits(device, dtype, scale)
    x, w = rand((70, 64), 1, dtype, device, scale), rand((300, 64), 2, dtype, device, scale)
    t = torch.arange(70, device=device)
    loss = ops.softmax_cross_entropy(x, w, t, reduction="none")
    z = x.double() @ w.double().t()
    want = z.amax(1) - z[torch.arange(70, device=device), t]
    error = 64 * E32 * (x.double().abs() @ w.double().abs().t()).amax(1)
    assert ((loss.double() - want).abs() <= 2 * error + 4 * E32 * want + math.log(300)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(5, 5000, 100), (6, 3000, 1032), (7, 33, 40), (8, 999, 1024),
                                   (8, 30_000, 64), (5, 7, 8), (2, 2000, 200), (8, 1, 4),
                                   (3, 4000, 512), (1, 3000, 2048), (4, 70, 1000)])
def test_ce_losses_of_few_rows_gpu(dtype, n, v, d):
    """Losses whose gradients nobody asks for: up to eight rows at once from registers."""
    x, w = rand((n, d), 1, dtype, "cuda", 0.5), rand((v, d), 2, dtype, "cuda", 0.5)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    b = rand((v,), 4)
    b[1::7] = -INF
    b[t] = 0.5
    b = b.cuda()
    none = (False, False, False)
    for bias in (None, b):
        ce_check(x, w, t.cuda(), bias, reduction="none", want=none)
    with torch.no_grad():  # (the same without a graph, whatever wants gradients)
        leaf = w.clone().requires_grad_()
        a = ops.softmax_cross_entropy(x, leaf, t.cuda(), b, reduction="none")
        assert torch.equal(a, ops.softmax_cross_entropy(x, w, t.cuda(), b, reduction="none"))
    t[n // 2] = -100
    x[n // 2] = math.nan
    w[b == -INF] = math.nan
    ce_check(x, w, t.cuda(), b, want=none)


@pytest.mark.gpu
def test_ce_few_rows_beyond_32_bits():
    """One row without gradients, weights of more than 2^31 elements."""
    v, d, tail = 1_200_000, 2000, 300
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    w[-tail:] = rand((tail, d), 1, torch.bfloat16, "cuda")
    x = rand((1, d), 2, torch.bfloat16, "cuda", 0.2)
    t = torch.tensor([v - 7], device="cuda")
    z = cpu64(x) @ cpu64(w[-tail:]).t()
    lse = torch.logsumexp(torch.cat([z, torch.full((1, 1), math.log(v - tail))], 1), 1)
    zerr = 2 * (d + 10) * E32 * (cpu64(x).abs() @ cpu64(w[-tail:]).abs().t()).max().item()
    check(ops.softmax_cross_entropy(x, w, t, reduction="none"), lse - z[:, tail - 7],
          zerr + 4 * E32 * (lse.abs().max() + 1), "loss")


@pytest.mark.gpu
def test_ce_split_rows_in_several_turns_gpu():
    """fp32 rows in two turns, classes in many pieces; losses and dx of rows on both sides of the
    border against 64 bits, some of them with losses of 1e-3 to 1e-6."""
    n, v, d = 9000, 2_000_000, 4
    x, w = rand((n, d), 1, device="cuda"), rand((v, d), 2, device="cuda", scale=0.5)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3)).cuda()
    w[:, 0] = 0
    w[77] = 0
    w[77, 0] = 1
    rows, classes, split = ce_plan(x, w, None, False)
    assert rows < n and split and ce_plan(x, w, None, True)[1] * 2 < v
    some = torch.tensor([0, 1, rows - 2, rows - 1, rows, rows + 1, n - 1], device="cuda")
    x[some, 0] = torch.tensor([3.0, 22.0, 25.0, 28.0, 28.0, 25.0, 22.0], device="cuda")
    t[some] = 77
    leaf = x.clone().requires_grad_()
    loss = ops.softmax_cross_entropy(leaf, w, t, reduction="none")
    dx, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    w64 = w.double()
    z = x[some].double() @ w64.t()
    lse = torch.logsumexp(z, 1)
    zerr = (d + 8) * E32 * (x[some].double().norm(dim=1).max() * w64.norm(dim=1).max()).item() \
        + 4 * E32 * lse.abs().max().item()
    # (15625 tiles of 128 classes: up to 977 joins in a row by a thread, three roundings each)
    ref = lse - z[:, 77]
    tol = 2 * zerr + 1000 * 3 * E32 + 4 * E32 * (ref.abs() + 20)
    assert ((loss[some].double() - ref).abs() <= tol).all()
    p = (z - lse[:, None]).exp()
    p[:, 77] = 0
    want, mag = p @ w64, p @ w64.abs()
    err = (dx[some].double() - want).abs()[:, 1:] / mag[:, 1:]
    assert (err <= 2 * zerr + 16 * E32 + 4000 * E32).all()
