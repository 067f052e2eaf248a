"""Training ops on torch tensors: the softmax loss over a catalogue, dropout from a counter-based
generator and the top-k gate of a mixture of experts.

A GPU tensor's op runs on its device and on torch's current stream there, without a
synchronisation, so it orders like any torch op and can be captured into a graph; its workspace
comes from torch's allocator for the length of the call.  A CPU tensor goes through the native
host engine (fp32 in, sums in fp64).  Float32, bfloat16 and float16 are taken; sums, softmax
statistics and choices are held in 32 bits or more, and a result is rounded once.

Before a backward pass is captured, what keeps an eager graph of the same leaves alive (its loss)
has to go: torch ties a leaf's gradient to the stream of the first graph that uses the leaf, and
a capture that waits for another stream fails.

The ops are local to the process: with row shards every rank calls them on its own rows and
reduces what it needs, as with any torch op.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _loader

__all__ = ["dropout", "route", "softmax_cross_entropy"]

_ELEM = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}
_M64 = (1 << 64) - 1
_F32 = torch.finfo(torch.float32)


def _float_tensor(name: str, t, dim: int | None = None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.dtype not in _ELEM:
        raise ValueError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if not (t.is_cuda or t.is_cpu) or t.layout != torch.strided:
        raise ValueError(f"{name}: expected a dense CPU or GPU tensor")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name}: expected a {dim}-D tensor, got shape {tuple(t.shape)}")


def _same(name: str, t, ref, shape=None, dtype=None):
    """t lies where ref does (and has the shape and type)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.device != ref.device:
        raise ValueError(f"{name}: on {t.device}, expected {ref.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")


def _rows(t):
    """A 2-D tensor whose rows are contiguous (a copy where they are not), and its row stride."""
    n, d = t.shape
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t, t.stride(0) if n > 1 else max(d, 1)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _where(t) -> tuple[int, int]:
    """(device, stream) of a native call; (-1, 0) is the host engine."""
    if t.is_cuda:
        index = t.get_device()
        # (the handle itself: a Stream object costs as much as a small op's launch)
        return index, torch._C._cuda_getCurrentRawStream(index)
    return -1, 0


def _first_order(backward):
    """A backward pass that refuses a second derivative.  Where no graph of the gradient is asked
    for, there is none to refuse, and the wrapper's 5 of a small op's 70 us are saved."""
    checked = once_differentiable(backward)

    def run(ctx, *grads):
        return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


def _work(nbytes: int, t):
    return torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None


# --------------------------------------------------------------------- softmax cross entropy
class _SoftmaxCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index, reduction, train):
        native = _loader.load()
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        n, d = x.shape
        v = weight.shape[0]
        # per row: max and sum and 1 - p of the target for the gradients, and the loss
        rows = torch.empty(4 * n, dtype=torch.float32, device=x.device)
        stat = rows.data_ptr()
        miss, loss = stat + 8 * n, stat + 12 * n
        out = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32,
                          device=x.device)
        total = 0
        if reduction == "none":
            loss = out.data_ptr()
        else:
            total = out.data_ptr()
        elem = _ELEM[x.dtype]
        dev, stream = _where(x)
        head = (elem, _ptr(xr), ldx, _ptr(wr), ldw, _ptr(bias))
        work = None
        if dev >= 0:
            work = _work(native.softmax_ce_forward_bytes(*head, n, v, d, train), x)
        native.softmax_ce_forward(dev, stream, *head, _ptr(target), ignore_index, n, v, d,
                                  train, loss, stat, miss, total, reduction == "mean",
                                  _ptr(work))
        ctx.save_for_backward(x, weight, bias, target, rows)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return out

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        native = _loader.load()
        x, weight, bias, target, rows = ctx.saved_tensors
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        n, d = x.shape
        v = weight.shape[0]
        want = ctx.needs_input_grad[:3]
        grad = grad.contiguous()
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device) if want[0] else None
        dw = torch.empty((v, d), dtype=x.dtype, device=x.device) if want[1] else None
        db = torch.empty(v, dtype=torch.float32, device=x.device) if want[2] else None
        elem = _ELEM[x.dtype]
        dev, stream = _where(x)
        head = (elem, _ptr(xr), ldx, _ptr(wr), ldw, _ptr(bias))
        work = None
        if dev >= 0:
            work = _work(native.softmax_ce_backward_bytes(*head, n, v, d, *want), x)
        native.softmax_ce_backward(dev, stream, *head, _ptr(target), ctx.ignore_index, n, v, d,
                                   _ptr(rows), _ptr(rows) + 8 * n, _ptr(grad),
                                   ctx.reduction == "none", ctx.reduction == "mean", _ptr(dx),
                                   _ptr(dw), _ptr(db), _ptr(work))
        return dx, dw, db, None, None, None, None


def softmax_cross_entropy(x, weight, target, bias=None, *, ignore_index: int = -100,
                          reduction: str = "mean"):
    """Cross entropy of a softmax over the rows of ``weight``: for every row of ``x`` (n x d) the
    loss ``log sum_j exp(z_j) - z_target`` with ``z = x . weight^T + bias`` (weight: classes x d,
    bias: classes).  The n x classes logits are never stored; the gradients for ``x``, ``weight``
    and ``bias`` form them again.

    ``target`` (n integers) holds the class of each row; rows with ``ignore_index`` have no loss
    and no gradient, whatever ``x`` holds there.  A class whose bias is ``-inf`` is left out: it
    has no probability and no gradient, whatever ``weight`` holds there, and a row whose target
    it is has the loss ``inf`` and the gradient of the classes that are left (finite biases below
    -2.3e38 exclude nothing and count as equal).  A target that is
    no class and not ``ignore_index`` gives its row the loss NaN and no gradient.

    ``reduction``: "mean" over the rows that are not ignored (0 if all are), "sum" or "none"
    (n losses; a row with the upstream gradient 0 takes no part in the gradients, whatever ``x``
    holds there).  Losses are float32, the gradients of ``x`` and ``weight`` have their type.
    Larger float32 problems form their products from 22 bits of every number (at least 2^-40 of its
    row's largest in ``x``, of all classes' largest in ``weight``; in the gradient of ``weight``
    2^-40 of all rows' largest in ``x``).  In float16 the coefficients of the gradients, upstream
    gradient times (probability - target), keep 11 bits down to 2^-28 of the largest upstream
    gradient and nothing below 2^-39 of it, so unlikely classes of a large catalogue, and rows with
    a small upstream gradient, lose bits of their gradient there.
    """
    _float_tensor("x", x, 2)
    _float_tensor("weight", weight, 2)
    n, d = x.shape
    v = weight.shape[0]
    if not 1 <= d <= 1 << 20 or v < 1:
        raise ValueError(f"softmax_cross_entropy: {d} features (1 to 2^20), {v} classes")
    _same("weight", weight, x, (v, d), x.dtype)
    _same("target", target, x, (n,))
    if target.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"target: expected int64 or int32, got {target.dtype}")
    if bias is not None:
        _float_tensor("bias", bias, 1)
        _same("bias", bias, x, (v,))
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index: expected a 64-bit integer, got {ignore_index}")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction: expected 'mean', 'sum' or 'none', got {reduction!r}")
    if target.dtype != torch.int64 or not target.is_contiguous():
        target = target.long().contiguous()
    if not x.is_cuda and x.dtype != torch.float32:
        x, weight = x.float(), weight.float()
    train = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, weight, bias))
    return _SoftmaxCrossEntropy.apply(x, weight, bias, target, ignore_index, reduction, train)


# ----------------------------------------------------------------------------------- dropout
def _drop(x, residual, p, seed, offset):
    y = torch.empty_like(x)
    dev, stream = _where(x)
    tensor = isinstance(seed, torch.Tensor)
    _loader.load().dropout(dev, stream, _ELEM[x.dtype], _ptr(x), _ptr(residual), _ptr(y),
                           x.numel(), offset, 0 if tensor else seed, _ptr(seed) if tensor else 0,
                           p)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.p, ctx.offset = p, offset
        ctx.seed = None
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)  # (a seed that is changed in between is an error)
        else:
            ctx.seed = seed
        return _drop(x.contiguous(), None if residual is None else residual.contiguous(), p, seed,
                     offset)

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _drop(grad.contiguous(), None, ctx.p, seed, ctx.offset)
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p: float, seed, *, offset: int = 0, residual=None):
    """``x / (1 - p)`` where an element is kept, 0 where it is dropped (probability ``p``), plus
    ``residual``.  The mask is not stored: it is a function of ``seed`` and of the element's
    index, formed again for the gradient.

    Element i (in row-major order) is kept when word ``(offset + i) & 3`` of Philox4x32-10 at
    counter ``(offset + i) >> 2`` under the key ``seed`` is at least ``round(p 2^32)``; a rank
    that holds the rows from r on of a global table with d columns passes ``offset = r * d`` and
    draws what one process would draw.  ``seed`` is an integer of at most 64 bits or a tensor of
    one int64 on x's device, which the kernel reads: a captured graph draws a new mask in every
    replay if the program changes it in between.  Every call of a program needs a seed (or a
    range of offsets) of its own.
    """
    _float_tensor("x", x)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p: expected a probability, got {p}")
    offset = int(offset)
    if not 0 <= offset < 1 << 64 or offset + x.numel() > 1 << 64:
        raise ValueError(f"offset: element indices must lie in [0, 2^64), got offset {offset}")
    if isinstance(seed, torch.Tensor):
        _same("seed", seed, x, dtype=torch.int64)
        if seed.numel() != 1:
            raise ValueError(f"seed: expected one number, got shape {tuple(seed.shape)}")
        seed = seed.detach()
    else:
        seed = int(seed)
        if not -(1 << 63) <= seed <= _M64:
            raise ValueError(f"seed: expected at most 64 bits, got {seed}")
        seed &= _M64
    if residual is not None:
        _same("residual", residual, x, x.shape, x.dtype)
    if not x.is_cuda and x.dtype != torch.float32:
        r32 = None if residual is None else residual.float()
        return _Dropout.apply(x.float(), r32, p, seed, offset).to(x.dtype)
    return _Dropout.apply(x, residual, p, seed, offset)


# ------------------------------------------------------------------------------------- route
class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, groups, top_groups, sigmoid, renormalize, scale):
        native = _loader.load()
        z, ld = _rows(logits)
        t, e = logits.shape
        dev, stream = _where(logits)
        weights = torch.empty((t, k), dtype=torch.float32, device=logits.device)
        indices = torch.empty((t, k), dtype=torch.int32, device=logits.device)
        counts = torch.empty(e, dtype=torch.int32, device=logits.device)
        work = _work(native.route_partial_bytes(t, e) if dev >= 0 else 0, logits)
        native.route(dev, stream, _ELEM[logits.dtype], _ptr(z), ld, _ptr(bias), t, e, k, groups,
                     top_groups, sigmoid, renormalize, scale, _ptr(weights), _ptr(indices),
                     _ptr(counts), _ptr(work))
        ctx.save_for_backward(logits, weights, indices)
        ctx.args = (k, sigmoid, renormalize, scale)
        ctx.mark_non_differentiable(indices, counts)
        ctx.set_materialize_grads(False)  # (no zeros for the integers' gradients)
        return weights, indices, counts

    @staticmethod
    @_first_order
    def backward(ctx, grad, _indices, _counts):
        if grad is None:
            return (None,) * 8
        logits, weights, indices = ctx.saved_tensors
        k, sigmoid, renormalize, scale = ctx.args
        z, ld = _rows(logits)
        t, e = logits.shape
        dev, stream = _where(logits)
        grad = grad.contiguous()
        out = torch.empty((t, e), dtype=logits.dtype, device=logits.device)
        _loader.load().route_grad(dev, stream, _ELEM[logits.dtype], _ptr(z), ld, _ptr(weights),
                                  _ptr(indices), _ptr(grad), t, e, k, sigmoid, renormalize, scale,
                                  _ptr(out))
        return (out,) + (None,) * 7


def route(logits, k: int, *, score: str = "softmax", bias=None, groups: int = 1,
          top_groups: int | None = None, renormalize: bool = True, scale: float = 1.0):
    """Chooses ``k`` of E experts for every row of ``logits`` (tokens x E).  Returns
    ``(weights float32 [tokens, k], indices int32 [tokens, k], counts int32 [E])``, the chosen in
    falling order and ``counts`` the number of tokens of each expert.

    Scores are the ``score`` ("softmax" or "sigmoid") of the logits.  The choice goes by score +
    ``bias`` (E float32 numbers that balance the experts' loads; they enter nothing else and get
    no gradient), without a bias by the logits; equal values go to the lowest index.  With
    ``groups`` > ``top_groups`` the experts form ``groups`` equal runs and only those of the
    ``top_groups`` runs with the highest sum of their two best values can be chosen.  What
    decides is formed in 64 bits.  A weight is the expert's score, over the sum of the chosen
    scores if ``renormalize``, times ``scale``.

    An expert whose logit is ``-inf`` or NaN, or whose bias is ``-inf`` or NaN, is left out; where
    fewer than ``k`` are left the last slots hold index -1 and weight 0.  A logit of ``+inf`` counts
    as the largest finite float32 number.  At most 1024 experts, 32 choices, 64 groups and 2^31 - 1
    tokens.  The gradient goes from ``weights`` to ``logits``.
    """
    _float_tensor("logits", logits, 2)
    native = _loader.load()
    t, e = logits.shape
    if t >= 1 << 31:
        raise ValueError(f"logits: expected less than 2^31 tokens, got {t}")
    if not 1 <= e <= native.route_max_experts:
        raise ValueError(f"logits: expected 1 to {native.route_max_experts} experts, got {e}")
    k, groups = int(k), int(groups)
    top_groups = groups if top_groups is None else int(top_groups)
    if not 1 <= groups <= native.route_max_groups or e % groups:
        raise ValueError(f"groups: {groups} do not divide {e} experts (at most "
                         f"{native.route_max_groups})")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups: expected 1 to {groups}, got {top_groups}")
    if not 1 <= k <= min(native.route_max_k, e // groups * top_groups):
        raise ValueError(f"k: expected 1 to {min(native.route_max_k, e // groups * top_groups)}, "
                         f"got {k}")
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score: expected 'softmax' or 'sigmoid', got {score!r}")
    scale = float(scale)
    if not _F32.tiny <= scale <= _F32.max:
        raise ValueError(f"scale: expected a positive float32 number, got {scale}")
    if bias is not None:
        _same("bias", bias, logits, (e,), torch.float32)
        bias = bias.detach().contiguous()
    z = logits if logits.is_cuda else logits.float()
    return _Route.apply(z, bias, k, groups, top_groups, score == "sigmoid", bool(renormalize),
                        scale)
