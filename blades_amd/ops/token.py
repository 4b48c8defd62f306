"""Training operators of token models (text and image transformers).

* :func:`layer_norm` — forward and backward, the parameters' gradients summed
  per client;
* :func:`linear_cross_entropy` — cross entropy of a linear head over a large
  vocabulary, without keeping its logits;
* :func:`gelu_act8`, :func:`linear_act8` — GELU and linear layers that keep
  their input in 8 bits for the backward pass.

float32 and bfloat16.  GPU tensors run the HIP kernels of ``csrc/`` (and
refuse to run without them) through dispatcher ops of the extension; CPU
tensors run the plain forms of :mod:`torch_ref` under the autograd functions
below, which have the same rules.  Every operator runs under
``torch.func.grad`` and ``torch.func.vmap`` in either nesting: a vmapped call is ONE launch over all
clients ("groups" below), with shared or per-client parameters, and
``vmap(grad(...))`` gets the parameters' gradients per client from the
kernels.  Vmaps nest as long as the inner one's clients share their parameters
and no gradient is taken per client at both levels; a loss that is summed or
averaged per client needs the parameters shared at both.  Other nestings are
refused.  The operators' gradients are not differentiable
again.

Under ``torch.autocast`` norms run in float32, products in bfloat16 where that
is autocast's type, and in float32 where it is float16.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch._C import _functorch
from torch.autograd import Function

from . import torch_ref as _ref

Tensor = torch.Tensor

_DTYPES = (torch.float32, torch.bfloat16)
_REDUCTIONS = ("none", "sum", "mean")


def _extension(x: Tensor):
    """The HIP extension, whose ops bring their own autograd and vmap rules,
    where ``x`` has to run on it; else None."""
    from blades_amd import ops

    return ops._route(x)


# ------------------------------------------------------------------ checks

def _check_input(name: str, x: Tensor, min_dim: int = 1) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {x.dtype}")
    if x.dim() < min_dim:
        raise ValueError(f"{name} needs at least {min_dim} dimension(s), got "
                         f"shape {tuple(x.shape)}")
    if x.shape[-1] == 0:
        raise ValueError(f"{name} has an empty last axis")


def _check_param(name: str, p: Optional[Tensor], x: Tensor, shape) -> None:
    if p is None:
        return
    if not isinstance(p, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(p).__name__}")
    if p.dtype != x.dtype:
        raise TypeError(f"{name} must have x's type {x.dtype}, got {p.dtype}")
    if p.device != x.device:
        raise ValueError(f"{name} must be on {x.device}, got {p.device}")
    if tuple(p.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got "
                         f"{tuple(p.shape)}")


def _autocast(x, kind: str, *rest):
    """``x`` and the parameters in the type that autocast runs the operator
    in, as torch has it: ``"norm"`` in float32, ``"product"`` in autocast's
    type, ``"any"`` in its input's.  float32 takes float16's place.  Outside
    of autocast they stay as they are."""
    device = x.device.type if isinstance(x, torch.Tensor) else ""
    if device not in ("cpu", "cuda") or not torch.is_autocast_enabled(device):
        return (x, *rest)
    want = torch.float32
    if kind == "any" and x.dtype != torch.float16:
        want = x.dtype
    elif kind == "product" and \
            torch.get_autocast_dtype(device) == torch.bfloat16:
        want = torch.bfloat16

    def cast(t):
        if isinstance(t, torch.Tensor) and t.dtype in (*_DTYPES,
                                                       torch.float16):
            return t.to(want)
        return t
    return tuple(cast(t) for t in (x, *rest))


# ------------------------------------------------------------- vmap helpers

def _batched(t, dim, size: int):
    """``t`` with its client axis first; a tensor without one is repeated."""
    if t is None:
        return None
    return t.movedim(dim, 0) if dim is not None else t.expand(size, *t.shape)


def _param_batched(t, dim):
    """Client axis first, or left shared."""
    return t if t is None or dim is None else t.movedim(dim, 0)


def _shared(p: Optional[Tensor], groups: int, dims: int) -> bool:
    """Of a call with groups: whether a parameter of ``dims`` dimensions is
    shared, so that its gradients per client have to be summed."""
    return bool(groups) and p is not None and p.dim() == dims


def _summed(grad, shared: bool):
    return grad.sum(0) if shared else grad


def _refuse_nested(groups: int, op: str) -> None:
    if groups:
        raise NotImplementedError(
            f"{op}: a vmap over clients inside another vmap is not supported")


def _groups3(t: Tensor, groups: int) -> Tensor:
    """[groups or 1, rows, last] contiguous."""
    g, last = max(groups, 1), t.shape[-1]
    rows = t.numel() // (g * last) if last else 0
    return t.reshape(g, rows, last).contiguous()


def _groups2(t: Tensor, groups: int) -> Tensor:
    """[groups or 1, rows] contiguous."""
    g = max(groups, 1)
    return t.reshape(g, t.numel() // g).contiguous()


class _NoSecond(Function):
    """Base of the gradient functions."""

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(
            "the gradients of blades_amd.ops token operators are not "
            "differentiable again")


# -------------------------------------------------------------- layer norm

class _NormGrad(_NoSecond):
    @staticmethod
    def forward(dy, x, w, mean, rstd, groups, params):
        g = max(groups, 1)
        dx, dw, db = _ref.norm_backward(
            _groups3(dy, groups), _groups3(x, groups),
            _groups2(mean, groups),
            _groups2(rstd, groups),
            None if w is None else w.contiguous(), params)
        if not groups and params:
            dw, db = dw[0], db[0]
        return dx.view(x.shape), dw, db

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, dy, x, w, mean, rstd, groups, params):
        _refuse_nested(groups, "layer_norm")
        n = info.batch_size
        out = _NormGrad.apply(
            _batched(dy, in_dims[0], n), _batched(x, in_dims[1], n),
            _param_batched(w, in_dims[2]), _batched(mean, in_dims[3], n),
            _batched(rstd, in_dims[4], n), n, params)
        per = 0 if params else None
        return out, (0, per, per)


class _Norm(Function):
    # groups: 0, or the number of clients on x's first axis; each of w and b
    # is then per client or shared

    @staticmethod
    def forward(x, w, b, eps, groups):
        y, mean, rstd = _ref.norm_forward(
            _groups3(x, groups), None if w is None else w.contiguous(),
            None if b is None else b.contiguous(), eps)
        lead = x.shape[:-1]
        return y.view(x.shape), mean.view(lead), rstd.view(lead)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, b, _, groups = inputs
        _, mean, rstd = output
        ctx.mark_non_differentiable(mean, rstd)
        ctx.save_for_backward(x, w, mean, rstd)
        ctx.groups = groups
        ctx.has_b = b is not None
        ctx.shared = _shared(w, groups, 1), _shared(b, groups, 1)

    @staticmethod
    def backward(ctx, dy, _mean, _rstd):
        x, w, mean, rstd = ctx.saved_tensors
        need_w = w is not None and ctx.needs_input_grad[1]
        need_b = ctx.has_b and ctx.needs_input_grad[2]
        dx, dw, db = _NormGrad.apply(dy, x, w, mean, rstd, ctx.groups,
                                     need_w or need_b)
        return (dx, _summed(dw, ctx.shared[0]) if need_w else None,
                _summed(db, ctx.shared[1]) if need_b else None, None, None)

    @staticmethod
    def vmap(info, in_dims, x, w, b, eps, groups):
        _refuse_nested(groups, "layer_norm")
        n = info.batch_size
        x = _batched(x, in_dims[0], n)
        if in_dims[1] is not None or in_dims[2] is not None:
            w, b, groups = (_param_batched(w, in_dims[1]),
                            _param_batched(b, in_dims[2]), n)
        return _Norm.apply(x, w, b, eps, groups), (0, 0, 0)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None,
               bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """Normalise ``x`` [..., dim] over its last axis, then scale and shift.

    ``weight``, ``bias``: [dim] in x's type, or None.  Statistics and the
    sums of the gradients are 32-bit; each output is rounded once.
    """
    x, weight, bias = _autocast(x, "norm", weight, bias)
    _check_input("x", x)
    _check_param("weight", weight, x, x.shape[-1:])
    _check_param("bias", bias, x, x.shape[-1:])
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    ext = _extension(x)
    if ext is not None:
        return ext.layer_norm(x, weight, bias, float(eps))
    return _Norm.apply(x, weight, bias, float(eps), 0)[0]


# -------------------------------------------------------- head cross entropy

class _HeadLossGrad(_NoSecond):
    @staticmethod
    def forward(grad, x, w, b, target, lse, count, ignore, reduction, groups,
                wants):
        g = max(groups, 1)
        dx, dw, db = _ref.loss_backward(
            _groups2(grad.float(), groups), _groups3(x, groups),
            w.contiguous(), _groups2(target, groups),
            None if b is None else b.contiguous(),
            lse.reshape(g, lse.numel() // (2 * g), 2).contiguous(),
            count.reshape(g).contiguous(),
            ignore, reduction, *wants)
        if not groups:
            dw = dw[0] if wants[1] else dw
            db = db[0] if wants[2] else db
        return (dx.view(x.shape) if wants[0] else dx), dw, db

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, grad, x, w, b, target, lse, count, ignore,
             reduction, groups, wants):
        _refuse_nested(groups, "linear_cross_entropy")
        n = info.batch_size
        out = _HeadLossGrad.apply(
            _batched(grad, in_dims[0], n), _batched(x, in_dims[1], n),
            _param_batched(w, in_dims[2]), _param_batched(b, in_dims[3]),
            _batched(target, in_dims[4], n), _batched(lse, in_dims[5], n),
            _batched(count, in_dims[6], n), ignore, reduction, n, wants)
        return out, tuple(0 if want else None for want in wants)


class _HeadLoss(Function):
    # groups: 0, or the number of clients on the first axis of x and target;
    # w and b are then shared or per client

    @staticmethod
    def forward(x, w, b, target, ignore, reduction, groups):
        g = max(groups, 1)
        loss, lse, count = _ref.loss_forward(
            _groups3(x, groups), w.contiguous(),
            _groups2(target, groups),
            None if b is None else b.contiguous(), ignore, reduction)
        if reduction == 0:
            loss = loss.view(target.shape)
        elif not groups:
            loss = loss[0]
        return (loss, lse.view(*target.shape, 2),
                count if groups else count[0])

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, b, target, ignore, reduction, groups = inputs
        _, lse, count = output
        ctx.mark_non_differentiable(lse, count)
        ctx.save_for_backward(x, w, b, target, lse, count)
        ctx.settings = (ignore, reduction, groups)

    @staticmethod
    def backward(ctx, grad, _lse, _count):
        x, w, b, target, lse, count = ctx.saved_tensors
        ignore, reduction, groups = ctx.settings
        wants = (ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                 b is not None and ctx.needs_input_grad[2])
        shared_w, shared_b = _shared(w, groups, 2), _shared(b, groups, 1)
        if shared_w and (shared_b or b is None):
            # shared parameters: one sum over all clients' rows, each row
            # with its client's share of the upstream gradient
            if reduction == 2:
                grad = grad / count
            if reduction != 0:
                ones = (1,) * (target.dim() - 1)
                grad = grad.view(-1, *ones).expand(target.shape)
            reduction, groups, count = 0, 0, count[:1]
            shared_w = shared_b = False
        dx, dw, db = _HeadLossGrad.apply(grad, x, w, b, target, lse, count,
                                         ignore, reduction, groups, wants)
        return (dx if wants[0] else None,
                _summed(dw, shared_w) if wants[1] else None,
                _summed(db, shared_b) if wants[2] else None, None, None, None,
                None)

    @staticmethod
    def vmap(info, in_dims, x, w, b, target, ignore, reduction, groups):
        n = info.batch_size
        x = _batched(x, in_dims[0], n)
        target = _batched(target, in_dims[3], n)
        own = in_dims[1] is not None or in_dims[2] is not None
        if not own and not groups and reduction == 0:
            # rows of shared parameters: no client is told from another
            return (_HeadLoss.apply(x, w, b, target, ignore, reduction, 0),
                    (0, 0, None))
        if not own and groups and w.dim() == 2 and (b is None or b.dim() == 1):
            # clients of an inner vmap who share the parameters with these:
            # as many groups as pairs
            out = _HeadLoss.apply(x.flatten(0, 1), w, b, target.flatten(0, 1),
                                  ignore, reduction, n * groups)
            return tuple(t.unflatten(0, (n, groups)) for t in out), (0, 0, 0)
        _refuse_nested(groups, "linear_cross_entropy")
        w, b = _param_batched(w, in_dims[1]), _param_batched(b, in_dims[2])
        return (_HeadLoss.apply(x, w, b, target, ignore, reduction, n),
                (0, 0, 0))


def linear_cross_entropy(x: Tensor, weight: Tensor, target: Tensor,
                         bias: Optional[Tensor] = None,
                         ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Cross entropy of the logits ``x @ weight.T + bias`` with ``target``,
    in float32, computed in tiles: the [rows, vocab] logits are never stored.
    The backward pass computes them again, a piece of the vocabulary at a
    time (at most 256 MiB of their gradient exists at once, or 512 words); it
    takes fewer than 2**22 rows a client, or of all clients together where
    they share the parameters and the gradient is that of the whole vmap.

    bfloat16 inputs are multiplied as they are and summed in float32.  The
    logits' gradient is rounded to bfloat16 before the products that give
    ``x``'s and ``weight``'s, which adds less than a hundredth to the error
    that their own rounding has.

    ``x``: [..., dim]; ``weight``: [vocab, dim]; ``bias``: [vocab] or None;
    ``target``: int64, x's leading shape.  Rows whose target is
    ``ignore_index`` have loss 0 and no gradient.  ``reduction``: ``"none"``
    (target's shape), ``"sum"``, or ``"mean"`` over the rows that count (NaN
    where none does, as torch has it; their gradient is zero).

    In float32 a value of ``x`` or ``weight`` that is not finite makes the
    results it enters NaN; in bfloat16 they are not finite.  An ignored row
    enters the weight's gradient with a factor of zero, so it has to be finite
    for that.

    A target outside the vocabulary cannot raise without stopping the GPU's
    stream: its row's loss, and every gradient it enters, is NaN.  ``bias``
    may hold -inf for words that are switched off.
    """
    x, weight, bias = _autocast(x, "product", weight, bias)
    _check_input("x", x)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be a [vocab, dim] tensor")
    if weight.shape[0] == 0:
        raise ValueError("weight has no rows")
    _check_param("weight", weight, x, (weight.shape[0], x.shape[-1]))
    _check_param("bias", bias, x, weight.shape[:1])
    if not isinstance(target, torch.Tensor) or target.dtype != torch.int64:
        raise TypeError("target must be an int64 tensor")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target must have shape {tuple(x.shape[:-1])}, got "
                         f"{tuple(target.shape)}")
    if target.device != x.device:
        raise ValueError(f"target must be on {x.device}, got {target.device}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got "
                         f"{reduction!r}")
    ext = _extension(x)
    if ext is not None:
        return ext.linear_cross_entropy(x, weight, target, bias,
                                        int(ignore_index),
                                        _REDUCTIONS.index(reduction))
    return _HeadLoss.apply(x, weight, bias, target, int(ignore_index),
                           _REDUCTIONS.index(reduction), 0)[0]


# ------------------------------------------------- 8-bit activation storage

class _GeluGrad(_NoSecond):
    @staticmethod
    def forward(dy, q, e, tie):
        return _ref.gelu_backward(dy.contiguous(), q.contiguous(),
                                  e.contiguous())

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, dy, q, e, tie):
        n = info.batch_size
        return _GeluGrad.apply(*(_batched(t, d, n) for t, d in
                                 zip((dy, q, e), in_dims)), tie), 0


class _Gelu8(Function):
    # The 8-bit values carry no history; `tie`, empty, does, so that their
    # gradient function sees that it depends on x.

    @staticmethod
    def forward(x, keep):
        return (*_ref.gelu_forward(x.contiguous(), keep), x.new_empty(0))

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, q, e, tie = output
        ctx.mark_non_differentiable(q, e)
        ctx.save_for_backward(q, e, tie)

    @staticmethod
    def backward(ctx, dy, _q, _e, _tie):
        return _GeluGrad.apply(dy, *ctx.saved_tensors), None

    @staticmethod
    def vmap(info, in_dims, x, keep):
        per = 0 if keep else None
        return (_Gelu8.apply(_batched(x, in_dims[0], info.batch_size), keep),
                (0, per, per, None))


def gelu_act8(x: Tensor) -> Tensor:
    """GELU, ``x * Phi(x)``, that keeps ``x`` in 8 bits for its gradient.

    Along the last axis every 128 values share the least power of two
    ``2**e`` (e >= -126) with ``max|x| <= 127 * 2**e`` and are held as int8:
    1.008 bytes a value.  The gradient is the formula's at the values held,
    which differ from ``x`` by at most ``2**(e-1)`` (what would round to
    2**128 is held as 63 * 2**122); a block of 128 that
    holds an infinity or NaN has gradient NaN.  The output comes from ``x``
    itself; in float32 its relative error is about 2**-22 at most for
    ``|x| < 1`` and grows with ``x**2`` in the negative tail.
    """
    x, = _autocast(x, "any")
    _check_input("x", x)
    ext = _extension(x)
    if ext is not None:
        return ext.gelu_act8(x)
    return _Gelu8.apply(x, _tracks(x))[0]


def _tracks(t: Tensor) -> bool:
    """Whether a gradient of ``t`` can be asked for, at any level of the
    torch.func transforms around the call."""
    if not torch.is_grad_enabled():
        return False
    while not t.requires_grad:
        if not _functorch.is_functorch_wrapped_tensor(t):
            return False
        t = _functorch.get_unwrapped(t)
    return True


def _product(x: Tensor, w: Tensor, groups: int, transpose: bool, b=None):
    """x @ w.T + b (or x @ w) with shared or per-client w."""
    x3 = _groups3(x, groups)
    y = (_ref.linear_forward(x3, w, b) if transpose
         else _ref.linear_grad_input(x3, w))
    return y.reshape(*x.shape[:-1], y.shape[-1])


class _LinearGrad(_NoSecond):
    @staticmethod
    def forward(dy, w, q, e, tie, groups, wants):
        g = max(groups, 1)
        dx = (_product(dy, w, groups, False) if wants[0]
              else dy.new_empty(0))
        dw = db = dy.new_empty(0)
        if wants[1] or wants[2]:
            dy3 = _groups3(dy, groups)
            if wants[1]:
                rows = dy3.shape[1]
                dw = _ref.linear_grad_weight(
                    dy3, q.reshape(g, rows, q.shape[-1]).contiguous(),
                    e.reshape(g, rows, e.shape[-1]).contiguous())
                dw = dw if groups else dw[0]
            if wants[2]:
                db = _ref.colsum(dy3)
                db = db if groups else db[0]
        return dx, dw, db

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, dy, w, q, e, tie, groups, wants):
        _refuse_nested(groups, "linear_act8")
        n = info.batch_size
        q, e = ((_batched(q, in_dims[2], n), _batched(e, in_dims[3], n))
                if wants[1] else (q, e))
        out = _LinearGrad.apply(_batched(dy, in_dims[0], n),
                                _param_batched(w, in_dims[1]), q, e, tie, n,
                                wants)
        return out, tuple(0 if want else None for want in wants)


class _Linear8(Function):
    # groups: as for _Norm; tie: as for _Gelu8

    @staticmethod
    def forward(x, w, b, keep, groups):
        y = _product(x, w, groups, True, b)
        if keep:
            q, e = _ref.act8_pack(x.contiguous())
        else:
            q = e = x.new_empty(0, dtype=torch.uint8)
            e = e.clone()
        return y, q, e, x.new_empty(0)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, w, b, _, groups = inputs
        _, q, e, tie = output
        ctx.mark_non_differentiable(q, e)
        ctx.save_for_backward(w, q, e, tie)
        ctx.groups = groups
        ctx.has_b = b is not None
        ctx.shared = _shared(w, groups, 2), _shared(b, groups, 1)

    @staticmethod
    def backward(ctx, dy, _q, _e, _tie):
        w, q, e, tie = ctx.saved_tensors
        wants = (ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                 ctx.has_b and ctx.needs_input_grad[2])
        shared_w, shared_b = ctx.shared
        # a shared weight's gradient is one product over all clients' rows
        apart = shared_w and not shared_b and wants[2]
        # only the weight's gradient depends on the layer's input
        dx, dw, db = _LinearGrad.apply(
            dy, w, q, e, tie if wants[1] else None,
            0 if shared_w else ctx.groups,
            (wants[0], wants[1], wants[2] and not apart))
        if apart:
            db = _LinearGrad.apply(dy, w, q, e, None, ctx.groups,
                                   (False, False, True))[2]
        return (dx if wants[0] else None, dw if wants[1] else None,
                _summed(db, shared_b and not shared_w) if wants[2] else None,
                None, None)

    @staticmethod
    def vmap(info, in_dims, x, w, b, keep, groups):
        _refuse_nested(groups, "linear_act8")
        n = info.batch_size
        x = _batched(x, in_dims[0], n)
        if in_dims[1] is not None or in_dims[2] is not None:
            w, b, groups = (_param_batched(w, in_dims[1]),
                            _param_batched(b, in_dims[2]), n)
        per = 0 if keep else None
        return _Linear8.apply(x, w, b, keep, groups), (0, per, per, None)


def linear_act8(x: Tensor, weight: Tensor,
                bias: Optional[Tensor] = None) -> Tensor:
    """``x @ weight.T + bias`` that keeps ``x`` [..., in] in 8 bits (see
    :func:`gelu_act8`) for the weight's gradient, ``dy.T @ x8``; the values
    held are used as they are in that product.  ``weight``: [out, in];
    ``bias``: [out] or None.

    In float32 a value that is not finite makes the results it enters NaN,
    and magnitudes below 2**-110 lose low bits.  One in ``x`` makes the
    weight's gradient NaN in all the columns of its block of 128, in either
    type.  ``in`` is below 2**22, and for a gradient ``out`` too.
    """
    x, weight, bias = _autocast(x, "product", weight, bias)
    _check_input("x", x)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be an [out, in] tensor")
    if weight.shape[0] == 0:
        raise ValueError("weight has no rows")
    _check_param("weight", weight, x, (weight.shape[0], x.shape[-1]))
    _check_param("bias", bias, x, weight.shape[:1])
    ext = _extension(x)
    if ext is not None:
        return ext.linear_act8(x, weight, bias)
    return _Linear8.apply(x, weight, bias, _tracks(weight), 0)[0]


__all__ = ["layer_norm", "linear_cross_entropy", "gelu_act8", "linear_act8"]
