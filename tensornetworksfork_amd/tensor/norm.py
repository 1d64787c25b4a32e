"""Layer norm and dropout of the rows a model learns from, differentiable (kernels: csrc/ttk_norm.hip).

    rows -> layer_norm -> dropout -> TensorTrainLayer -> logits

`layer_norm(..., p=...)` runs both in one pass over the rows; its backward pass returns the gradients of the rows, the
weight and the bias.  The dropout mask is a function of (seed, offset + element number) and is never stored: the backward
pass recomputes it, and a shard of a data set that passes the element number of its first row as `offset` draws the mask of
the whole set.  `offset` may be an int64 device tensor of one element, read when the kernel runs: a captured graph draws a
new mask on every replay if the graph (or the caller between replays) advances it.  Its value has to stay until the backward
pass has run; changing it in place before that raises, as for any tensor autograd has saved.

Gradients of gradients and forward-mode derivatives (dual tensors, torch.func.jvp) are not defined here (asking for them
raises).  Graphs: capture the forward pass together with its
backward pass, while no eager graph of the same leaves is alive (autograd adds up a leaf's gradient on the stream its first
graph was recorded on, which a capture on another stream does not survive).  The modules count their masks on the host: a
captured pass replays one mask (pass an `offset` tensor to `layer_norm` / `dropout` for new ones), and a pass that is computed
twice, as by checkpointing, draws two; `offset` is a plain attribute, to be kept by whoever resumes a training run.
"""
import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["layer_norm", "dropout", "LayerNorm", "Dropout"]


def _rows(t):
    """t, or a contiguous copy where its axes do not fold into rows of one distance."""
    if not isinstance(t, torch.Tensor) or t.ndim == 0 or t.is_contiguous():
        return t
    try:
        ops.rows_view(t)
    except ops._lib.TTKError:
        return t.contiguous()
    return t


def _once(backward):
    """`backward` without gradients of its own (asking for them raises); the guard costs more than the whole check here, so
    it is only put on where autograd records the backward pass."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _recorded(*ts):
    """Whether autograd has to remember the call.  Dual tensors, which require no gradient by themselves, are refused."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ops._lib.TTKError("layer norm and dropout have no forward-mode derivatives")
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in ts)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, p, seed, offset):
        y, mean, rstd = ops.layer_norm(x, weight, bias, eps, p, seed, offset)
        off = offset if isinstance(offset, torch.Tensor) else None
        ctx.save_for_backward(x, weight, mean, rstd, off)
        ctx.wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        ctx.drop = (float(p), int(seed), 0 if off is not None else int(offset))
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, mean, rstd, off = ctx.saved_tensors
        drop = (*ctx.drop, None if off is None else off.data_ptr())
        grads = ops.norm_gradients(_rows(dy), x, mean, rstd, weight, drop, ctx.needs_input_grad, ctx.wdtype)
        return (*grads, None, None, None, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        off = offset if isinstance(offset, torch.Tensor) else None
        ctx.save_for_backward(off)
        ctx.drop = (p, seed, None if off is not None else offset)
        return ops.dropout(x, p, seed, offset)

    @staticmethod
    @_once
    def backward(ctx, dy):
        off, = ctx.saved_tensors
        p, seed, offset = ctx.drop
        return ops.dropout(dy.contiguous(), p, seed, offset if off is None else off), None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, p=0.0, seed=0, offset=0):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, followed by dropout with probability p."""
    x = _rows(x)
    if not _recorded(x, weight, bias):
        return ops.layer_norm(x, weight, bias, eps, p, seed, offset, stats=False)[0]
    return _LayerNorm.apply(x, weight, bias, eps, p, seed, offset)


def dropout(x, p, seed, offset=0):
    """Each element kept with probability 1 - p and divided by it; the mask is a function of (seed, offset + element)."""
    x = x.contiguous() if isinstance(x, torch.Tensor) else x
    if not _recorded(x):
        return ops.dropout(x, p, seed, offset)
    return _Dropout.apply(x, p, seed, offset)


class LayerNorm(nn.Module):
    """Layer norm over the last axis of `cols` columns, with an optional learnable weight and bias, and dropout (probability
    p, while training) as its epilogue.  Every training pass draws the next elements of the mask that `seed` names."""

    def __init__(self, cols, eps=1e-5, affine=True, p=0.0, seed=0, device=None, dtype=None):
        super().__init__()
        self.cols, self.eps, self.p, self.seed = int(cols), float(eps), float(p), int(seed)
        self.offset = 0
        if affine:
            self.weight = nn.Parameter(torch.ones(self.cols, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(self.cols, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x):
        if x.ndim == 0 or x.shape[-1] != self.cols:
            raise ops._lib.TTKError(f"LayerNorm: expected {self.cols} columns, got shape {tuple(x.shape)}")
        if not self.training or self.p == 0.0:
            return layer_norm(x, self.weight, self.bias, self.eps)
        offset, self.offset = self.offset, self.offset + x.numel()
        return layer_norm(x, self.weight, self.bias, self.eps, self.p, self.seed, offset)

    def extra_repr(self):
        return f"{self.cols}, eps={self.eps}, affine={self.weight is not None}, p={self.p}"


class Dropout(nn.Module):
    """Dropout while training; every training pass draws the next elements of the mask that `seed` names."""

    def __init__(self, p, seed=0):
        super().__init__()
        self.p, self.seed, self.offset = float(p), int(seed), 0

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        offset, self.offset = self.offset, self.offset + x.numel()
        return dropout(x, self.p, self.seed, offset)

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"
