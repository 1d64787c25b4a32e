"""Gradient of a tensor train with respect to its inputs, so that what stands in front of it (layer norm, dropout, any
torch module) can be trained through it.

Output y[s,c] = sum L[s,c,l] core[l,p,r] G[s,p] R[s,r] is linear in every site's feature vector G, so with the output's
gradient g
    dG[s,p] = sum_{l,r} (sum_c g[s,c] L[s,c,l]) core[l,p,r] R[s,r]
which is an environment step with the core's feature axis in the place of its left bond; a conv or operator column then
applies its feature node once more (one row GEMM).  Environments are the ones the forward pass's engine caches.
"""
import warnings

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops


def _nodes(engine):
    return [n for col in engine.cols for n in (col.A, col.F) if n is not None]


class _Forward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, layer, shared, *xs):
        tn = layer.tensor_network
        x, d = tn._engine.data_for_recorded(xs, shared)
        tn.set_input(x, d)
        y = tn._predict(d)                      # (S, C), in the order of the engine's labels
        ctx.engine, ctx.data, ctx.shared = tn._engine, d, shared
        ctx.nodes = [(n, n.tensor, n.tensor._version) for n in _nodes(tn._engine)]
        ctx.like = [(x.dtype, x.device) for x in xs]
        ctx.save_for_backward(*xs)              # the environments are those of these values
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        eng, d = ctx.engine, ctx.data
        ctx.saved_tensors                       # (raises where an input was changed in place since)
        if any(n.tensor is not t or t._version != v for n, t, v in ctx.nodes):
            raise RuntimeError("a node of the tensor network has changed since the forward pass: its input gradient is gone")
        eng.net._user_guard(d)
        eng.sync(d)
        g = ops.prep(dy.reshape(d.S, -1))
        need = ctx.needs_input_grad[2:]
        grads = [None] * len(need)
        for k, col in enumerate(eng.cols):
            at = 0 if ctx.shared else col.xin
            if not need[at]:
                continue
            dx = _site_gradient(eng, d, k, g)
            grads[at] = dx if grads[at] is None else grads[at] + dx
        grads = [None if t is None else t.to(dtype=dt, device=dev) for t, (dt, dev) in zip(grads, ctx.like)]
        return (None, None, *grads)


def _site_gradient(eng, d, k, g):
    """d (sum_s,c g y) / d x_k in x_k's own shape, float64."""
    L, R = eng.left(d, k), eng.right(d, k)
    core = eng.canonA(k).permute(1, 0, 2).contiguous()          # (p, rl, rr)
    ca, cb, S, p = L.shape[0], R.shape[0], d.S, core.shape[0]
    dG = [ops.env_step_right(R[b].contiguous(), ops.gl(g, L[a].contiguous()), core) for a in range(ca) for b in range(cb)]
    col = eng.cols[k]
    if col.kind == "plain":
        return dG[0]
    F = eng.canonF(k)
    if col.kind == "conv":                                      # F (ca, px, cb):  dx[s,p,x] = sum_ab dG_ab[s,p] F[a,x,b]
        A = torch.stack(dG, dim=2).reshape(S * p, ca * cb)
        B = F.permute(0, 2, 1).reshape(ca * cb, -1).contiguous()
        return ops.gemm_rows(A, B, B.shape[1]).reshape(S, p, -1)
    A = torch.cat(dG, dim=1)                                    # F (ca, u, d, cb):  dx[s,d] = sum_abu dG_ab[s,u] F[a,u,d,b]
    B = F.permute(0, 3, 1, 2).reshape(A.shape[1], -1).contiguous()
    return ops.gemm_rows(A, B, B.shape[1])


def _inputs(x):
    return [t for t in (x if isinstance(x, (list, tuple)) else [x]) if isinstance(t, torch.Tensor)]


def wants_input_gradient(layer, x):
    """Whether a forward pass of `layer` on `x` has to be recorded: grad mode, an input that requires it, a tensor train."""
    from .engine import ChainEngine
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in _inputs(x)):
        return False
    eng = layer.tensor_network._engine
    return type(eng) is ChainEngine and eng.cols is not None


def warn_of_lost_derivatives(x, out):
    """Where a derivative was asked for that the pass does not have: other networks than trains, forward mode."""
    xs = _inputs(x)
    if torch.is_grad_enabled() and any(t.requires_grad for t in xs) and not out.requires_grad:
        warnings.warn("only tensor trains have a gradient with respect to their inputs: the output of this network has none",
                      stacklevel=5)
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in xs) \
            and forward_ad.unpack_dual(out).tangent is None:
        warnings.warn("tensor networks have no forward-mode derivative: the output carries none", stacklevel=5)


def forward(layer, x):
    shared = not isinstance(x, (list, tuple))
    out = layer.tensor_network._shape_output(_Forward.apply(layer, shared, *([x] if shared else x)))
    if layer.labels is not None:
        out.permute_first(*layer.labels)
    return out.tensor
