"""Plain 64-bit restatements of layer norm, dropout and label sampling (NumPy / torch on the CPU), used by the tests."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24          # half a step of float32, relative
U64 = 2.0 ** -53


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of two subnormals: the absolute part of a rounding near zero."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def unit(dtype):
    """Half a step of the arithmetic the rows' kernels compute in."""
    return U64 if dtype == torch.float64 else U32


def philox(counter_lo, counter_hi, seed):
    """Philox4x32-10 words (..., 4) for counters (lo, hi, 0, 0)."""
    m32 = np.uint64(0xFFFFFFFF)
    c = [np.asarray(counter_lo, np.uint64), np.asarray(counter_hi, np.uint64)]
    c += [np.zeros_like(c[0]), np.zeros_like(c[0])]
    k0, k1 = np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k0, p1 & m32, (p0 >> np.uint64(32)) ^ c[3] ^ k1, p0 & m32]
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & m32, (k1 + np.uint64(0xBB67AE85)) & m32
    return np.stack(c, axis=-1)


def keep_mask(n, p, seed, offset=0):
    """(n,) bool: element offset + i is kept."""
    if p == 0.0:
        return torch.ones(n, dtype=torch.bool)
    if p == 1.0:
        return torch.zeros(n, dtype=torch.bool)
    e = np.arange(n, dtype=np.uint64) + np.uint64(offset)
    b = e >> np.uint64(2)
    first = b[0] if n else np.uint64(0)
    nb = int(b[-1] - first) + 1 if n else 0
    blocks = first + np.arange(nb, dtype=np.uint64)
    words = philox(blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), seed).reshape(-1)
    at = (e - first * np.uint64(4)).astype(np.int64)
    t = min(int(round(p * 2.0 ** 32)), 2 ** 32 - 1)
    return torch.from_numpy(words[at] >= np.uint64(t))


def dropout(x, p, seed, offset=0):
    x = x.double()
    if p == 1.0:
        return torch.zeros_like(x)
    m = keep_mask(x.numel(), p, seed, offset).reshape(x.shape)
    return torch.where(m, x / (1.0 - p), torch.zeros_like(x))


def norm_forward(x, w=None, b=None, eps=1e-5):
    x = x.double()
    mean = x.mean(dim=-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(dim=-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h if w is None else h * w.double()
    return y if b is None else y + b.double(), mean, rstd, h


def norm_backward(dy, x, mean, rstd, w=None):
    """mean / rstd (..., 1) as given; dy already masked."""
    g, x = dy.double(), x.double()
    h = (x - mean) * rstd
    a = g if w is None else g * w.double()
    dx = rstd * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    lead = tuple(range(g.ndim - 1))
    return dx, (g * h).sum(dim=lead), g.sum(dim=lead), h, a


def sample_row(z, u, T=1.0, k=0, P=1.0, M=0.0):
    """(label, margin): the drawn index, and how far the decisions of the row are from a border, relative to the sums they
    compare (a kernel that sums in another order may decide otherwise only below its rounding)."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, np.float64))
    V = z.size
    m = z.max()
    if m == -np.inf:
        return -1, 1.0
    if not T > 0:
        return int(np.argmax(z)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == m, 1.0, np.exp((z - m) / T))
    order = np.argsort(-z, kind="stable")
    margin = 1.0
    if 0 < k < V:
        order = order[:k]
    if P < 1.0:
        ws = w[order]
        before = np.concatenate(([0.0], np.cumsum(ws)[:-1]))
        total = math.fsum(ws)
        keep = before < max(P, 0.0) * total
        keep[0] = True
        if P > 0 and before.size > 1:      # (the first is kept whatever the sums are)
            margin = min(margin, np.min(np.abs(before[1:] - P * total)) / total)
        order = order[keep]
    if M > 0:
        margin = min(margin, np.min(np.abs(w[order] - min(M, 1.0)) + (w[order] == 1.0)))
        order = order[w[order] >= min(M, 1.0)]
    sel = np.sort(order)
    c = np.cumsum(w[sel])
    t = min(max(u, 0.0), 1.0) * c[-1]
    live = w[sel] > 0
    if u > 0:
        margin = min(margin, np.min(np.abs(c[live] - t)) / c[-1])
    hit = np.flatnonzero((c > t) & live)
    at = hit[0] if hit.size else np.flatnonzero(live)[-1]
    return int(sel[at]), margin
