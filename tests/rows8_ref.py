"""Rows in 8 bits and what is computed from them, from their definitions in float64 on the CPU."""
import math

import torch


def held_values(x):
    """The values that quantize_rows(x) stands for (float64), group by group from the definition."""
    x = x.double().cpu()
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], 32):
        for r in range(x.shape[0]):
            g = x[r, a:a + 32]
            if not bool(torch.isfinite(g).all()):
                out[r, a:a + 32] = math.nan
                continue
            top = float(g.abs().max())
            p = -126
            if top > 0:
                p = math.frexp(top)[1] - 7
                if top / 2.0 ** p >= 127.5:
                    p += 1
                p = min(max(p, -126), 121)
            s = 2.0 ** p
            out[r, a:a + 32] = torch.round(g / s).clamp(-127, 127) * s
    return out


def aggregate(values, ptr, idx, reduce, edge_value=None):
    """(result, sum of the terms' absolute values, degrees) in float64; ids outside the rows count as zeros."""
    n, rows = ptr.shape[0] - 1, values.shape[0]
    ptr, idx = ptr.long().cpu(), idx.long().cpu()[:int(ptr[-1])]
    ok = (idx >= 0) & (idx < rows)
    terms = values[torch.where(ok, idx, torch.zeros_like(idx))] * ok.double().unsqueeze(1)
    if edge_value is not None:
        terms = terms * edge_value.double().cpu()[:idx.shape[0]].unsqueeze(1)
    deg = ptr[1:] - ptr[:-1]
    dst = torch.repeat_interleave(torch.arange(n), deg)
    out = torch.zeros((n, values.shape[1]), dtype=torch.float64).index_add_(0, dst, terms)
    mag = torch.zeros_like(out).index_add_(0, dst, terms.abs())
    if reduce == "mean":
        d = deg.clamp(min=1).double().unsqueeze(1)
        out, mag = out / d, mag / d
    return out, mag, deg


def norm(v, layer, eps, weight=None, bias=None):
    if layer:
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def residual(x, f, gate, scale, post, w2, b2, following, w1, b1, layer, eps):
    """(y, h or None), differentiable, in the type of its arguments."""
    y = x
    if f is not None:
        n = norm(f, layer, eps, w2, b2) if post else f
        if gate is not None:
            g = gate.reshape(-1, 1) if gate.numel() == x.shape[0] and gate.shape != x.shape else gate
            n = n * torch.sigmoid(g)
        y = x + (n if scale is None else scale * n)
    return y, norm(y, layer, eps, w1, b1) if following else None
