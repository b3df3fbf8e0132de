"""Plain 64-bit forms of the 8-bit operators, on the CPU (test infrastructure)."""
import math

import torch


def quantize(y):
    """(codes, scale) of float64 rows; a row that is not finite: codes 0, scale NaN."""
    y = y.double()
    top = y.abs().amax(-1) if y.shape[-1] else torch.zeros(y.shape[:-1], dtype=torch.float64)
    bad = ~torch.isfinite(y).all(-1)
    scale = torch.where(bad, torch.full_like(top, math.nan), top / 127)
    step = torch.where(bad | (top == 0), torch.ones_like(top), top / 127)
    codes = torch.where((bad | (top == 0))[..., None], torch.zeros_like(y), torch.round(y / step[..., None]))
    return codes, scale


def rmsnorm(x, w, eps, delta=None):
    """(residual, normed rows) in float64"""
    r = x.double() + (0 if delta is None else delta.double())
    return r, r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * w.double()


def swiglu(x, block):
    x = x.double()
    p = x.reshape(x.shape[0], -1, 2, block)
    g, u = p[:, :, 0], p[:, :, 1]
    return (g / (1 + torch.exp(-g)) * u).reshape(x.shape[0], -1)


def gemm(a, sa, w, sw, bias=None):
    c = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    return c if bias is None else c + bias.double()


def spans(starts, lens, rows):
    """(sequence, row of the arrays, position) of every row that a sequence owns"""
    for b in range(len(lens)):
        first, last = starts[b], min(starts[b + 1], rows)
        for t in range(first, last):
            yield b, t, lens[b] - (last - first) + (t - first)


def attention(q, k, v, slots, starts, lens, causal, scale):
    """q [rows][heads][dim]; k, v [slots][kv heads][ctx][dim] as values, float64.  Rows that no sequence owns: NaN."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    per = q.shape[1] // k.shape[1]
    for b, t, pos in spans(starts, lens, q.shape[0]):
        if not 0 <= slots[b] < k.shape[0]:
            out[t] = 0
            continue
        n = max(0, min(k.shape[2], pos + 1 if causal else lens[b]))
        if n == 0:
            out[t] = 0
            continue
        kk, vv = (x[slots[b], :, :n].repeat_interleave(per, 0) for x in (k, v))           # [heads][n][dim]
        s = (kk @ q[t].double()[:, :, None])[..., 0] * scale
        out[t] = (torch.softmax(s, -1)[:, None] @ vv)[:, 0]
    return out
