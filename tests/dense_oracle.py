"""The layer's dense operators from their definitions, in 64 bits on the CPU: test infrastructure."""
import math

import torch


def layer_norm(x, weight, bias, eps, residual=None):
    """(out, mean, rstd)"""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    y = (x - mean) * rstd
    y = y * (1 if weight is None else weight.double()) + (0 if bias is None else bias.double())
    return (y if residual is None else y + residual.double()), mean[:, 0], rstd[:, 0]


def layer_norm_backward(dout, x, weight, stats):
    dy, x, stats = dout.double(), x.double(), stats.double()
    xh = (x - stats[:, :1]) * stats[:, 1:]
    g = dy if weight is None else dy * weight.double()
    dx = stats[:, 1:] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    """x [batch, tokens, heads, head_dim], positions [batch, tokens, axes]"""
    x = x.double()
    pairs = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = positions.double()[..., axis] * inv_freq.double() * (-1 if inverse else 1)
    cos, sin = angle.cos().unsqueeze(2), angle.sin().unsqueeze(2)
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :pairs], turned[..., pairs:])
    c, d = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([y, rest], -1)


def visible(queries, keys, length, first, window, sinks):
    """[queries, keys] truth values"""
    at = torch.arange(queries)[:, None] + int(first)
    j = torch.arange(keys)[None, :]
    seen = (j < min(max(int(length), 0), keys)).expand(queries, keys).clone()
    if window[0] >= 0:
        seen &= (j >= at - window[0]) | (j < sinks)
    if window[1] >= 0:
        seen &= j <= at + window[1]
    return seen


def attention(q, k, v, scale=None, window=(-1, -1), sinks=0, lengths=None, first=None):
    B, Q, H, D = q.shape
    K, G = k.shape[1:3]
    out = torch.zeros(B, Q, H, D, dtype=torch.float64)
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        seen = visible(Q, K, K if lengths is None else lengths[b], 0 if first is None else first[b], window, sinks)
        some = seen.any(1)
        for h in range(H):
            g = h // (H // G)
            s = (q[b, :, h].double() @ k[b, :, g].double().T) * scale
            s = torch.where(seen, s, -math.inf)
            w = torch.softmax(s[some], 1)
            out[b, some, h] = torch.where(w > 0, w, 0) @ torch.where(seen.any(0)[:, None], v[b, :, g].double(), 0)
    return out


def close(got, want, dtype, steps=1.0, floor=0.0):
    """|got - want| within `steps` roundings of `dtype` at the value, and `floor` (what fp32 arithmetic on the way may leave)."""
    got, want = got.double().cpu(), want.double().cpu()
    off = (got - want).abs()
    allowed = steps * torch.finfo(dtype).eps / 2 * want.abs() + floor
    bad = ~(off <= allowed)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off - allowed).max()):.3g} beyond {float(allowed.max()):.3g}"
