"""The norm and position rotation of query and key heads restated plainly (torch, any device), step by step as the kernels define
them, and in 64 bits throughout."""
import torch


def turned(x, positions, freq, layout, factor, weight, eps):
    """[rows, heads, dim] -> the same shape and type. freq fp64 [rot / 2] or None, eps None: no norm. The squares' mean, its inverse
    root, angles, cosines and sines in 64 bits, each rounded to fp32 once; the rest single fp32 operations; one rounding at the end."""
    y = x.float()
    if eps is not None:
        y = y * (1.0 / torch.sqrt(y.double().square().mean(-1, keepdim=True) + eps)).float()
        if weight is not None:
            y = y * weight.float()
    if freq is None:
        return y.to(x.dtype)
    a = positions.double()[:, None, None] * freq
    c, s = (torch.cos(a) * factor).float(), (torch.sin(a) * factor).float()
    n = freq.shape[0]
    u, w, rest = _pairs(y, n, layout)
    return _back(u * c - w * s, w * c + u * s, rest, layout).to(x.dtype)


def turned64(x, positions, freq, layout, factor, weight, eps):
    """The same in float64, unrounded."""
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    if freq is None:
        return y
    a = positions.double()[:, None, None] * freq
    u, w, rest = _pairs(y, freq.shape[0], layout)
    c, s = torch.cos(a) * factor, torch.sin(a) * factor
    return _back(u * c - w * s, w * c + u * s, rest, layout)


def _pairs(y, n, layout):
    if layout == "half":
        return y[..., :n], y[..., n:2 * n], y[..., 2 * n:]
    return y[..., 0:2 * n:2], y[..., 1:2 * n:2], y[..., 2 * n:]


def _back(u, w, rest, layout):
    if layout == "half":
        return torch.cat([u, w, rest], -1)
    return torch.cat([torch.stack([u, w], -1).flatten(-2), rest], -1)
