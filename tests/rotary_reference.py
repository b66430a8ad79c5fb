"""Norms with rotation in plain 64-bit torch on the CPU: the oracle of the kernels' tests. Their first and
second derivatives come from torch's autograd of this plain form."""

from __future__ import annotations

import torch


def rotate(x, positions, frequencies, interleaved):
    """Rows x (T, N, H) with the pairs of their first columns turned; positions (T,)."""
    if frequencies is None:
        return x
    half = frequencies.shape[0]
    angle = (positions.double()[:, None] * frequencies.double())[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def norm(x, weight, eps):
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return n if weight is None else n * weight


def apply(x, weight, positions, frequencies, interleaved, eps):
    return rotate(x if eps is None else norm(x, weight, eps), positions, frequencies, interleaved)


def derivatives(x, weight, positions, frequencies, interleaved, eps, dy, u=None, z=None):
    """y, dx, dw, and for cotangents u of dx and z of dw: those of x, weight and dy; in 64 bits."""
    double = lambda t: None if t is None else t.detach().double().cpu().requires_grad_()
    x, weight, dy = double(x), double(weight), double(dy)
    y = apply(x, weight, positions, frequencies, interleaved, eps)
    leaves = [x] if weight is None else [x, weight]
    first = torch.autograd.grad(y, leaves, dy, create_graph=u is not None)
    got = {"y": y.detach(), "dx": first[0].detach(), "dw": None if weight is None else first[1].detach()}
    if u is not None:
        cotangents = [t.double().cpu() for t in (u, z) if t is not None]
        second = torch.autograd.grad(first, [*leaves, dy], cotangents, allow_unused=True)
        got["dx2"] = torch.zeros_like(x) if second[0] is None else second[0]
        got["dw2"] = None if weight is None else second[1]
        got["ddy"] = second[-1]
    return got


def scales(x, weight, eps, dy, u, z):
    """What roundings of the row's terms are relative to, (rows, 1): the sums of the magnitudes that the
    formulas add, from the largest element of each factor in a row, with g of dy's 2-norm over pairs."""
    x, dy, u = x.double().cpu(), dy.double().cpu(), u.double().cpu()
    top = lambda t: t.abs().amax(-1, keepdim=True)
    if eps is None:
        zero = torch.zeros_like(top(x))
        return {"y": 2 * top(x), "dx": 2 * top(dy), "ddy": 2 * top(u), "dx2": zero}
    w = 1.0 if weight is None else float(weight.abs().max())
    zmax = 0.0 if z is None else float(z.abs().max())
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n, g = r * top(x), 2 * top(dy)  # (a turned pair's element is at most sqrt 2 times the larger)
    mean = lambda a, b: torch.sqrt((a * a).mean(-1, keepdim=True) * (b * b).mean(-1, keepdim=True))  # >= mean |a b|
    C, U = 2 * w * mean(dy, r * x), mean(u, r * x)
    A, Z = 2 * w * mean(u, dy), 2 * zmax * mean(dy, r * x)
    rest = top(u) + U * n
    return {"y": 2 * n * w, "dx": r * (g * w + C * n), "ddy": 2 * (r * w * rest + zmax * n),
            "dx2": r * r * (n * (3 * C * U + A) + U * g * w + C * top(u)) + r * (zmax * g + Z * n),
            "dw": g * n, "dw2": r * g * rest}
