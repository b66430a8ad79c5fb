"""Windowed attention and its first two derivatives in 64 bits on the CPU, from the closed
forms with whole score matrices: the oracle of the windowed kernels' tests."""

from __future__ import annotations

import torch


def visible(n_q, n_k, alignment, window, sinks):
    """(n_q, n_k) mask: key j is visible to query i at position p iff p - window < j <= p or
    j < sinks, j <= p. window 0: no window."""
    p = (torch.arange(n_q) + (n_k - n_q if alignment == "bottom_right" else 0))[:, None]
    j = torch.arange(n_k)[None, :]
    if not window:
        return j <= p
    return (j <= p) & ((j > p - window) | (j < sinks))


def _heads_first(x, group):
    x = x.detach().double().cpu().transpose(1, 2)
    return x.repeat_interleave(group, dim=1) if group > 1 else x


def _fold(x, group):
    """(B, H, T, D) -> (B, T, H / group, D), summed over groups."""
    return x.unflatten(1, (-1, group)).sum(2).transpose(1, 2)


def forward(q, k, v, mask, scale):
    """O (B, T, H, D) and L (B, H, T); a row that sees nothing has O = 0 and L = +inf."""
    group = q.shape[2] // k.shape[2]
    q, k, v = _heads_first(q, 1), _heads_first(k, group), _heads_first(v, group)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, -1)
    lse = torch.where(torch.isinf(lse), torch.full_like(lse, float("inf")), lse)
    return (torch.exp(s - lse[..., None]) @ v).transpose(1, 2), lse


def _common(q, k, v, o, do, lse, mask, scale):
    group = q.shape[2] // k.shape[2]
    q, k, v, o, do = (_heads_first(x, g) for x, g in ((q, 1), (k, group), (v, group), (o, 1), (do, 1)))
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~mask, float("-inf"))
    p = torch.exp(s - lse.double().cpu()[..., None])
    dp = do @ v.transpose(-1, -2)
    d = (o * do).sum(-1, keepdim=True)
    return group, q, k, v, do, p, dp, d


def backward(q, k, v, o, do, lse, mask, scale):
    """dQ, dK, dV and D (B, H, T)."""
    group, q, k, _, do, p, dp, d = _common(q, k, v, o, do, lse, mask, scale)
    ds = scale * p * (dp - d)
    return ((ds @ k).transpose(1, 2), _fold(ds.transpose(-1, -2) @ q, group), _fold(p.transpose(-1, -2) @ do, group),
            d[..., 0])


def double_backward(q, k, v, o, do, ddq, ddk, ddv, lse, mask, scale):
    """dQ2, dK2, dV2, ddO."""
    group, q, k, v, do, p, dp, d = _common(q, k, v, o, do, lse, mask, scale)
    ddq, ddk, ddv = _heads_first(ddq, 1), _heads_first(ddk, group), _heads_first(ddv, group)
    t = lambda x: x.transpose(-1, -2)
    dds = scale * (ddq @ t(k) + q @ t(ddk))
    dd = (dds * p).sum(-1, keepdim=True)
    dp2 = do @ t(ddv) - dp * dd - dds * d + dp * dds
    b = (dp2 * p).sum(-1, keepdim=True)
    ds, ds2, ddp = scale * p * (dp - d), scale * p * (dp2 - b), p * (dds - dd)
    return ((ds @ ddk + ds2 @ k).transpose(1, 2), _fold(t(ds) @ ddq + t(ds2) @ q, group), _fold(t(ddp) @ do, group),
            (p @ ddv + ddp @ v).transpose(1, 2))
