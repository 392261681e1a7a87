"""Attention over a stream of tokens and the 4-bit format, from their definitions in 64 bits."""

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def visible(at, n, window, sinks):
    """[len(at), n]: key j <= p and (j > p - window or j < sinks)."""
    at, j = at[:, None], torch.arange(n, device=at.device)[None]
    return (j <= at) & ((j > at - window) | (j < sinks))


def attend(q, k, v, vis, scale=None):
    """q [Sq, Hq, D], k / v [n, Hkv, D], vis [Sq, n] -> (o, bound) in float64, [Sq, Hq, D] each.

    bound: how far a bf16 result may be from o.  One rounding of o (2^-8 |o|) and one of every probability (2^-8 p |v|);
    in 32 bits the scores (D + 1 operations on sums of at most S = max sum_d |q_d k_d| scale, and the rounding of the
    exponent's argument: S (D + 4) 2^-24 in the exponent of every p), the sums over the keys (n 2^-24 each for p and for
    p v), and exp2, divide and rescaling (8 roundings), each of them on p |v| in all:
    A (2^-8 + 2^-23 (n + S (D + 4) + 8)), A = sum p |v|; and half of bf16's smallest step."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    G = q.shape[1] // k.shape[1]
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(q.shape[1]):
        kh, vh = k[:, h // G], v[:, h // G]
        s = (q[:, h] @ kh.t().contiguous()) * scale
        s = torch.where(vis, s, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(vis.any(-1, keepdim=True), p, 0.0)
        keep = vis.any(0)
        # (a key that nobody sees may hold anything; one that some see counts where it is seen)
        vv = torch.where(keep[:, None], vh, 0.0)
        if not torch.isfinite(vv).all():
            o[:, h] = torch.where(vis[:, :, None], p[:, :, None] * vv[None], 0.0).sum(1)
        else:
            o[:, h] = p @ vv
        S = torch.nan_to_num((q[:, h].abs() @ torch.where(keep[:, None], kh, 0.0).abs().t().contiguous()) * scale).max() if vis.any() else 0.0
        n = int(vis.sum(-1).max()) if vis.numel() else 0
        rel = 2.0 ** -8 + 2.0 ** -23 * (n + float(S) * (q.shape[-1] + 4) + 8)
        bound[:, h] = 2.0 ** -8 * o[:, h].abs() + rel * (torch.nan_to_num(p) @ torch.nan_to_num(vv).abs()) + 2.0 ** -134
    return o, bound


def nearest(x):
    """[..., D] -> the float64 values that it stands for in 4 bits (NaN blocks where something is not finite), on the
    CPU, whose powers of two are exact."""
    b = x.cpu().double().unflatten(-1, (-1, 32))
    finite = torch.isfinite(b).all(-1, keepdim=True)
    b = torch.where(finite, b, 0.0)
    f, p = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (p - 3 + (f >= 0.875).to(p.dtype)).clamp(-125, 125)  # amax = 2 f 2^(p - 1)
    e = torch.where(f == 0, -125, e).double()
    y = (b * torch.pow(2.0, -e)).abs()
    odd = torch.tensor([0.0, 1e-12] * 4, dtype=torch.float64)  # of two as near, the even code
    code = ((y[..., None] - GRID).abs() + odd).argmin(-1)
    v = torch.where(torch.signbit(b), -GRID[code], GRID[code]) * torch.pow(2.0, e)
    return torch.where(finite, v, math.nan).flatten(-2).to(x.device)
