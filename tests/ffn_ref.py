"""The gated feed-forward block and its gradient in float64, and bounds on the errors of a computation that
accumulates in FP32 and holds gu, h, dgu, dx and y in FP16.

E = 2^-23: one step of FP32, which an addition on the tensor cores may lose whole (they cut, not round), so a
sum of K products is off by at most K E of the sum of their sizes.  H = 2^-11: half a step of FP16 (2^-25 below
its normal range).  The activation and its derivative are right to 2^-20 relative to their terms.
"""
import math

import torch

E, H, TINY, ACT = 2.0 ** -23, 2.0 ** -11, 2.0 ** -25, 2.0 ** -20


def act(z, kind):
    """act(z), act'(z) and the size of the terms of act'(z)."""
    if kind == "silu":
        s, dr = torch.sigmoid(z), torch.ones_like(z)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        s, dr = torch.sigmoid(c * (z + 0.044715 * z ** 3)), c * (1 + 3 * 0.044715 * z ** 2)
    a = z * s
    return a, s + a * (1 - s) * dr, s + (a * (1 - s) * dr).abs() + (a * s * dr).abs()


def half_step(v):
    return H * v.abs() + TINY


def fwd(x, wgu, wd, bgu, bd, residual, kind):
    """{name: (value, bound)} of gu, h and y."""
    x, wgu, wd = x.double(), wgu.double(), wd.double()
    D, F = x.shape[1], wd.shape[1]
    z, S = x @ wgu.T, x.abs() @ wgu.abs().T
    if bgu is not None:
        z, S = z + bgu.double(), S + bgu.double().abs()
    dz = (D + 1) * E * S
    g, u = z[:, :F], z[:, F:]
    a, _, _ = act(g, kind)
    da = 1.13 * dz[:, :F]                                  # |act'| < 1.13 for both activations
    h = a * u
    dh = da * u.abs() + (a.abs() + da) * dz[:, F:] + 2 * ACT * h.abs()
    dh = dh + H * (h.abs() + dh) + TINY
    y, Sy = h @ wd.T, h.abs() @ wd.abs().T
    dy = dh @ wd.abs().T
    for t in (bd, residual):
        if t is not None:
            y, Sy = y + t.double(), Sy + t.double().abs()
    dy = dy + (F + 2) * E * (Sy + dy)
    return {"gu": (z, dz + H * (z.abs() + dz) + TINY), "h": (h, dh), "y": (y, dy + H * (y.abs() + dy) + TINY)}


def bwd(dy, x, gu, wgu, wd, kind):
    """{name: (value, bound)} of h, dgu, dx, dwgu, dbgu, dwd and dbd."""
    dy, x, gu, wgu, wd = (t.double() for t in (dy, x, gu, wgu, wd))
    N, D = dy.shape
    F = wd.shape[1]
    g, u = gu[:, :F], gu[:, F:]
    a, da, sa = act(g, kind)
    dh, edh = dy @ wd, D * E * (dy.abs() @ wd.abs())
    h = a * u
    dgu = torch.cat((dh * u * da, dh * a), 1)
    e = torch.cat((edh * (u * da).abs() + ACT * 4 * (dh.abs() + edh) * u.abs() * sa,
                   edh * a.abs() + ACT * 4 * (dh.abs() + edh) * a.abs()), 1)
    e = e + H * (dgu.abs() + e) + TINY
    big = dgu.abs() + e
    dx = dgu @ wgu
    edx = e @ wgu.abs() + 2 * F * E * (big @ wgu.abs())
    eh = 2 * ACT * h.abs() + H * h.abs() * 1.01 + TINY
    return {
        "h": (h, eh), "dgu": (dgu, e), "dx": (dx, edx + H * (dx.abs() + edx) + TINY),
        "dwgu": (dgu.T @ x, e.T @ x.abs() + (N + 1) * E * (big.T @ x.abs())),
        "dbgu": (dgu.sum(0), e.sum(0) + (N + 1) * E * big.sum(0)),
        "dwd": (dy.T @ h, dy.abs().T @ eh + (N + 1) * E * (dy.abs().T @ (h.abs() + eh))),
        "dbd": (dy.sum(0), (N + 1) * E * dy.abs().sum(0)),
    }
