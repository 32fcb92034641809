"""Per-head RMS norm + rotary position embedding and its gradient, in float64 from the formulas."""
import torch


def freqs(rot, theta, inv_freq=None):
    if inv_freq is not None:
        return torch.tensor(list(inv_freq), dtype=torch.float64)
    i = torch.arange(rot // 2, dtype=torch.float64)
    return torch.tensor(theta, dtype=torch.float64) ** (-2.0 * i / max(rot, 1))


def angles(B, S, rot, theta, positions=None, pos0=0, inv_freq=None):
    """[B, S, 1, rot / 2] float64, each reduced to a turn before the cosine (positions are whole numbers, so the
    product of position and frequency is formed in extended precision by splitting the position)."""
    f = freqs(rot, theta, inv_freq) / (2 * torch.pi)
    p = (pos0 + torch.arange(S)).expand(B, S) if positions is None else positions.cpu().long()
    hi, lo = (p >> 12).double(), (p & 4095).double()
    fh = torch.round(f * 2 ** 26) / 2 ** 26                # f in two parts: every product below is exact or tiny
    fl = f - fh
    turns = torch.zeros(B, S, len(f), dtype=torch.float64)
    for part, w in ((hi, 4096.0), (lo, 1.0)):
        for g in (fh, fl):
            t = part[..., None] * g
            t = (t - torch.floor(t)) * w
            turns = turns + (t - torch.floor(t))
    turns = turns - torch.floor(turns)
    return (2 * torch.pi * turns)[:, :, None]


def pairs(rot, inter):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)


def rotate(x, ang, rot, inter, sign=1.0):
    ia, ib = pairs(rot, inter)
    y = x.clone()
    c, s = torch.cos(ang).to(x.device), sign * torch.sin(ang).to(x.device)
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


def size(x, rot, inter):
    """|a| + |b| of each rotated pair, |x| elsewhere: what a rounding in the rotation is relative to."""
    ia, ib = pairs(rot, inter)
    m = x.abs().clone()
    m[..., ia] = m[..., ib] = x[..., ia].abs() + x[..., ib].abs()
    return m


def fwd(x, gain, ang, rot, inter, eps):
    x = x.double()
    z = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if gain is not None:
        z = z * gain.double()
    return rotate(z, ang, rot, inter), size(z, rot, inter)


def bwd(dy, x, gain, ang, rot, inter, eps):
    """(dx, dgain, and for each the size that its rounding errors are relative to)."""
    x, dy = x.double(), dy.double()
    dh = x.shape[-1]
    g = torch.ones(dh, dtype=torch.float64, device=x.device) if gain is None else gain.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    xh = x * r
    d, m = rotate(dy, ang, rot, inter, -1.0), size(dy, rot, inter)
    w, mw = d * g, m * g.abs()
    dx = r * (w - xh * (w * xh).mean(-1, keepdim=True))
    mx = r * (mw + xh.abs() * (mw * xh.abs()).mean(-1, keepdim=True))
    return dx, (d * xh).sum((0, 1, 2)), mx, (m * xh.abs()).sum((0, 1, 2))
