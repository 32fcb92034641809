"""Measured cases of the operators of a gated decoder block: per-head query / key
normalisation with the rotary position embedding, the gated feed-forward network, and
clipping by the gradients' global norm; forward and backward, training and decoding.

  qk    y = rotate(x * gain / sqrt(mean(x^2) + eps)) for each head of the queries and keys; backward
        dx and the gains' gradients.
  ffn   y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual, gate and up weights stacked in
        wgu [2F, D]; the training call also gives the pre-activations gu and the product h.  Backward
        from the saved gu: dgu, h again, and dx.  (The weight gradients are then plain products of dgu
        and h with x and dy, by the weight-gradient GEMM that this library already has.)
  clip  norm = sqrt(sum over all tensors of (g / loss scale)^2), and g * min(1, max_norm / norm).

`run` gives the plain form, in FP32 torch operations, or with `own` the library's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rubidium-train_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from rbk import ops
    return ops


# ---------------------------------------------------------------------- cases --

def _qk(name, back, B, S, Hq, Hk, dh, rot=None, inter=False, pos="seq", theta=10000.0):
    """pos "seq": row s of each sequence is position s; "far": each row has its own position, up to a million."""
    return dict(name=name, kind="qk", back=back, B=B, S=S, Hq=Hq, Hk=Hk, dh=dh, rot=dh if rot is None else rot,
                inter=inter, pos=pos, theta=theta)


def _ffn(name, back, N, D, F, act="silu", bias=False, res=False, save=True):
    return dict(name=name, kind="ffn", back=back, N=N, D=D, F=F, act=act, bias=bias, res=res, save=save)


def _clip(name, L, D, F, V, T, types="f32", rank=0, shift=0, ratio=8.0):
    """Tensors of an L-layer gated decoder (rank > 0: only its rank-r adapters).  ratio: norm / max_norm.  shift:
    elements by which every gradient starts off a 16-byte boundary."""
    return dict(name=name, kind="clip", L=L, D=D, F=F, V=V, T=T, types=types, rank=rank, shift=shift, ratio=ratio)


def listed():
    return [
        # one new token for each of 32 sequences of the 1.3B decoder (H 16, d_head 128), far into their texts
        _qk("qk_decode_32", False, 32, 1, 16, 16, 128, pos="far"),
        # a training micro-batch of the 1.3B decoder, 8 x 2048 tokens
        _qk("qk_fwd_16k", False, 8, 2048, 16, 16, 128),
        # its backward pass
        _qk("qk_bwd_16k", True, 8, 2048, 16, 16, 128),
        # GPT-2-small heads, 16 x 1024 tokens, backward
        _qk("qk_bwd_gpt2", True, 16, 1024, 12, 12, 64),
        # ragged: shared key heads, an odd sequence length, a partial rotation of neighbouring pairs
        _qk("qk_bwd_ragged", True, 3, 347, 10, 2, 80, rot=32, inter=True, pos="far", theta=500000.0),
        # one new token through a block of width 2048: the weights are all that counts
        _ffn("ffn_decode_1", False, 1, 2048, 5632, res=True, save=False),
        # a small odd batch with biases
        _ffn("ffn_decode_21", False, 21, 1000, 2664, act="gelu", bias=True, save=False),
        # a training micro-batch, 4 x 2048 tokens
        _ffn("ffn_fwd_8k", False, 8192, 2048, 5632),
        # its backward pass
        _ffn("ffn_bwd_8k", True, 8192, 2048, 5632),
        # ragged sizes, narrow block, GELU
        _ffn("ffn_bwd_ragged", True, 1999, 776, 2056, act="gelu"),
        # rank-16 adapters of a 12-layer decoder: 48 small tensors
        _clip("clip_adapters", 12, 768, 2048, 50257, 1024, rank=16),
        # every gradient of a GPT-2-small-sized gated decoder
        _clip("clip_124m", 12, 768, 2048, 50257, 1024),
    ]


def _log(rng, a, b, step=1):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b))) / step)) * step))


def draw(rng):
    kind = rng.choice(["qk", "ffn", "clip"])
    if kind == "qk":
        dh = rng.choice([16, 40, 64, 72, 80, 96, 128, 128, 200, 256])
        Hk = rng.randint(1, 16)
        Hq = Hk * rng.randint(1, max(1, 16 // Hk))
        B = _log(rng, 1, 32)
        S = _log(rng, 1, max(1, 8 * 2048 * 32 * 128 // (B * (Hq + Hk) * dh)))
        S = min(S, 8192)
        inter = rng.random() < 0.4
        step = 8 if inter else 16
        rot = rng.choice([dh // step, rng.randint(1, dh // step)]) * step
        c = _qk("", rng.random() < 0.5, B, S, Hq, Hk, dh, rot, inter, rng.choice(["seq", "far"]),
                rng.choice([10000.0, 500000.0]))
    elif kind == "ffn":
        D, F = _log(rng, 256, 2048, 8), _log(rng, 256, 5632, 8)
        back = rng.random() < 0.5
        N = _log(rng, 1, 64) if not back and rng.random() < 0.5 else _log(rng, 64, 8192)
        c = _ffn("", back, N, D, F, rng.choice(["silu", "gelu"]), rng.random() < 0.5, rng.random() < 0.5,
                 rng.random() < 0.5)
    else:
        rank = rng.choice([0, 0, 4, 16, 64])
        c = _clip("", rng.randint(1, 12), _log(rng, 64, 768), _log(rng, 64, 2048), _log(rng, 256, 50257),
                  _log(rng, 64, 1024), rng.choice(["f32", "f16", "mixed"]), rank, rng.choice([0, 0, 1, 3]),
                  math.exp(rng.uniform(math.log(0.3), math.log(30.0))))
    del c["name"]
    return c


def _shapes(c):
    """[(elements, dtype)] of the tensors that a clip case covers."""
    D, F, L = c["D"], c["F"], c["L"]
    mat = torch.float32 if c["types"] == "f32" else torch.float16
    vec = torch.float16 if c["types"] == "f16" else torch.float32
    if c["rank"]:
        return [(D * c["rank"], mat)] * (4 * L)
    layer = [(D, vec), (D * D, mat), (D * D, mat), (D * D, mat), (D, vec), (D * D, mat), (D, vec), (D, vec),
             (2 * F * D, mat), (2 * F, vec), (F * D, mat), (D, vec)]
    return [(c["V"] * D, mat), (c["T"] * D, mat)] + layer * L + [(D, vec), (c["V"] * D, mat), (c["V"], vec)]


def work(c):
    if c["kind"] == "qk":
        n = c["B"] * c["S"] * (c["Hq"] + c["Hk"]) * c["dh"]
        if c["back"]:
            return {"bytes": 6 * n + 12 * c["dh"], "flops": 14 * n}
        return {"bytes": 4 * n + 4 * c["dh"], "flops": 7 * n}
    if c["kind"] == "ffn":
        N, D, F = c["N"], c["D"], c["F"]
        if c["back"]:                                  # dy, gu, wd, wgu in; dgu, h, dx out
            return {"bytes": 2 * (2 * N * D + 5 * N * F + 3 * F * D), "flops": 6 * N * D * F}
        b = 2 * (2 * N * D + 3 * F * D + (3 * N * F if c["save"] else 0) + (N * D if c["res"] else 0))
        return {"bytes": b + (2 * (2 * F + D) if c["bias"] else 0), "flops": 6 * N * D * F}
    n = sum(k for k, _ in _shapes(c))
    return {"bytes": 2 * sum(k * t.itemsize for k, t in _shapes(c)) + 4, "flops": 3 * n}


# --------------------------------------------------------------------- inputs --

def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def r(*shape, scale=1.0):
        return torch.randn(*shape, device=DEV, generator=g).mul_(scale)

    s = dict(c)
    if c["kind"] == "qk":
        B, S, Hq, Hk, dh = c["B"], c["S"], c["Hq"], c["Hk"], c["dh"]
        # the projections of queries and keys side by side, as one GEMM leaves them; the results go next to
        # the values, where the attention reads them
        qk = r(B, S, Hq + Hk, dh).half()
        s["q"], s["k"] = qk[:, :, :Hq], qk[:, :, Hq:]
        s["gq"], s["gk"] = (1 + r(dh, scale=0.1)).half(), (1 + r(dh, scale=0.1)).half()
        if c["back"]:
            dqkv = r(B, S, Hq + 2 * Hk, dh).half()
            s["dyq"], s["dyk"] = dqkv[:, :, :Hq], dqkv[:, :, Hq:Hq + Hk]
        else:
            qkv = torch.zeros(B, S, Hq + 2 * Hk, dh, device=DEV, dtype=torch.float16)
            s["out"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        s["positions"] = None
        if c["pos"] == "far":
            s["positions"] = torch.randint(0, 1000000, (B, S), device=DEV, generator=g, dtype=torch.int32)
    elif c["kind"] == "ffn":
        N, D, F = c["N"], c["D"], c["F"]
        s["x"] = r(N, D).half()
        s["wgu"], s["wd"] = r(2 * F, D, scale=D ** -0.5).half(), r(D, F, scale=F ** -0.5).half()
        s["bgu"], s["bd"] = (r(2 * F, scale=0.1).half(), r(D, scale=0.1).half()) if c["bias"] else (None, None)
        s["residual"] = r(N, D).half() if c["res"] else None
        if c["back"]:
            s["dy"] = r(N, D).half()
            s["gu"] = (s["x"] @ s["wgu"].T).half()     # what the forward pass has saved
    else:
        shapes = _shapes(c)
        n = sum(k for k, _ in shapes)
        loss_scale = 1024.0
        sigma = c["ratio"] * loss_scale / math.sqrt(n)
        s["max_norm"] = 1.0
        # the device-resident loss scaler: its first word is the scale
        s["scaler"] = torch.tensor([loss_scale, 0, 0, 0, 0, 0, 0, 0], device=DEV).view(torch.int32)
        s["grads"] = [r(k + c["shift"], scale=sigma).to(t)[c["shift"]:] for k, t in shapes]
        # the clipped gradients go into one arena for each type, every tensor on a multiple of 64 elements
        s["arenas"], s["out"], used = {}, [], {}
        for k, t in shapes:
            used[t] = used.get(t, 0) + (k + 63) // 64 * 64
        for t, m in used.items():
            s["arenas"][t] = torch.zeros(m, device=DEV, dtype=t)
        at = dict.fromkeys(used, 0)
        for k, t in shapes:
            s["out"].append(s["arenas"][t][at[t]:at[t] + k])
            at[t] += (k + 63) // 64 * 64
    return s


# ---------------------------------------------------------------- plain forms --

def _turns(s):
    """cos and sin [B or 1, S, 1, rot / 2] of the positions' angles, computed in 64 bits."""
    if s["positions"] is None:
        p = torch.arange(s["S"], device=DEV, dtype=torch.float64)[None]
    else:
        p = s["positions"].double()
    i = torch.arange(s["rot"] // 2, device=DEV, dtype=torch.float64)
    a = p[:, :, None, None] * s["theta"] ** (-2.0 * i / s["rot"])
    return a.cos().float(), a.sin().float()


def _pairs(s, x):
    rot = s["rot"]
    if s["inter"]:
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]


def _joined(s, a, b, rest):
    ab = torch.stack((a, b), -1).flatten(-2) if s["inter"] else torch.cat((a, b), -1)
    return torch.cat((ab, rest), -1)


def _qk_fwd(s, x, gain, cos, sin):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
    a, b, rest = _pairs(s, y)
    return _joined(s, a * cos - b * sin, a * sin + b * cos, rest).half()


def _qk_bwd(s, dy, x, gain, cos, sin):
    x = x.float()
    a, b, rest = _pairs(s, dy.float())
    d = _joined(s, a * cos + b * sin, b * cos - a * sin, rest)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xhat = x * rstd
    dgain = (d * xhat).sum((0, 1, 2))
    d = d * gain.float()
    return (rstd * (d - xhat * (d * xhat).mean(-1, keepdim=True))).half(), dgain


def _act(s, z):
    """The activation and its derivative."""
    if s["act"] == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    c, a = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (z + a * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * a * z * z)


def _ffn_fwd(s):
    gu = s["x"].float() @ s["wgu"].float().T
    if s["bias"]:
        gu = gu + s["bgu"].float()
    g, u = gu.chunk(2, -1)
    h = _act(s, g)[0] * u
    y = h @ s["wd"].float().T
    if s["bias"]:
        y = y + s["bd"].float()
    if s["res"]:
        y = y + s["residual"].float()
    return {"y": y.half(), "gu": gu.half(), "h": h.half()} if s["save"] else {"y": y.half()}


def _ffn_bwd(s):
    dh = s["dy"].float() @ s["wd"].float()
    g, u = s["gu"].float().chunk(2, -1)
    f, df = _act(s, g)
    dgu = torch.cat((dh * u * df, dh * f), -1)
    return {"dx": (dgu @ s["wgu"].float()).half(), "dgu": dgu.half(), "h": (f * u).half()}


def _clip_all(s):
    scale = s["scaler"][:1].view(torch.float32)
    squares = torch.stack([(g.float() / scale).square().sum(dtype=torch.float64) for g in s["grads"]])
    norm = squares.sum().sqrt().float()
    coef = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
    [o.copy_(g.float() * coef) for o, g in zip(s["out"], s["grads"])]
    return {"norm": norm.reshape(1), "clipped": list(s["arenas"].values())}


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "qk":
        cos, sin = _turns(s)
        if s["back"]:
            dq, dgq = _qk_bwd(s, s["dyq"], s["q"], s["gq"], cos, sin)
            dk, dgk = _qk_bwd(s, s["dyk"], s["k"], s["gk"], cos, sin)
            return {"dq": dq, "dk": dk, "dgq": dgq, "dgk": dgk}
        return {"yq": _qk_fwd(s, s["q"], s["gq"], cos, sin), "yk": _qk_fwd(s, s["k"], s["gk"], cos, sin)}
    if s["kind"] == "ffn":
        return _ffn_bwd(s) if s["back"] else _ffn_fwd(s)
    return _clip_all(s)


# ------------------------------------------------------------ the library's calls --

def _run_own(s):
    ops = _ops()
    if s["kind"] == "qk":
        how = dict(positions=s["positions"], theta=s["theta"], rot=s["rot"], interleaved=s["inter"], eps=EPS)
        if s["back"]:
            dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(s["dyq"], s["dyk"], s["q"], s["k"], s["gq"], s["gk"], **how)
            return {"dq": dq, "dk": dk, "dgq": dgq, "dgk": dgk}
        yq, yk = ops.qk_norm_rope_fwd(s["q"], s["k"], s["gq"], s["gk"], out=s["out"], **how)
        return {"yq": yq, "yk": yk}
    if s["kind"] == "ffn":
        if s["back"]:
            dx, dgu, h = ops.gated_ffn_bwd(s["dy"], s["x"], s["gu"], s["wgu"], s["wd"], act=s["act"])
            return {"dx": dx, "dgu": dgu, "h": h}
        y, gu, h = ops.gated_ffn_fwd(s["x"], s["wgu"], s["wd"], bgu=s["bgu"], bd=s["bd"], residual=s["residual"],
                                     act=s["act"], save=s["save"])
        return {"y": y, "gu": gu, "h": h} if s["save"] else {"y": y}
    norm = ops.clip_grad_norm(s["grads"], s["max_norm"], scaler=s["scaler"], out=s["out"])
    return {"norm": norm, "clipped": list(s["arenas"].values())}


# ------------------------------------------------------------- exact, in 64 bits --

def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "qk":
        return _exact_qk(c, s)
    if c["kind"] == "ffn":
        return _exact_ffn(c, s)
    scale = float(s["scaler"][:1].view(torch.float32))
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"])) / scale
    coef = min(1.0, s["max_norm"] / norm)
    arenas = {t: a.double() for t, a in s["arenas"].items()}
    at = dict.fromkeys(arenas, 0)
    for g in s["grads"]:
        arenas[g.dtype][at[g.dtype]:at[g.dtype] + g.numel()] = g.double() * coef
        at[g.dtype] += (g.numel() + 63) // 64 * 64
    return {"norm": torch.tensor([norm], dtype=torch.float64), "clipped": list(arenas.values())}


def _exact_qk(c, s):
    """The rotation as a product of complex numbers."""
    rot, dh = c["rot"], c["dh"]
    at = np.arange(rot).reshape(-1, 2) if c["inter"] else np.arange(rot).reshape(2, -1).T
    re, im = (torch.from_numpy(np.ascontiguousarray(at[:, j])).to(DEV) for j in (0, 1))
    freq = torch.from_numpy(np.float64(c["theta"]) ** (-np.arange(0, rot, 2) / rot)).to(DEV)
    if s["positions"] is None:
        p = torch.arange(c["S"], device=DEV).double().expand(c["B"], -1)
    else:
        p = s["positions"].double()
    one = torch.ones((), device=DEV, dtype=torch.float64)
    turn = torch.polar(one, p[..., None] * freq)[:, :, None]                       # [B, S, 1, rot / 2]

    def rotated(v, w):
        z = torch.complex(v[..., re], v[..., im]) * w
        v = v.clone()
        v[..., re], v[..., im] = z.real, z.imag
        return v

    def each(dy, x, gain):
        gain, v = gain.double(), x.double()
        rms = (v.square().sum(-1, keepdim=True) / dh + EPS).sqrt()
        if dy is None:
            return rotated(v / rms * gain, turn), None
        d = rotated(dy.double(), turn.conj())
        w = d * gain
        return w / rms - v * (w * v).sum(-1, keepdim=True) / (dh * rms ** 3), (d * v / rms).flatten(0, 2).sum(0)

    if c["back"]:
        (dq, dgq), (dk, dgk) = each(s["dyq"], s["q"], s["gq"]), each(s["dyk"], s["k"], s["gk"])
        return {"dq": dq, "dk": dk, "dgq": dgq, "dgk": dgk}
    return {"yq": each(None, s["q"], s["gq"])[0], "yk": each(None, s["k"], s["gk"])[0]}


def _exact_ffn(c, s):
    """Gate and up apart, the activations as z times a logistic function of z."""
    N, D, F = c["N"], c["D"], c["F"]
    wg, wu, wd = s["wgu"][:F].double(), s["wgu"][F:].double(), s["wd"].double()

    def gate(z):
        """(p, k): act(z) = z p, act'(z) = p + z p (1 - p) k."""
        if c["act"] == "silu":
            return torch.special.expit(z), 1.0
        a, b = math.sqrt(8 / math.pi), 0.044715 * math.sqrt(8 / math.pi)
        return torch.special.expit(a * z + b * z ** 3), a + 3 * b * z ** 2

    if c["back"]:
        dh, g, u = s["dy"].double() @ wd, s["gu"][:, :F].double(), s["gu"][:, F:].double()
        p, k = gate(g)
        dg, du = dh * u * (p + g * p * (1 - p) * k), dh * (g * p)
        return {"dx": dg @ wg + du @ wu, "dgu": torch.cat((dg, du), 1), "h": g * p * u}
    x = s["x"].double()
    g, u = x @ wg.T, x @ wu.T
    if c["bias"]:
        g, u = g + s["bgu"][:F].double(), u + s["bgu"][F:].double()
    h = g * gate(g)[0] * u
    y = h @ wd.T
    if c["bias"]:
        y = y + s["bd"].double()
    if c["res"]:
        y = y + s["residual"].double()
    return {"y": y, "gu": torch.cat((g, u), 1), "h": h} if c["save"] else {"y": y}
