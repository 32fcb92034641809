"""Torch-tensor face of the librbk kernels.

Each function mirrors the reference operator it replaces (names and argument
meaning of src/cuda_kernels.cuh), launches on torch's current CUDA stream and
calls straight into librbk.so through the C ABI.  Tensors must live on the
device of the active context; there is no host or PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
import itertools
import operator
import struct
import threading

import torch

from ._lib import FFN_BWD_PACK, FFN_PACK, QK_PACK, GemmDesc, RbkError, Scaler, TailArgs, call, lib

EPI_STORE_F16, EPI_BIAS_GELU, EPI_GELU_BWD, EPI_ACC_F32, EPI_STORE_F32 = range(5)
LN_REFERENCE_FORMULA = 1

_tls = threading.local()
# The current device's index and a device's current stream.  torch.cuda's own functions take 0.2 and 1.3 us a call,
# those below it 0.1 each, which counts where a call takes some ten; a torch without them (a CPU build) imports all the same.
_dev = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)


class Context:
    """rbk_ctx bound to one device (scratch arena + flags)."""

    def __init__(self, device: int | None = None):
        if device is None:
            device = torch.cuda.current_device()
        self.device = device
        h = C.c_void_p()
        call("rbk_ctx_create", C.byref(h), device)
        self.handle = h

    def close(self):
        if self.handle:
            lib().rbk_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def device_error() -> int:
    """Read and clear the context's device status word (0, or RBK_ERR_TIMEOUT after a bounded wait gave up)."""
    torch.cuda.synchronize()
    st = C.c_int(0)
    call("rbk_ctx_device_error", ctx().handle, C.byref(st))
    return st.value


def ctx() -> Context:
    dev = torch.cuda.current_device()
    cache = getattr(_tls, "ctxs", None)
    if cache is None:
        cache = _tls.ctxs = {}
    if dev not in cache:
        cache[dev] = Context(dev)
    return cache[dev]


def _s():
    return C.c_void_p(_raw_stream(torch.cuda.current_device()))


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _need(t, dtype, name):
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor, got {t.dtype} on {t.device}")


def _refuse(t, dtype, name, shape, what):
    raise ValueError(f"{name}: expected {what} {dtype} tensor of shape {tuple(shape)} on cuda:{torch.cuda.current_device()}, "
                     f"got {t.dtype}, shape {tuple(t.shape)}, strides {t.stride()} on {t.device}")


def _here(t, dtype, name, shape):
    """The address of a contiguous tensor of this type and shape on the current device."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == _dev() and t.is_contiguous():
        return t.data_ptr()
    _refuse(t, dtype, name, shape, "a contiguous")


# ----------------------------------------------------------------- LayerNorm --

def ln_fwd(x, gamma, beta, eps=1e-5):
    """layer_norm_fp16_forward (src/cuda_kernels.cuh:99): returns (y, mean, rstd)."""
    _need(x, torch.float16, "x")
    N, D = x.shape
    y = torch.empty_like(x)
    mean = torch.empty(N, dtype=torch.float32, device=x.device)
    rstd = torch.empty(N, dtype=torch.float32, device=x.device)
    call("rbk_ln_fwd", ctx().handle, _p(y), _p(mean), _p(rstd), _p(x), _p(gamma), _p(beta), N, D,
         C.c_float(eps), _s())
    return y, mean, rstd


def ln_bwd(dy, x, gamma, mean, rstd, dres=None, want_dbias=False, ref_formula=False, dgamma=None, dbeta=None):
    """layer_norm_fp16_backward (src/cuda_kernels.cuh:102): returns (dx, dgamma, dbeta, dbias|None).
    dgamma/dbeta accumulate into the given FP32 tensors (zeros when omitted)."""
    _need(dy, torch.float16, "dy")
    N, D = x.shape
    dx = torch.empty_like(x)
    dgamma = torch.zeros(D, dtype=torch.float32, device=x.device) if dgamma is None else dgamma
    dbeta = torch.zeros(D, dtype=torch.float32, device=x.device) if dbeta is None else dbeta
    dbias = torch.zeros(D, dtype=torch.float32, device=x.device) if want_dbias else None
    call("rbk_ln_bwd", ctx().handle, _p(dx), _p(dgamma), _p(dbeta), _p(dbias), _p(dy), _p(dres), _p(x),
         _p(gamma), _p(mean), _p(rstd), N, D, LN_REFERENCE_FORMULA if ref_formula else 0, _s())
    return dx, dgamma, dbeta, dbias


# ------------------------------------------------------------- cross entropy --

def softmax_xent_bwd(logits, targets, scale=None, dscale=None, out=None, V=None, want_loss=True):
    """cross_entropy_fp32_forward + _backward (src/cuda_kernels.cuh:127-128) in one pass.
    logits: half [N, ld] (first V columns valid).  scale defaults to 1/N, the
    reference's mean (src/cpu_mat.h:233).  Returns (dlogits, row_loss)."""
    N, ld = logits.shape
    V = ld if V is None else V
    scale = 1.0 / N if scale is None else scale
    d = torch.empty_like(logits) if out is None else out
    row_loss = torch.empty(N, dtype=torch.float32, device=logits.device) if want_loss else None
    call("rbk_softmax_xent_bwd", ctx().handle, _p(d), _p(logits), ld, _p(targets), N, V, C.c_float(scale),
         _p(dscale), _p(row_loss), _s())
    return d, row_loss


def attn_softmax_bwd(P, dP, causal=True, out=None):
    """softmax_fp16_backward over stacked [T, T] matrices (src/cuda_kernels.cuh:120)."""
    T = P.shape[-1]
    nmat = P.numel() // (T * T)
    dS = torch.empty_like(P) if out is None else out
    call("rbk_attn_softmax_bwd", ctx().handle, _p(dS), _p(P), _p(dP), nmat, T, int(causal), _s())
    return dS


# ---------------------------------------------------------------- embeddings --

def embed_fwd(tok_emb, pos_emb, tokens, B, S):
    V, D = tok_emb.shape
    x = torch.empty(B * S, D, dtype=torch.float16, device=tok_emb.device)
    call("rbk_embed_fwd", ctx().handle, _p(x), _p(tok_emb), _p(pos_emb), _p(tokens), B, S, D, V, _s())
    return x


def embed_bwd(dx, tokens, B, S, V, dtok=None, dpos=None):
    D = dx.shape[1]
    dtok = torch.zeros(V, D, dtype=torch.float32, device=dx.device) if dtok is None else dtok
    dpos = torch.zeros(S, D, dtype=torch.float32, device=dx.device) if dpos is None else dpos
    call("rbk_embed_bwd", ctx().handle, _p(dtok), _p(dpos), _p(dx), _p(tokens), B, S, D, V, _s())
    return dtok, dpos


# --------------------------------------------------------------------- tail --

def new_scaler(scale=65536.0, interval=2000, device=None):
    """A device-resident rbk_scaler (8 int32-sized fields)."""
    s = Scaler(scale, 0, interval, 0, 0, 0, 0, 0)
    buf = torch.empty(8, dtype=torch.int32, device=device or torch.cuda.current_device())
    host = torch.frombuffer(bytearray(bytes(s)), dtype=torch.int32)
    buf.copy_(host)
    return buf


def read_scaler(buf) -> Scaler:
    raw = buf.cpu().numpy().tobytes()
    return Scaler.from_buffer_copy(raw)


def adam_tail(p32, g, m, v, p16, scaler_buf, lr, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, t=0,
              seg_off=None, seg_len=None, max_norm=0.0):
    """Fused unscale + inf check + skip + clip + AdamW + fp16 copy + grad zero."""
    a = TailArgs()
    a.p32, a.g, a.m, a.v = p32.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr()
    a.p16 = p16.data_ptr() if p16 is not None else None
    a.n = p32.numel()
    if seg_off is not None:
        so = (C.c_int64 * len(seg_off))(*seg_off)
        sl = (C.c_int64 * len(seg_len))(*seg_len)
        a.seg_off = C.cast(so, C.POINTER(C.c_int64))
        a.seg_len = C.cast(sl, C.POINTER(C.c_int64))
        a.nseg = len(seg_off)
    a.max_norm = max_norm
    a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = lr, b1, b2, eps, wd
    a.t = t
    a.scaler = scaler_buf.data_ptr()
    call("rbk_adam_tail", ctx().handle, C.byref(a), _s())


RBK_CLIP_WS_BYTES = 16 << 10
_dtype = operator.attrgetter("dtype")


def clip_grad_norm(grads, max_norm, scaler=None, out=None):
    """Clip by the norm over all tensors (rbk_clip_grad_norm): returns the FP32 norm [1] of the gradients divided by
    the loss scale, and multiplies them by min(1, max_norm / norm), in place or into `out`.

    grads: contiguous FP32 or half tensors.  scaler: a new_scaler() buffer (None: no loss scale).  out: a tensor for each
    of its gradient's type and size, or None in a place to count that gradient and not write it.  max_norm <= 0: only
    the norm is computed (and `out` is a copy).  The norm is over what this call is given: not for a model with the
    sharded optimizer (dp_init(shard=True)), whose ranks hold different slices of the reduced gradients."""
    dev, n = _dev(), len(grads)
    f32, f16 = torch.float32, torch.float16
    T = torch.Tensor
    kinds = list(map(_dtype, grads))
    sizes = list(map(T.numel, grads))
    if (set(kinds) - {f32, f16} or set(map(T.get_device, grads)) - {dev} or not all(map(T.is_contiguous, grads))):
        raise ValueError(f"grads: expected contiguous FP32 or half tensors on cuda:{dev}, got "
                         f"{sorted({(str(g.dtype), str(g.device), g.is_contiguous()) for g in grads})}")
    at = to = list(map(T.data_ptr, grads))
    if out is not None:
        some = [g if o is None else o for g, o in zip(grads, out)]
        if (len(out) != n or list(map(_dtype, some)) != kinds or list(map(T.numel, some)) != sizes
                or set(map(T.get_device, some)) - {dev} or not all(map(T.is_contiguous, some))):
            raise ValueError(f"out: expected {n} contiguous tensors (or None) of the gradients' types and sizes on cuda:{dev}")
        to = [0 if o is None else o.data_ptr() for o in out]
    sc = None if scaler is None else _here(scaler, torch.int32, "scaler", (8,))
    table = struct.pack(f"{4 * n}q", *itertools.chain.from_iterable(zip(at, to, sizes, [k is f16 for k in kinds])))
    norm = torch.empty(1, dtype=f32, device="cuda")
    ws = torch.empty(RBK_CLIP_WS_BYTES, dtype=torch.uint8, device="cuda")
    call("rbk_clip_grad_norm", ctx().handle, table, n, max_norm, sc, norm.data_ptr(), ws.data_ptr(), _s())
    return norm


# --------------------------------------------------------------------- LoRA --

def lora_fwd(x, A, B, y, scaling, xa=None):
    """One LoRA adapter (rbk_lora_fwd): xa = x A, y += scaling xa B (y in place, any row
    stride).  x [N, in], A [in, r], B [r, out] FP16.  Returns xa."""
    N, in_ = x.shape[0], A.shape[0]
    r, out = B.shape
    xa = torch.empty(N, r, dtype=torch.float16, device=x.device) if xa is None else xa
    call("rbk_lora_fwd", ctx().handle, _p(y), y.stride(0), _p(xa), _p(x), x.stride(0), _p(A), _p(B), N, in_, r, out,
         C.c_float(scaling), _s())
    return xa


def lora_bwd(dy, x, xa, A, B, scaling, dA, dB, dx=None):
    """Its backward (rbk_lora_bwd): dB += s xa^T dy, dA += x^T (s dy B^T), dx += (s dy B^T) A^T."""
    N, in_ = x.shape[0], A.shape[0]
    r, out = B.shape
    dyb = torch.empty(N, r, dtype=torch.float16, device=x.device)
    call("rbk_lora_bwd", ctx().handle, _p(dA), _p(dB), _p(dx) if dx is not None else None,
         dx.stride(0) if dx is not None else 0, _p(dyb), _p(dy), dy.stride(0), _p(x), x.stride(0), _p(xa), _p(A), _p(B),
         N, in_, r, out, C.c_float(scaling), _s())


# --------------------------------------------------------------------- GEMM --

def gemm(A, B, M, N, K, a_major=0, b_major=0, C_out=None, epilogue=EPI_STORE_F16, bias=None, aux=None,
         aux_out=None, dbias_rows=None, alpha=1.0, split_k=0, lda=None, ldb=None, ldc=None, ld_aux=0, store_c=True):
    """C[M,N] = op(A)[M,K] op(B)[N,K]^T on tcgen05 (see rbk_gemm_desc).  store_c=False with
    EPI_BIAS_GELU stores only the activation (aux_out)."""
    d = GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.A, d.lda, d.a_major = A.data_ptr(), lda or A.shape[-1], a_major
    d.B, d.ldb, d.b_major = B.data_ptr(), ldb or B.shape[-1], b_major
    if C_out is None:
        dt = torch.float32 if epilogue in (EPI_ACC_F32, EPI_STORE_F32) else torch.float16
        C_out = (torch.zeros if epilogue == EPI_ACC_F32 else torch.empty)(M, N, dtype=dt, device=A.device)
    d.C, d.ldc = (C_out.data_ptr() if store_c else None), ldc or C_out.shape[-1]
    d.epilogue = epilogue
    d.bias = bias.data_ptr() if bias is not None else None
    d.aux = aux.data_ptr() if aux is not None else None
    d.ld_aux = ld_aux
    d.aux_out = aux_out.data_ptr() if aux_out is not None else None
    d.dbias_rows = dbias_rows.data_ptr() if dbias_rows is not None else None
    d.alpha = alpha
    d.split_k = split_k
    call("rbk_gemm", ctx().handle, C.byref(d), _s())
    return C_out


def linear_fwd(X, W, bias=None, residual=None):
    """linear_forward_fp16 (src/cuda_kernels.cuh:190): Y = X W^T (+ b) (+ residual)."""
    N, fin = X.shape
    out = W.shape[0]
    Y = torch.empty(N, out, dtype=torch.float16, device=X.device)
    call("rbk_linear_fwd", ctx().handle, _p(Y), _p(X), _p(W), _p(bias), _p(residual), N, fin, out, _s())
    return Y


def gemm_dgrad(dY, W, gelu_pre=None):
    """gemm_fp16_accum_fp32_backward_dA (src/cuda_kernels.cuh:144): dX = dY W [* gelu'(pre)]."""
    N, out = dY.shape
    fin = W.shape[1]
    dX = torch.empty(N, fin, dtype=torch.float16, device=dY.device)
    call("rbk_gemm_dgrad", ctx().handle, _p(dX), _p(dY), _p(W), N, fin, out, _p(gelu_pre), _s())
    return dX


def gemm_wgrad(dY, X, dW=None, dbias=None):
    """gemm_fp16_accum_fp32_backward_dB (src/cuda_kernels.cuh:146): dW += dY^T X, dbias += colsum(dY)."""
    N, out = dY.shape
    fin = X.shape[1]
    dW = torch.zeros(out, fin, dtype=torch.float32, device=dY.device) if dW is None else dW
    call("rbk_gemm_wgrad", ctx().handle, _p(dW), _p(dbias), _p(dY), _p(X), N, fin, out, _s())
    return dW


# ---------------------------------------------------------------- attention --

def attn_fwd(qkv, B, S, H, dh, scale=None):
    """Causal flash attention forward: returns (o [B*S, H*dh] half, lse [B, H, S] fp32)."""
    scale = dh ** -0.5 if scale is None else scale
    o = torch.empty(B * S, H * dh, dtype=torch.float16, device=qkv.device)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=qkv.device)
    call("rbk_attn_fwd", ctx().handle, _p(o), _p(lse), _p(qkv), B, S, H, dh, C.c_float(scale), _s())
    return o, lse


def attn_bwd(qkv, o, dout, lse, B, S, H, dh, scale=None, dbias=None):
    scale = dh ** -0.5 if scale is None else scale
    dqkv = torch.empty_like(qkv)
    call("rbk_attn_bwd", ctx().handle, _p(dqkv), _p(dbias), _p(qkv), _p(o), _p(dout), _p(lse), B, S, H, dh,
         C.c_float(scale), _s())
    return dqkv


# ------------------------------------------------- query / key norm, rotation --

RBK_QK_BWD_WS_BYTES = 1024 * 256 * 4


_F16, _F32 = torch.float16, torch.float32
_NO_HEADS = (0, 0, 0, 0)


def _heads(t, name, shape):
    """Address and strides of half heads [B, S, H, dh] with contiguous channels (an rbk_heads)."""
    st = t.stride()
    if (t.dtype is _F16 and t.shape == shape and t.get_device() == _dev() and len(st) == 4
            and (st[3] == 1 or shape[3] == 1)):
        if (st[0] | st[1] | st[2]) & 7:                     # the stride of an axis of size 1 says nothing
            st = [s if n > 1 else 0 for s, n in zip(st, shape)]
        return t.data_ptr(), st[0], st[1], st[2]
    _refuse(t, _F16, name, shape, "heads [B, S, H, dh] with contiguous channels, a")


def _qk_call(name, q, k, gq, gk, positions, pos0, theta, inv_freq, rot, interleaved, eps, out, back=None):
    """Checks the tensors, allocates what is not given and calls rbk_qk_norm_rope_*; returns the two outputs."""
    shape = q.shape
    hq = _heads(q, "q", shape)
    B, S, Hq, dh = shape
    rot = dh if rot is None else rot
    freq = None
    if inv_freq is not None:
        if len(inv_freq) != rot // 2:
            raise ValueError(f"inv_freq: expected {rot // 2} values, got {len(inv_freq)}")
        freq = (C.c_double * max(1, len(inv_freq)))(*[float(x) for x in inv_freq])
    pos = 0 if positions is None else _here(positions, torch.int32, "positions", (B, S))
    pq = 0 if gq is None else _here(gq, _F16, "gq", (dh,))
    pk = 0 if gk is None else _here(gk, _F16, "gk", (dh,))
    if k is None:
        Hk, kshape, hk, ok = 0, None, _NO_HEADS, _NO_HEADS
    else:
        Hk = k.shape[2]
        kshape = (B, S, Hk, dh)
        hk = _heads(k, "k", kshape)
    if out is None:
        # sizes as separate integers: 1.4 us a tensor; torch.empty of a shape, type and device takes 3.1
        oq = q.new_empty(B, S, Hq, dh)
        ok = None if k is None else k.new_empty(B, S, Hk, dh)
        out = oq, ok
        oq = oq.data_ptr(), S * Hq * dh, Hq * dh, dh
        ok = _NO_HEADS if k is None else (ok.data_ptr(), S * Hk * dh, Hk * dh, dh)
    else:
        out = out[0], (None if k is None else out[1])
        oq = _heads(out[0], "out[0]", shape)
        if k is not None:
            ok = _heads(out[1], "out[1]", kshape)
    if back is None:
        tail = _NO_HEADS + _NO_HEADS + (0, 0, 0, 0)
    else:
        dyq, dyk, dgq, dgk, add, ws = back
        tail = (_heads(dyq, "dyq", shape) + (_NO_HEADS if k is None else _heads(dyk, "dyk", kshape))
                + (dgq, dgk, add, ws.data_ptr()))
    call(name, ctx().handle, QK_PACK.pack(B, S, Hq, Hk, dh, rot, bool(interleaved), eps, theta,
                                          C.addressof(freq) if freq else 0, pos, pos0, pq, pk, *hq, *hk, *oq, *ok,
                                          *tail), _s())
    return out


def qk_norm_rope_fwd(q, k, gq=None, gk=None, positions=None, pos0=0, theta=10000.0, inv_freq=None, rot=None,
                     interleaved=False, eps=1e-6, out=None):
    """Per-head RMS norm of queries and keys, then the rotary position embedding (rbk_qk_norm_rope_fwd).

    q [B, S, Hq, dh], k [B, S, Hk, dh] (or None): half, any strides with contiguous channels.  gq, gk: half
    [dh] gains.  positions: int32 [B, S], or None for pos0 + s.  inv_freq: rot / 2 host numbers, or None for
    theta^(-2 i / rot).  rot: leading channels that turn (default dh).  out: (yq, yk), e.g. the q and k blocks of
    the qkv rows that attn_fwd reads, or (q, k) themselves; by default new tensors.  Returns (yq, yk)."""
    return _qk_call("rbk_qk_norm_rope_fwd", q, k, gq, gk, positions, pos0, theta, inv_freq, rot, interleaved, eps, out)


def qk_norm_rope_bwd(dyq, dyk, q, k, gq=None, gk=None, positions=None, pos0=0, theta=10000.0, inv_freq=None,
                     rot=None, interleaved=False, eps=1e-6, out=None, dgq=None, dgk=None):
    """Its backward (rbk_qk_norm_rope_bwd): q, k as the forward read them.  Returns (dq, dk, dgq, dgk); given
    FP32 [dh] dgq, dgk accumulate, else both are new.  out: (dq, dk), may be (dyq, dyk)."""
    dh, add = q.shape[-1], dgq is not None
    if add != (dgk is not None) and k is not None:
        raise ValueError("dgq and dgk: give both or neither")
    if add:
        _here(dgq, _F32, "dgq", (dh,))
        if k is not None:
            _here(dgk, _F32, "dgk", (dh,))
    else:
        dgq = torch.empty(dh, dtype=_F32, device=q.device)
        dgk = None if k is None else torch.empty_like(dgq)
    ws = torch.empty(RBK_QK_BWD_WS_BYTES, dtype=torch.uint8, device=q.device)
    dq, dk = _qk_call("rbk_qk_norm_rope_bwd", q, k, gq, gk, positions, pos0, theta, inv_freq, rot, interleaved, eps, out,
                      (dyq, dyk, dgq.data_ptr(), 0 if k is None else dgk.data_ptr(), add, ws))
    return dq, dk, dgq, (None if k is None else dgk)


# ------------------------------------------------------ gated feed-forward --

ACT_SILU, ACT_GELU = range(2)
_ACTS = {"silu": ACT_SILU, "gelu": ACT_GELU}


def _rows(t, name, shape):
    """Address and row stride of a half [N, D] tensor with contiguous rows."""
    st = t.stride()
    if t.dtype is _F16 and t.shape == shape and t.get_device() == _dev() and (st[1] == 1 or shape[1] == 1):
        return t.data_ptr(), (st[0] if shape[0] > 1 else shape[1])
    _refuse(t, _F16, name, shape, "contiguous rows, a")


def _ffn_ws(handle, N, D, F, back, device):
    """The workspace that the call needs, if any, from torch's allocator (a captured graph keeps its own)."""
    n = lib().rbk_gated_ffn_ws_bytes(handle, N, D, F, back)
    if n < 0:
        raise RbkError(n, "rbk_gated_ffn_ws_bytes", lib().rbk_last_error().decode(errors="replace"))
    if n == 0:
        return None, 0, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def gated_ffn_fwd(x, wgu, wd, bgu=None, bd=None, residual=None, act="silu", save=True, out=None):
    """y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual (rbk_gated_ffn_fwd).

    x [N, D], wgu [2F, D] (gate rows, then up rows), wd [D, F], biases [2F] and [D]: half.  act: "silu" or "gelu"
    (tanh form).  Returns (y, gu, h): gu [N, 2F] the two projections, for gated_ffn_bwd (None with save False),
    and h [N, F] the product.  out: y, may be residual."""
    shape, dev = x.shape, x.device
    N, D = shape
    F = wd.shape[1]
    px, ldx = _rows(x, "x", shape)
    pwgu, pwd = _here(wgu, _F16, "wgu", (2 * F, D)), _here(wd, _F16, "wd", (D, F))
    pbgu = 0 if bgu is None else _here(bgu, _F16, "bgu", (2 * F,))
    pbd = 0 if bd is None else _here(bd, _F16, "bd", (D,))
    pres, ldr = (0, 0) if residual is None else _rows(residual, "residual", shape)
    if out is None:
        y = torch.empty_like(x)                             # contiguous, whatever x's row stride
        py, ldy = y.data_ptr(), D
    else:
        y = out
        py, ldy = _rows(y, "out", shape)
    h = x.new_empty(N, F)
    gu, pgu = None, 0
    if save:
        gu = x.new_empty(N, 2 * F)
        pgu = gu.data_ptr()
    handle = ctx().handle
    # few rows need none: the kernels that stream the weights split nothing
    ws, pws, nws = (None, 0, 0) if N <= 32 else _ffn_ws(handle, N, D, F, 0, dev)
    call("rbk_gated_ffn_fwd", handle, FFN_PACK.pack(N, D, F, _ACTS[act], px, ldx, pwgu, pbgu, pwd, pbd, pres, ldr, py,
                                                    ldy, pgu, h.data_ptr(), pws, nws), _s())
    return y, gu, h


def gated_ffn_bwd(dy, x, gu, wgu, wd, act="silu", h=None, want_dx=True, dwgu=None, dbgu=None, dwd=None, dbd=None,
                  dgu=None, out=None):
    """Its backward (rbk_gated_ffn_bwd) from the saved gu.  h: the forward's, or None to have it computed again.
    dwgu [2F, D], dbgu [2F], dwd [D, F], dbd [D]: FP32, accumulate; those left out are not computed.  dgu: may be gu.
    x: may be None without dwgu, which alone reads it.  out: dx, may be dy or x.  Returns (dx or None, dgu, h)."""
    shape, dev = dy.shape, dy.device
    N, D = shape
    F = wd.shape[1]
    pdy, lddy = _rows(dy, "dy", shape)
    px, ldx = (0, 0) if x is None else _rows(x, "x", shape)
    pgu = _here(gu, _F16, "gu", (N, 2 * F))
    pwgu, pwd = _here(wgu, _F16, "wgu", (2 * F, D)), _here(wd, _F16, "wd", (D, F))
    recompute = h is None
    if recompute:
        h = gu.new_empty(N, F)
        ph = h.data_ptr()
    else:
        ph = _here(h, _F16, "h", (N, F))
    if dgu is None:
        dgu = torch.empty_like(gu)
        pdgu = dgu.data_ptr()
    else:
        pdgu = _here(dgu, _F16, "dgu", (N, 2 * F))
    handle = ctx().handle
    dx, pdx, lddx, ws, pws, nws = None, 0, D, None, 0, 0
    if want_dx:
        if out is None:
            dx = torch.empty_like(dy)                       # contiguous, whatever dy's row stride
            pdx = dx.data_ptr()
        else:
            dx = out
            pdx, lddx = _rows(dx, "out", shape)
        ws, pws, nws = _ffn_ws(handle, N, D, F, 1, dev)
    p1 = 0 if dwgu is None else _here(dwgu, _F32, "dwgu", (2 * F, D))
    p2 = 0 if dbgu is None else _here(dbgu, _F32, "dbgu", (2 * F,))
    p3 = 0 if dwd is None else _here(dwd, _F32, "dwd", (D, F))
    p4 = 0 if dbd is None else _here(dbd, _F32, "dbd", (D,))
    call("rbk_gated_ffn_bwd", handle, FFN_BWD_PACK.pack(N, D, F, _ACTS[act], pdy, lddy, px, ldx, pgu, pwgu, pwd, ph,
                                                        recompute, pdgu, pdx, lddx, p1, p2, p3, p4, pws, nws), _s())
    return dx, dgu, h
