"""A gated decoder block put together from the operators, as a trainer and a decoder use them.

    h1 = LN(x);  q, k = qk_norm_rope(h1 Wqk);  v = h1 Wv;  x1 = x + attention(q, k, v) Wo
    h2 = LN(x1);  y = x1 + gated_ffn(h2)
    loss = sum(y * target);  gradients;  clip by their global norm;  rbk_adam_tail

compared with torch autograd in float64 on the same FP16 weights and inputs.  Tolerance (relative L2): every
tensor between two operators is rounded to FP16 once, by at most 2^-11; a value passes at most 16 such
roundings on the way to y and 32 on the way to a gradient: 16 * 2^-11 and 32 * 2^-11.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

B, S, H, DH, F = 2, 128, 4, 64, 520
D, N = H * DH, B * S
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    from rbk import ops as o
    torch.cuda.set_device(0)
    return o


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, scale):
        return (scale * torch.randn(*shape, device="cuda", generator=g)).half()

    w = dict(ln1=1 + r(D, scale=0.1), ln1b=r(D, scale=0.1), ln2=1 + r(D, scale=0.1), ln2b=r(D, scale=0.1),
             wqk=r(2 * D, D, scale=D ** -0.5), wv=r(D, D, scale=D ** -0.5), wo=r(D, D, scale=D ** -0.5),
             gq=1 + r(DH, scale=0.1), gk=1 + r(DH, scale=0.1), wgu=r(2 * F, D, scale=D ** -0.5),
             wd=r(D, F, scale=F ** -0.5))
    return w, r(N, D, scale=1.0), r(N, D, scale=1.0)


def forward(ops, w, x):
    """The block's forward; everything that its backward reads."""
    s = {}
    s["h1"], s["m1"], s["r1"] = ops.ln_fwd(x, w["ln1"], w["ln1b"])
    s["qk"] = ops.linear_fwd(s["h1"], w["wqk"]).view(B, S, 2 * H, DH)
    qkv = torch.empty(B, S, 3 * H, DH, device="cuda", dtype=torch.float16)
    # the values go straight to their block of the attention's rows, the queries and keys next to them
    ops.gemm(s["h1"], w["wv"], N, D, D, C_out=qkv.view(N, 3 * D)[:, 2 * D:], ldc=3 * D)
    ops.qk_norm_rope_fwd(s["qk"][:, :, :H], s["qk"][:, :, H:], w["gq"], w["gk"], out=(qkv[:, :, :H], qkv[:, :, H:2 * H]))
    s["qkv"] = qkv.view(N, 3 * D)
    s["o"], s["lse"] = ops.attn_fwd(s["qkv"], B, S, H, DH)
    s["x1"] = ops.linear_fwd(s["o"], w["wo"], residual=x)
    s["h2"], s["m2"], s["r2"] = ops.ln_fwd(s["x1"], w["ln2"], w["ln2b"])
    s["y"], s["gu"], s["h"] = ops.gated_ffn_fwd(s["h2"], w["wgu"], w["wd"], residual=s["x1"])
    return s


def backward(ops, w, x, s, dy, g):
    """Adds the block's gradients to the FP32 tensors g; returns dx."""
    dh2, _, _ = ops.gated_ffn_bwd(dy, s["h2"], s["gu"], w["wgu"], w["wd"], h=s["h"], dwgu=g["wgu"], dwd=g["wd"])
    dx1, _, _, _ = ops.ln_bwd(dh2, s["x1"], w["ln2"], s["m2"], s["r2"], dres=dy, dgamma=g["ln2"], dbeta=g["ln2b"])
    ops.gemm_wgrad(dx1, s["o"], g["wo"])
    do = ops.gemm_dgrad(dx1, w["wo"])
    dqkv = ops.attn_bwd(s["qkv"], s["o"], do, s["lse"], B, S, H, DH)
    d = dqkv.view(B, S, 3 * H, DH)
    dqk = torch.empty(B, S, 2 * H, DH, device="cuda", dtype=torch.float16)
    ops.qk_norm_rope_bwd(d[:, :, :H], d[:, :, H:2 * H], s["qk"][:, :, :H], s["qk"][:, :, H:], w["gq"], w["gk"],
                         out=(dqk[:, :, :H], dqk[:, :, H:]), dgq=g["gq"], dgk=g["gk"])
    dqk, dv = dqk.view(N, 2 * D), dqkv[:, 2 * D:].contiguous()
    ops.gemm_wgrad(dqk, s["h1"], g["wqk"])
    ops.gemm_wgrad(dv, s["h1"], g["wv"])
    dh1 = ops.gemm_dgrad(dqk, w["wqk"]) + ops.gemm_dgrad(dv, w["wv"])
    return ops.ln_bwd(dh1, x, w["ln1"], s["m1"], s["r1"], dres=dx1, dgamma=g["ln1"], dbeta=g["ln1b"])[0]


def reference(w, x):
    """The same block in float64."""
    def norm(t, a, b):
        t = t - t.mean(-1, keepdim=True)
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * a + b

    def heads(t, gain):
        t = t.view(B, S, H, DH)
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * gain
        i = torch.arange(DH // 2, device="cuda", dtype=torch.float64)
        a = (torch.arange(S, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / DH))[:, None]
        u, v = t[..., :DH // 2], t[..., DH // 2:]
        return torch.cat((u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()), -1).transpose(1, 2)

    h1 = norm(x, w["ln1"], w["ln1b"])
    qk = h1 @ w["wqk"].T
    q, k = heads(qk[:, :D], w["gq"]), heads(qk[:, D:], w["gk"])
    v = (h1 @ w["wv"].T).view(B, S, H, DH).transpose(1, 2)
    sc = q @ k.transpose(2, 3) * DH ** -0.5
    sc = sc.masked_fill(torch.ones(S, S, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
    o = (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(N, D)
    x1 = x + o @ w["wo"].T
    z = norm(x1, w["ln2"], w["ln2b"]) @ w["wgu"].T
    g, u = z.chunk(2, -1)
    return x1 + (g * torch.sigmoid(g) * u) @ w["wd"].T


def test_block_forward_and_gradients(ops):
    w, x, target = weights()
    s = forward(ops, w, x)
    w64 = {k: v.double().requires_grad_() for k, v in w.items()}
    x64 = x.double().requires_grad_()
    y64 = reference(w64, x64)
    assert rel(s["y"], y64.detach()) < 16 * 2.0 ** -11
    (y64 * target.double()).sum().backward()
    g = {k: torch.zeros(v.shape, device="cuda") for k, v in w.items()}
    dx = backward(ops, w, x, s, target, g)
    assert rel(dx, x64.grad) < 32 * 2.0 ** -11
    for k in g:
        assert rel(g[k], w64[k].grad) < 32 * 2.0 ** -11, k
    assert ops.device_error() == 0


def test_block_training_step_with_global_clipping(ops):
    """Loss-scaled gradients of separate tensors, clipped together, then the fused tail on the arena they share."""
    w, x, target = weights(1)
    scale, max_norm = 64.0, 0.25
    names = list(w)
    size = {k: (w[k].numel() + 63) // 64 * 64 for k in names}
    n = sum(size.values())
    p32, m, v, grad = (torch.zeros(n, device="cuda") for _ in range(4))
    p16 = torch.zeros(n, device="cuda", dtype=torch.float16)
    at, views, g = 0, {}, {}
    for k in names:
        views[k] = p16[at:at + w[k].numel()].view(w[k].shape)
        views[k].copy_(w[k])
        g[k] = grad[at:at + w[k].numel()].view(w[k].shape)
        at += size[k]
    p32.copy_(p16)
    sc = ops.new_scaler(scale=scale)
    s = forward(ops, views, x)
    backward(ops, views, x, s, (target * (scale / N)).half(), g)
    before = grad.clone()
    norm = ops.clip_grad_norm([g[k] for k in names], max_norm, scaler=sc)
    want = float(before.double().norm()) / scale
    assert abs(float(norm) - want) < 1e-6 * want and want > max_norm
    assert rel(grad, before.double() * (max_norm / want)) < 2.0 ** -22
    ops.adam_tail(p32, grad, m, v, p16, sc, lr=1e-3)
    assert rel(m, 0.1 * before.double() / scale * (max_norm / want)) < 2.0 ** -20
    assert bool((grad == 0).all()) and ops.read_scaler(sc).applied_steps == 1
    y = forward(ops, views, x)["y"]                        # the tail's FP16 weights are the ones that run
    assert bool(y.isfinite().all()) and not torch.equal(y, s["y"])


def test_block_rows_one_at_a_time(ops):
    """Decoding: each row by itself, through the kernels for few rows and with its own position, gives the row of the
    whole sequence (both are right to FP16's rounding of the same value, and h is rounded in between: 3 * 2^-11)."""
    w, x, _ = weights(2)
    s = forward(ops, w, x)
    for n in (0, 1, 77, 200, 255):
        pos = torch.tensor([[n % S]], device="cuda", dtype=torch.int32)
        row = s["qk"].view(N, 1, 2 * H, DH)[n:n + 1]
        yq, yk = ops.qk_norm_rope_fwd(row[:, :, :H], row[:, :, H:], w["gq"], w["gk"], positions=pos)
        qkv = s["qkv"].view(N, 3 * H, DH)[n]
        assert torch.equal(yq[0, 0], qkv[:H]) and torch.equal(yk[0, 0], qkv[H:2 * H])
        y, _, _ = ops.gated_ffn_fwd(s["h2"][n:n + 1], w["wgu"], w["wd"], residual=s["x1"][n:n + 1], save=False)
        assert rel(y, s["y"][n:n + 1]) < 3 * 2.0 ** -11


def test_threads_with_their_own_streams(ops):
    """Four host threads, each with its own context and stream, run the operators at once: every one gets the bits of a
    run by itself."""
    import threading
    w, x, _ = weights(3)
    s = forward(ops, w, x)
    q, k = s["qk"][:, :, :H], s["qk"][:, :, H:]
    dyq, dyk = (torch.randn(B, S, H, DH, device="cuda").half() for _ in range(2))
    grads = [torch.randn(n, device="cuda") for n in (100003, 7, 40000)]

    def run():
        out = [*ops.qk_norm_rope_fwd(q, k, w["gq"], w["gk"]), *ops.qk_norm_rope_bwd(dyq, dyk, q, k, w["gq"], w["gk"])]
        for n in (3, N):
            out += ops.gated_ffn_fwd(s["h2"][:n], w["wgu"], w["wd"], residual=s["x1"][:n])
        out += ops.gated_ffn_bwd(x, s["h2"], s["gu"], w["wgu"], w["wd"])
        clipped = [torch.empty_like(g) for g in grads]
        return out + [ops.clip_grad_norm(grads, 1.0, out=clipped)] + clipped

    want = run()
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = run()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(i)
        except Exception as e:                             # a thread's exception is not pytest's
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
