"""rbk_gated_ffn_fwd / _bwd against float64, element by element, within the bounds of ffn_ref.py."""
import pytest

torch = pytest.importorskip("torch")

import ffn_ref as ref   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rbk import ops as o
    torch.cuda.set_device(0)
    return o


def within(name, got, want, bound):
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), f"{name}: off by up to {float(over.max())} more than the bound"


def case(N, D, F, bias=False, res=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * N + D + 7 * F)

    def r(*shape, scale=1.0):
        return (scale * torch.randn(*shape, device="cuda", generator=g)).half()

    return dict(x=r(N, D), wgu=r(2 * F, D, scale=D ** -0.5), wd=r(D, F, scale=F ** -0.5),
                bgu=r(2 * F, scale=0.3) if bias else None, bd=r(D, scale=0.3) if bias else None,
                residual=r(N, D) if res else None, dy=r(N, D))


SIZES = [(1, 8, 8), (1, 64, 128), (2, 72, 24), (7, 520, 40), (8, 256, 264), (9, 64, 1000), (16, 136, 16), (17, 776, 520),
         (31, 8, 2056), (32, 1024, 72), (33, 8, 8), (33, 64, 24), (64, 264, 136), (23, 520, 2504), (10, 264, 2504),
         (47, 776, 2504), (64, 2504, 1256), (50, 1256, 2512), (65, 64, 136), (129, 72, 520), (257, 512, 1032),
         (300, 776, 256), (1000, 136, 2056), (2500, 256, 640)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("N,D,F", SIZES)
def test_forward(ops, N, D, F, act):
    bias, res = N % 2 == 1, F % 16 == 8
    c = case(N, D, F, bias, res)
    want = ref.fwd(c["x"], c["wgu"], c["wd"], c["bgu"], c["bd"], c["residual"], act)
    how = dict(bgu=c["bgu"], bd=c["bd"], residual=c["residual"], act=act)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], **how)
    for name, t in (("gu", gu), ("h", h), ("y", y)):
        within(name, t, *want[name])
    y2, none, h2 = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], save=False, **how)
    assert none is None and torch.equal(y, y2) and torch.equal(h, h2)
    assert ops.device_error() == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("N,D,F", SIZES)
def test_backward(ops, N, D, F, act):
    c = case(N, D, F, seed=1)
    gu = (c["x"].float() @ c["wgu"].float().T).half()
    want = ref.bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act)
    grads = dict(dwgu=torch.zeros(2 * F, D, device="cuda"), dbgu=torch.zeros(2 * F, device="cuda"),
                 dwd=torch.zeros(D, F, device="cuda"), dbd=torch.zeros(D, device="cuda"))
    dx, dgu, h = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act=act, **grads)
    for name, t in dict(grads, dx=dx, dgu=dgu, h=h).items():
        within(name, t, *want[name])
    # the forward's h kept, gradients over the saved activations, nothing else asked for
    over = gu.clone()
    dx2, dgu2, _ = ops.gated_ffn_bwd(c["dy"], c["x"], over, c["wgu"], c["wd"], act=act, h=h, dgu=over)
    assert dgu2 is over and torch.equal(dgu2, dgu) and torch.equal(dx2, dx)
    assert ops.device_error() == 0


# Between few rows and full tiles: rows in one to sixteen blocks of 128, K in one to eight parts, rows of K that start
# on 128 bytes and not, narrow and wide blocks.
MIDDLE = [(34, 8, 8), (66, 768, 2048), (127, 264, 5640), (128, 512, 1024), (129, 1144, 3872), (131, 1448, 992),
          (200, 1024, 2816), (257, 2048, 264), (286, 1192, 2040), (384, 768, 2048), (440, 672, 2088), (513, 400, 3344),
          (630, 1736, 864), (899, 600, 408), (1025, 512, 1024), (1121, 2008, 336), (2047, 72, 264)]


@pytest.mark.parametrize("N,D,F", MIDDLE)
def test_middle_sizes(ops, N, D, F):
    """Against float64; the same bits from a second call, and from dx with and without weight gradients before it."""
    act = "gelu" if N % 2 else "silu"
    c = case(N, D, F, N % 3 == 0, N % 4 < 2, seed=11)
    how = dict(bgu=c["bgu"], bd=c["bd"], residual=c["residual"], act=act)
    want = ref.fwd(c["x"], c["wgu"], c["wd"], c["bgu"], c["bd"], c["residual"], act)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], **how)
    for name, t in (("gu", gu), ("h", h), ("y", y)):
        within(name, t, *want[name])
    again = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], **how)
    assert all(torch.equal(s, t) for s, t in zip(again, (y, gu, h)))
    want = ref.bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act)
    dx, dgu, h = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act=act)
    for name, t in dict(dx=dx, dgu=dgu, h=h).items():
        within(name, t, *want[name])
    dwd = torch.zeros(D, F, device="cuda")
    dx2, dgu2, h2 = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act=act, dwd=dwd)
    assert torch.equal(dx2, dx) and torch.equal(dgu2, dgu) and torch.equal(h2, h)
    within("dwd", dwd, *want["dwd"])
    assert ops.device_error() == 0


def test_middle_sizes_on_two_streams(ops):
    """Calls on two streams at once, whose clusters share the SMs, give what each gives alone."""
    cases = [case(N, D, F, seed=12) for N, D, F in ((300, 768, 2048), (129, 1144, 1000))]
    want = [ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"]) for c in cases]
    back = [ops.gated_ffn_bwd(c["dy"], c["x"], w[1], c["wgu"], c["wd"]) for c, w in zip(cases, want)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for c, w, st in zip(cases, want, streams):
            with torch.cuda.stream(st):
                got.append((ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"]),
                            ops.gated_ffn_bwd(c["dy"], c["x"], w[1], c["wgu"], c["wd"])))
    torch.cuda.synchronize()
    for i, (f, b) in enumerate(got):
        assert all(torch.equal(s, t) for s, t in zip(f + b, want[i % 2] + back[i % 2]))


def test_backward_accumulates_and_reads_the_kept_product(ops):
    N, D, F = 200, 128, 264
    c = case(N, D, F, seed=2)
    gu = (c["x"].float() @ c["wgu"].float().T).half()
    h = torch.randn(N, F, device="cuda").half()            # not the one gu would give: it must be what dwd reads
    dwd = torch.full((D, F), 3.0, device="cuda")
    dx, _, h2 = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], h=h, want_dx=False, dwd=dwd)
    assert dx is None and h2 is h
    want = 3.0 + c["dy"].double().T @ h.double()
    within("dwd", dwd, want, (N + 2) * ref.E * (3.0 + c["dy"].double().abs().T @ h.double().abs()))


@pytest.mark.parametrize("over", ["dy", "x"])
@pytest.mark.parametrize("ws", [False, True])
def test_dx_over_what_is_read_and_the_scratch_of_the_context(ops, over, ws):
    """dx over dy or over x, with the call's own workspace and with the context's scratch, in the deterministic mode
    whose weight gradients use that scratch too."""
    import ctypes as C

    from rbk._lib import FFN_BWD_PACK, call, lib
    N, D, F = 600, 264, 3208
    c = case(N, D, F, seed=6)
    gu = (c["x"].float() @ c["wgu"].float().T).half()
    want = {k: torch.zeros(s, device="cuda") for k, s in (("dwgu", (2 * F, D)), ("dwd", (D, F)))}
    got = {k: torch.zeros_like(v) for k, v in want.items()}
    fresh = ops.Context()                                  # no scratch yet: the first use allocates it
    call("rbk_ctx_set_deterministic", fresh.handle, 1)
    call("rbk_ctx_set_deterministic", ops.ctx().handle, 1)
    dx, dgu, h = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], **want)
    call("rbk_ctx_set_deterministic", ops.ctx().handle, 0)
    t = c[over]
    n = lib().rbk_gated_ffn_ws_bytes(fresh.handle, N, D, F, 1)
    assert n > 0                                           # these sizes share K out
    buf = torch.empty(n, dtype=torch.uint8, device="cuda")
    h2, dgu2 = torch.empty_like(h), torch.empty_like(dgu)
    args = FFN_BWD_PACK.pack(N, D, F, 0, c["dy"].data_ptr(), D, c["x"].data_ptr(), D, gu.data_ptr(), c["wgu"].data_ptr(),
                             c["wd"].data_ptr(), h2.data_ptr(), 1, dgu2.data_ptr(), t.data_ptr(), D,
                             got["dwgu"].data_ptr(), 0, got["dwd"].data_ptr(), 0, buf.data_ptr() if ws else 0,
                             n if ws else 0)
    call("rbk_gated_ffn_bwd", fresh.handle, args, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(t, dx) and torch.equal(h2, h) and torch.equal(dgu2, dgu)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_a_workspace_that_is_too_small_is_refused(ops):
    from rbk._lib import FFN_BWD_PACK, FFN_PACK, lib
    N, D, F = 600, 264, 8712
    c = case(N, D, F, seed=7)
    gu, dgu, dx = (torch.zeros(N, k, device="cuda").half() for k in (2 * F, 2 * F, D))
    y, h, ws = torch.zeros_like(c["x"]), torch.zeros(N, F, device="cuda").half(), torch.zeros(256, device="cuda")
    args = FFN_PACK.pack(N, D, F, 0, c["x"].data_ptr(), D, c["wgu"].data_ptr(), 0, c["wd"].data_ptr(), 0, 0, 0,
                         y.data_ptr(), D, 0, h.data_ptr(), ws.data_ptr(), 256)
    assert lib().rbk_gated_ffn_fwd(ops.ctx().handle, args, None) == -1
    assert b"are needed" in lib().rbk_last_error()
    args = FFN_BWD_PACK.pack(N, D, F, 0, c["dy"].data_ptr(), D, c["x"].data_ptr(), D, gu.data_ptr(), c["wgu"].data_ptr(),
                             c["wd"].data_ptr(), h.data_ptr(), 1, dgu.data_ptr(), dx.data_ptr(), D, 0, 0, 0, 0,
                             ws.data_ptr(), 256)
    assert lib().rbk_gated_ffn_bwd(ops.ctx().handle, args, None) == -1
    assert b"are needed" in lib().rbk_last_error()
    assert not any(bool(t.any()) for t in (y, h, dgu, dx))     # nothing has run


@pytest.mark.parametrize("N", [5, 100])
def test_strides_and_what_lies_beside(ops, N):
    """Row strides of x, residual and y; y over the residual; neighbours of the rows stay as they were."""
    D, F = 136, 72
    c = case(N, D, F, True, True, seed=3)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=c["residual"])
    wide = torch.full((N, D + 24), 9.0, device="cuda", dtype=torch.float16)
    xs, ys = wide.clone()[:, 8:8 + D], wide[:, 16:16 + D]
    xs.copy_(c["x"])
    ys.copy_(c["residual"])
    y2, gu2, h2 = ops.gated_ffn_fwd(xs, c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=ys, out=ys)
    assert y2 is ys and torch.equal(y2, y) and torch.equal(gu2, gu) and torch.equal(h2, h)
    assert bool((wide[:, :16] == 9.0).all()) and bool((wide[:, 16 + D:] == 9.0).all())
    dys = wide.clone()[:, 8:8 + D]
    dys.copy_(c["dy"])
    grads = [dict(dwgu=torch.zeros(2 * F, D, device="cuda"), dwd=torch.zeros(D, F, device="cuda")) for _ in range(2)]
    a = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], **grads[0])
    b = ops.gated_ffn_bwd(dys, xs, gu, c["wgu"], c["wd"], **grads[1])
    assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("N", [1, 31, 47, 65, 255, 257])
def test_rows_behind_the_last_stay(ops, N):
    """y, and through the C entry gu and h, in larger buffers: the rows from N on stay as they were."""
    import ctypes as C

    from rbk._lib import FFN_PACK, call
    D, F = 136, 264
    c = case(N, D, F, seed=8)
    bufs = [torch.full((N + 300, k), 9.0, device="cuda").half() for k in (D, 2 * F, F)]
    args = FFN_PACK.pack(N, D, F, 0, c["x"].data_ptr(), D, c["wgu"].data_ptr(), 0, c["wd"].data_ptr(), 0, 0, 0,
                         bufs[0].data_ptr(), D, bufs[1].data_ptr(), bufs[2].data_ptr(), 0, 0)
    call("rbk_gated_ffn_fwd", ops.ctx().handle, args, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    for got, want in zip(bufs, ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"])):
        assert torch.equal(got[:N], want) and bool((got[N:] == 9.0).all())


@pytest.mark.parametrize("N", [6, 70])
def test_a_row_that_is_not_finite_spoils_itself_only(ops, N):
    D, F = 64, 136
    c = case(N, D, F, seed=4)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"])
    x = c["x"].clone()
    x[2, 5] = float("nan")
    x[4, 0] = float("inf")
    y2, gu2, h2 = ops.gated_ffn_fwd(x, c["wgu"], c["wd"])
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[2] = keep[4] = False
    for a, b in ((y, y2), (gu, gu2), (h, h2)):
        assert torch.equal(a[keep], b[keep]) and not bool(b[~keep].isfinite().all(1).any())


def test_extreme_gates(ops):
    """Pre-activations of FP16's largest size: act(-big) is 0, act(big) is big, their slopes 0 and 1."""
    N, D, F = 3, 8, 16
    x = torch.ones(N, D, device="cuda", dtype=torch.float16)
    wgu = torch.zeros(2 * F, D, device="cuda", dtype=torch.float16)
    wgu[:F // 2, 0], wgu[F // 2:F, 0], wgu[F:, 0] = 60000.0, -60000.0, 0.5
    wd = torch.zeros(D, F, device="cuda", dtype=torch.float16)
    wd[0] = 2.0 ** -6
    dy = torch.ones(N, D, device="cuda", dtype=torch.float16)
    for act in ("silu", "gelu"):
        y, gu, h = ops.gated_ffn_fwd(x, wgu, wd, act=act)
        assert bool((h[:, :F // 2] == 30000).all()) and bool((h[:, F // 2:] == 0).all())
        dx, dgu, h2 = ops.gated_ffn_bwd(dy, x, gu, wgu, wd, act=act)
        assert torch.equal(h, h2)
        d = 2.0 ** -6
        assert bool((dgu[:, :F // 2] == d * 0.5).all()) and bool((dgu[:, F // 2:F] == 0).all())
        assert bool((dgu[:, F:F + F // 2] == d * 60000).all()) and bool((dgu[:, F + F // 2:] == 0).all())


def test_few_rows_need_no_workspace(ops):
    from rbk._lib import lib
    for N in (1, 8, 32):
        for D, F in ((8, 8), (264, 8192), (2048, 5632), (8192, 8192)):
            assert lib().rbk_gated_ffn_ws_bytes(ops.ctx().handle, N, D, F, 0) == 0


def test_no_rows(ops):
    x = torch.empty(0, 64, device="cuda", dtype=torch.float16)
    wgu, wd = torch.ones(256, 64, device="cuda").half(), torch.ones(64, 128, device="cuda").half()
    y, gu, h = ops.gated_ffn_fwd(x, wgu, wd)
    assert y.shape == (0, 64) and gu.shape == (0, 256) and h.shape == (0, 128)
    dw = torch.ones(256, 64, device="cuda")
    dx, dgu, _ = ops.gated_ffn_bwd(x, x, gu, wgu, wd, dwgu=dw)
    assert dx.shape == (0, 64) and bool((dw == 1).all())


@pytest.mark.parametrize("N", [3, 200])
def test_repeats_bits_on_streams_and_in_graphs(ops, N):
    D, F = 256, 520
    c = case(N, D, F, True, True, seed=5)

    def both():
        y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=c["residual"])
        return (y, gu, h) + ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])

    want = both()
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                out = both()
        graphs.append((side, gr, out))
    torch.cuda.synchronize()
    for _ in range(4):
        for side, gr, out in graphs:
            with torch.cuda.stream(side):
                for t in out:
                    t.zero_()
                gr.replay()
    torch.cuda.synchronize()
    for _, _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert ops.device_error() == 0


def test_refused_tensors(ops):
    c = case(4, 64, 128)
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(c["x"].float(), c["wgu"], c["wd"])
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(c["x"], c["wgu"][:128], c["wd"])
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"].T)
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bd=c["x"][0].float())
    with pytest.raises(KeyError):
        ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], act="relu")
    with pytest.raises(RuntimeError, match="multiples of 8"):
        ops.gated_ffn_fwd(c["x"][:, :60], c["wgu"][:, :60].contiguous(), c["wd"][:60].contiguous())


@pytest.mark.parametrize("N,D,F,back", [(100, 768, 2048, False), (100, 768, 2048, True), (300, 256, 2048, False)])
def test_a_wait_that_runs_out(ops, N, D, F, back):
    """Tiles whose loads never complete: the waits give up after 1 ms with every slot's copies issued, the launch returns,
    RBK_ERR_TIMEOUT is reported, and the same call again gives the bits of a call before (backward: a cluster shares
    K out)."""
    from rbk._lib import call
    c = case(N, D, F, seed=13)
    gu = (c["x"].float() @ c["wgu"].float().T).half()

    def once():
        if back:
            return ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])
        return ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"])

    want = once()
    assert ops.device_error() == 0
    call("rbk_ctx_arm_ffn_timeout_test", ops.ctx().handle, 1e-3)
    once()
    assert ops.device_error() == -4                        # RBK_ERR_TIMEOUT
    assert all(torch.equal(a, b) for a, b in zip(once(), want))
    assert ops.device_error() == 0


# The kernels that the sizes above do not reach; with them every kernel that a call can choose runs (a CPU test,
# test_block_ops_host.py, holds these lists against rbk_gated_ffn_plan).
REST = [(7, 2504, 1256), (5, 136, 1192), (12, 2504, 72), (30, 2384, 264), (61, 264, 1496), (48, 768, 2048),
        (40, 1248, 4616), (132, 8, 4856), (140, 456, 5192), (200, 2048, 5632), (392, 8, 4760), (405, 8, 5384),
        (287, 1064, 3952), (526, 1048, 2568), (259, 1032, 4792), (280, 1096, 5256), (264, 1040, 5688), (405, 1064, 4464),
        (131, 1592, 8), (131, 1592, 1032), (521, 1960, 8), (933, 1208, 456), (4285, 72, 3104)]
# Full tiles in the forward and the backward: K of the down projection in 12 parts, in 2 and whole; several tiles a pair
# of CTAs; last tiles of 8 columns and of 128 or 256.
PAIRS = [(600, 264, 8712), (2049, 776, 2056), (4100, 520, 2568), (4097, 776, 2560)]


def full_tiles(ops, N, D, F):
    """The calls of these sizes run on CTA pairs; whether their second products share K out."""
    import ctypes as C

    from rbk._lib import call
    split = []
    for back in (0, 1):
        plan = (C.c_int * 6)()
        call("rbk_gated_ffn_plan", ops.ctx().handle, N, D, F, back, plan)
        assert plan[0] == plan[3] == 2, list(plan)
        split.append(plan[5] > 1)
    return split


@pytest.mark.parametrize("N,D,F", REST)
def test_every_other_kernel(ops, N, D, F):
    act = "gelu" if (N + F // 8) % 2 else "silu"
    c = case(N, D, F, N % 3 != 0, N % 4 < 2, seed=14)
    how = dict(bgu=c["bgu"], bd=c["bd"], residual=c["residual"], act=act)
    want = ref.fwd(c["x"], c["wgu"], c["wd"], c["bgu"], c["bd"], c["residual"], act)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], **how)
    for name, t in (("gu", gu), ("h", h), ("y", y)):
        within(name, t, *want[name])
    y2, _, h2 = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], save=False, **how)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    want = ref.bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act)
    dx, dgu, h = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act=act)
    for name, t in dict(dx=dx, dgu=dgu, h=h).items():
        within(name, t, *want[name])
    assert ops.device_error() == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N,D,F", PAIRS)
def test_full_tiles(ops, N, D, F, bias, act):
    """Everything of a training step against float64, without and with biases and a residual; the same bits without the
    saved projections, with y over the residual, with dgu over gu, with the kept h and without the weights' gradients."""
    split = full_tiles(ops, N, D, F)
    assert split == [F != 2568 and F != 2560] * 2
    c = case(N, D, F, bias, bias, seed=15)
    how = dict(bgu=c["bgu"], bd=c["bd"], act=act)
    want = ref.fwd(c["x"], c["wgu"], c["wd"], c["bgu"], c["bd"], c["residual"], act)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], residual=c["residual"], **how)
    for name, t in (("gu", gu), ("h", h), ("y", y)):
        within(name, t, *want[name])
    over = c["residual"].clone() if bias else torch.empty_like(y)
    y2, none, h2 = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], residual=over if bias else None, save=False, out=over, **how)
    assert y2 is over and none is None and torch.equal(y, y2) and torch.equal(h, h2)
    want = ref.bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act)
    grads = dict(dwgu=torch.zeros(2 * F, D, device="cuda"), dwd=torch.zeros(D, F, device="cuda"))
    if bias:
        grads.update(dbgu=torch.zeros(2 * F, device="cuda"), dbd=torch.zeros(D, device="cuda"))
    dx, dgu, hb = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], act=act, **grads)
    for name, t in dict(grads, dx=dx, dgu=dgu, h=hb).items():
        within(name, t, *want[name])
    over = gu.clone()
    dx2, dgu2, _ = ops.gated_ffn_bwd(c["dy"], c["x"], over, c["wgu"], c["wd"], act=act, h=hb, dgu=over)
    assert dgu2 is over and torch.equal(dgu2, dgu) and torch.equal(dx2, dx)
    assert ops.device_error() == 0


@pytest.mark.parametrize("N,D,F", PAIRS[:2])
def test_full_tiles_rows_that_are_not_finite(ops, N, D, F):
    """A row of x or dy that is not finite spoils itself only."""
    full_tiles(ops, N, D, F)
    c = case(N, D, F, seed=16)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"])
    dx, dgu, _ = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])
    x, dy = c["x"].clone(), c["dy"].clone()
    bad = [0, 77, 255, 256, N - 1]
    x[bad[0::2], 5], x[bad[1::2], 0] = float("nan"), float("inf")
    dy[bad[0::2], 0], dy[bad[1::2], 7] = float("-inf"), float("nan")
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[bad] = False
    for a, b in zip((y, gu, h), ops.gated_ffn_fwd(x, c["wgu"], c["wd"])):
        assert torch.equal(a[keep], b[keep]) and not bool(b[~keep].isfinite().all(1).any())
    dx2, dgu2, _ = ops.gated_ffn_bwd(dy, c["x"], gu, c["wgu"], c["wd"])
    for a, b in ((dx, dx2), (dgu, dgu2)):
        assert torch.equal(a[keep], b[keep]) and not bool(b[~keep].isfinite().all(1).any())


def test_full_tiles_extreme_gates(ops):
    """test_extreme_gates on CTA pairs: gates of FP16's largest size, half of the columns each way."""
    N, D, F = PAIRS[0]
    full_tiles(ops, N, D, F)
    x = torch.ones(N, D, device="cuda", dtype=torch.float16)
    wgu = torch.zeros(2 * F, D, device="cuda", dtype=torch.float16)
    wgu[:F // 2, 0], wgu[F // 2:F, 0], wgu[F:, 0] = 60000.0, -60000.0, 0.5
    wd = torch.zeros(D, F, device="cuda", dtype=torch.float16)
    wd[0] = 2.0 ** -6
    dy = torch.ones(N, D, device="cuda", dtype=torch.float16)
    for act in ("silu", "gelu"):
        _, gu, h = ops.gated_ffn_fwd(x, wgu, wd, act=act)
        assert bool((h[:, :F // 2] == 30000).all()) and bool((h[:, F // 2:] == 0).all())
        _, dgu, h2 = ops.gated_ffn_bwd(dy, x, gu, wgu, wd, act=act)
        assert torch.equal(h, h2)
        d = 2.0 ** -6
        assert bool((dgu[:, :F // 2] == d * 0.5).all()) and bool((dgu[:, F // 2:F] == 0).all())
        assert bool((dgu[:, F:F + F // 2] == d * 60000).all()) and bool((dgu[:, F + F // 2:] == 0).all())


def test_full_tiles_rows_behind_the_last_stay(ops):
    """Through the C entry: the rows of y, gu, h, dgu and dx from N on stay as they were."""
    import ctypes as C

    from rbk._lib import FFN_BWD_PACK, FFN_PACK, call
    N, D, F = PAIRS[1]
    full_tiles(ops, N, D, F)
    c = case(N, D, F, seed=17)
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    y, gu, h, dgu, dx, hb = [torch.full((N + 300, k), 9.0, device="cuda").half() for k in (D, 2 * F, F, 2 * F, D, F)]
    call("rbk_gated_ffn_fwd", ops.ctx().handle, FFN_PACK.pack(
        N, D, F, 1, c["x"].data_ptr(), D, c["wgu"].data_ptr(), 0, c["wd"].data_ptr(), 0, 0, 0, y.data_ptr(), D,
        gu.data_ptr(), h.data_ptr(), 0, 0), st)
    call("rbk_gated_ffn_bwd", ops.ctx().handle, FFN_BWD_PACK.pack(
        N, D, F, 1, c["dy"].data_ptr(), D, c["x"].data_ptr(), D, gu.data_ptr(), c["wgu"].data_ptr(), c["wd"].data_ptr(),
        hb.data_ptr(), 1, dgu.data_ptr(), dx.data_ptr(), D, 0, 0, 0, 0, 0, 0), st)
    want = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], act="gelu")
    back = ops.gated_ffn_bwd(c["dy"], c["x"], want[1], c["wgu"], c["wd"], act="gelu")
    for got, w in zip((y, gu, h, dx, dgu, hb), want + back):
        assert torch.equal(got[:N], w) and bool((got[N:] == 9.0).all())


def test_full_tiles_in_graphs(ops):
    """Two captured graphs replayed at the same time give the bits of the calls."""
    N, D, F = PAIRS[0]
    c = case(N, D, F, True, True, seed=18)

    def both():
        y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=c["residual"])
        return (y, gu, h) + ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])

    want = both()
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                out = both()
        graphs.append((side, gr, out))
    torch.cuda.synchronize()
    for _ in range(4):
        for side, gr, out in graphs:
            with torch.cuda.stream(side):
                for t in out:
                    t.zero_()
                gr.replay()
    torch.cuda.synchronize()
    for _, _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert ops.device_error() == 0


@pytest.mark.parametrize("N", [5, 100, 2100])
def test_backward_without_x_and_into_given_rows(ops, N):
    """dx and dgu need no x; dx may go over dy or x, with weight gradients too, or into rows of its own stride."""
    D, F = 136, 2056
    c = case(N, D, F, seed=19)
    gu = (c["x"].float() @ c["wgu"].float().T).half()
    grads = [dict(dwgu=torch.zeros(2 * F, D, device="cuda"), dwd=torch.zeros(D, F, device="cuda")) for _ in range(3)]
    dx, dgu, h = ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"], **grads[0])
    dx2, dgu2, h2 = ops.gated_ffn_bwd(c["dy"], None, gu, c["wgu"], c["wd"])
    assert torch.equal(dx, dx2) and torch.equal(dgu, dgu2) and torch.equal(h, h2)
    for i, over in ((1, "dy"), (2, "x")):
        t = {k: c[k].clone() for k in ("dy", "x")}
        dx3, _, _ = ops.gated_ffn_bwd(t["dy"], t["x"], gu, c["wgu"], c["wd"], out=t[over], **grads[i])
        assert dx3 is t[over] and torch.equal(dx3, dx)
        # FP32 additions in another order where K is shared out: twice the bound of one sum
        for k, a, b in (("dwgu", dgu, c["x"]), ("dwd", c["dy"], h)):
            lim = 2 * (N + 1) * ref.E * (a.double().abs().T @ b.double().abs())
            assert bool(((grads[i][k] - grads[0][k]).double().abs() <= lim).all())
    wide = torch.full((N, D + 24), 9.0, device="cuda", dtype=torch.float16)
    ops.gated_ffn_bwd(c["dy"], None, gu, c["wgu"], c["wd"], out=wide[:, 8:8 + D])
    assert torch.equal(wide[:, 8:8 + D], dx) and bool((wide[:, :8] == 9).all()) and bool((wide[:, 8 + D:] == 9).all())
    with pytest.raises(RuntimeError, match="x is NULL"):
        ops.gated_ffn_bwd(c["dy"], None, gu, c["wgu"], c["wd"], dwgu=grads[0]["dwgu"])


def test_offsets_beyond_32_bits(ops):
    """gate | up, h and dgu of more than 2^31 elements: the last rows are right, forward and backward."""
    N, D, F = 1100000, 64, 2056
    g = torch.Generator(device="cuda").manual_seed(20)
    c = dict(wgu=(torch.randn(2 * F, D, device="cuda", generator=g) * D ** -0.5).half(),
             wd=(torch.randn(D, F, device="cuda", generator=g) * F ** -0.5).half(),
             x=torch.randn(N, D, device="cuda", generator=g).half(), dy=torch.randn(N, D, device="cuda", generator=g).half())
    full_tiles(ops, N, D, F)
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"])
    assert h.numel() > 2 ** 31
    for rows in (slice(0, 200), slice(N - 300, N)):
        want = ref.fwd(c["x"][rows], c["wgu"], c["wd"], None, None, None, "silu")
        for name, t in (("gu", gu), ("h", h), ("y", y)):
            within(name, t[rows], *want[name])
    dx, dgu, h2 = ops.gated_ffn_bwd(c["dy"], None, gu, c["wgu"], c["wd"])
    for rows in (slice(0, 200), slice(N - 300, N)):
        want = ref.bwd(c["dy"][rows], c["x"][rows], gu[rows], c["wgu"], c["wd"], "silu")
        for name, t in (("dgu", dgu), ("h", h2), ("dx", dx)):
            within(name, t[rows], *want[name])
    assert ops.device_error() == 0
    del gu, h, dgu, h2
    torch.cuda.empty_cache()


def test_full_tiles_from_threads(ops):
    """Four host threads with their own contexts and streams, whose first calls of the pair kernels may meet."""
    import threading
    N, D, F = PAIRS[0]
    full_tiles(ops, N, D, F)
    c = case(N, D, F, True, True, seed=21)
    got, wrong = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=c["residual"])
                    got[i] = (y, gu, h) + ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                             # a thread's exception is not pytest's
            wrong.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    y, gu, h = ops.gated_ffn_fwd(c["x"], c["wgu"], c["wd"], bgu=c["bgu"], bd=c["bd"], residual=c["residual"])
    want = (y, gu, h) + ops.gated_ffn_bwd(c["dy"], c["x"], gu, c["wgu"], c["wd"])
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
