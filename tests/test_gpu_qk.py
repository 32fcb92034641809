"""rbk_qk_norm_rope_fwd / _bwd against float64.

Tolerances, in steps e = 2^-24 of FP32 (a rounding is off by at most e relatively):
  y: the row's sum of squares has at most 16 + 4 sequential additions of positive terms and one rounding
  each, 21 e, halved by the root; mean, eps and rsqrtf (2 ulp = 4 e) 6 e; two products 2 e; the angle is
  right to 2^-26 turns = 1.6 e, cosine and sine to 2 ulp = 4 e; products and sum of the rotation 3 e: below
  32 e = 2^-19 of |a| + |b|.  Then one FP16 rounding: 2^-11 of the value (2^-25 among the subnormals).
  dx: the same for d, and for the mean of w xhat at most 20 additions more: below 64 e = 2^-18 of
  rstd (|w| + |xhat| mean |w xhat|), and the FP16 rounding.
  dgain: at most one addition per row and head in sequence, and 64 e of the terms: (64 + rows) e of the sum
  of |d xhat|.
"""
import pytest

torch = pytest.importorskip("torch")

import qk_ref as ref   # noqa: E402

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    from rbk import ops as o
    torch.cuda.set_device(0)
    return o


def heads(g, B, S, H, dh, layout, scale=1.0):
    """Random half heads [B, S, H, dh]: "rows" one tensor, "fused" a column block of wider rows, "planes" [B, H, S, dh]."""
    def r(*shape):
        return (scale * torch.randn(*shape, device="cuda", generator=g)).half()
    if layout == "rows":
        return r(B, S, H, dh)
    if layout == "fused":
        return r(B, S, H + 3, dh)[:, :, 2:H + 2]
    return r(B, H, S, dh).transpose(1, 2)


def close_f16(got, want, size, steps):
    lim = 2.0 ** -11 * want.abs() + 2.0 ** -25 + steps * E * size
    over = (got.double() - want).abs() - lim
    assert bool((over <= 0).all()), f"off by up to {float(over.max())} more than the bound"


# B, S, Hq, Hk, dh, rot, interleaved, layout, positions
CASES = [
    (1, 1, 1, 1, 8, 8, True, "rows", "seq"),
    (1, 1, 16, 16, 128, 128, False, "rows", "far"),
    (2, 5, 3, 1, 16, 16, False, "rows", "seq"),
    (3, 7, 4, 2, 24, 16, False, "fused", "far"),
    (2, 9, 5, 5, 24, 8, True, "planes", "seq"),
    (2, 33, 12, 12, 64, 64, False, "fused", "seq"),
    (1, 130, 33, 3, 64, 32, True, "rows", "far"),
    (4, 3, 7, 7, 72, 72, True, "planes", "far"),
    (2, 19, 6, 2, 80, 32, False, "fused", "edge"),
    (2, 19, 6, 2, 80, 80, False, "planes", "seq"),
    (1, 67, 10, 1, 128, 0, False, "rows", "seq"),
    (3, 21, 9, 3, 128, 96, True, "fused", "edge"),
    (2, 11, 4, 4, 200, 192, False, "rows", "far"),
    (2, 40, 3, 2, 256, 256, False, "fused", "edge"),
    (2, 40, 2, 3, 256, 248, True, "planes", "far"),
    (3, 1500, 8, 4, 64, 64, False, "fused", "far"),
    (2, 2000, 5, 5, 128, 128, True, "rows", "seq"),
    (7, 31, 2, 0, 64, 64, False, "rows", "seq"),
    (3, 401, 3, 3, 80, 80, False, "fused", "far"),
    (2, 333, 7, 5, 40, 40, True, "planes", "far"),
    (5, 97, 11, 2, 48, 48, False, "rows", "seq"),
    (1, 700, 6, 6, 96, 64, False, "rows", "far"),
    (2, 150, 5, 3, 88, 88, True, "fused", "edge"),
    (3, 55, 4, 1, 136, 128, False, "planes", "far"),
    (2, 123, 7, 7, 152, 152, True, "rows", "seq"),
    (1, 64, 3, 2, 160, 160, False, "fused", "seq"),
    (4, 37, 8, 8, 104, 96, False, "rows", "far"),
]


def case(B, S, Hq, Hk, dh, rot, inter, layout, pos, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 131 * dh + S)
    q = heads(g, B, S, Hq, dh, layout)
    k = heads(g, B, S, Hk, dh, layout, 3.0) if Hk else None
    gq = (1 + 0.2 * torch.randn(dh, device="cuda", generator=g)).half()
    gk = (1 + 0.2 * torch.randn(dh, device="cuda", generator=g)).half()
    dyq = heads(g, B, S, Hq, dh, layout)
    dyk = heads(g, B, S, Hk, dh, layout) if Hk else None
    positions = None
    if pos == "far":
        positions = torch.randint(0, 1 << 20, (B, S), device="cuda", generator=g, dtype=torch.int32)
    elif pos == "edge":
        positions = torch.randint(-5, 5, (B, S), device="cuda", generator=g, dtype=torch.int32)
        positions.view(-1)[0::3] = 2 ** 31 - 1
        positions.view(-1)[1::3] = -(2 ** 31)
    return q, k, gq, gk, dyq, dyk, positions


@pytest.mark.parametrize("c", CASES, ids=lambda c: "x".join(str(v) for v in c))
def test_fwd_and_bwd(ops, c):
    B, S, Hq, Hk, dh, rot, inter, layout, pos = c
    q, k, gq, gk, dyq, dyk, positions = case(*c)
    how = dict(positions=positions, pos0=17, theta=10000.0, rot=rot, interleaved=inter, eps=EPS)
    ang = ref.angles(B, S, rot, 10000.0, positions, 17)
    yq, yk = ops.qk_norm_rope_fwd(q, k, gq, gk if Hk else None, **how)
    dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(dyq, dyk, q, k, gq, gk if Hk else None, **how)
    for x, gain, y, dy, dx, dg in ((q, gq, yq, dyq, dq, dgq), (k, gk, yk, dyk, dk, dgk)):
        if x is None:
            assert y is None and dx is None and dg is None
            continue
        want, m = ref.fwd(x, gain, ang, rot, inter, EPS)
        close_f16(y, want, m, 32)
        wdx, wdg, mx, mg = ref.bwd(dy, x, gain, ang, rot, inter, EPS)
        close_f16(dx, wdx, mx, 64)
        assert bool(((dg.double() - wdg).abs() <= (64 + B * S * x.shape[2]) * E * mg).all())


def test_no_gain_own_frequencies_and_accumulation(ops):
    B, S, H, dh, rot = 2, 37, 4, 64, 32
    q, k, _, _, dyq, dyk, _ = case(B, S, H, H, dh, rot, False, "rows", "seq", 3)
    freq = [0.7 ** i * (-1) ** i * 2.5 for i in range(rot // 2)]
    how = dict(rot=rot, inv_freq=freq, pos0=1000, eps=1e-5)
    ang = ref.angles(B, S, rot, 0.0, None, 1000, freq)
    yq, yk = ops.qk_norm_rope_fwd(q, k, **how)
    for x, y in ((q, yq), (k, yk)):
        want, m = ref.fwd(x, None, ang, rot, False, 1e-5)
        close_f16(y, want, m, 32)
    dgq, dgk = torch.full((dh,), 100.0, device="cuda"), torch.full((dh,), -7.0, device="cuda")
    a, b = dgq.clone(), dgk.clone()
    ops.qk_norm_rope_bwd(dyq, dyk, q, k, dgq=a, dgk=b, **how)
    _, _, nq, nk = ops.qk_norm_rope_bwd(dyq, dyk, q, k, **how)
    assert torch.equal(a, dgq + nq) and torch.equal(b, dgk + nk)


def test_the_last_positions(ops):
    """Batched rows that end at position 2^31 - 1, counted from pos0, give the bits of the same positions listed."""
    B, S, H, dh = 33, 3, 2, 64
    q, k, gq, gk, dyq, dyk, _ = case(B, S, H, H, dh, dh, False, "rows", "seq", 4)
    pos0 = 2 ** 31 - S
    positions = (pos0 + torch.arange(S)).to(torch.int32).cuda().expand(B, S).contiguous()
    for a, b in zip(ops.qk_norm_rope_fwd(q, k, gq, gk, pos0=pos0),
                    ops.qk_norm_rope_fwd(q, k, gq, gk, positions=positions)):
        assert torch.equal(a, b)
    with pytest.raises(Exception, match="positions beyond"):
        ops.qk_norm_rope_fwd(q, k, gq, gk, pos0=pos0 + 1)


def test_one_gain_for_queries_and_keys(ops):
    B, S, dh = 2, 90, 64
    q, k, g, _, dyq, dyk, _ = case(B, S, 6, 2, dh, dh, False, "rows", "seq", 9)
    _, _, a, b = ops.qk_norm_rope_bwd(dyq, dyk, q, k, g, g)
    both = torch.full((dh,), 5.0, device="cuda")
    ops.qk_norm_rope_bwd(dyq, dyk, q, k, g, g, dgq=both, dgk=both)
    _, _, _, mq = ref.bwd(dyq, q, g, ref.angles(B, S, dh, 10000.0), dh, False, EPS)
    _, _, _, mk = ref.bwd(dyk, k, g, ref.angles(B, S, dh, 10000.0), dh, False, EPS)
    # the same terms in another order
    assert bool(((both - 5.0 - (a + b)).abs() <= (64 + B * S * 8) * E * (mq + mk + 5.0)).all())


def test_in_place_and_into_attention_rows(ops):
    """y over x gives the bits of y apart, and a qkv row's value block and its neighbours stay as they were."""
    B, S, H, dh = 2, 50, 6, 64
    q, k, gq, gk, dyq, dyk, _ = case(B, S, H, H, dh, dh, False, "rows", "seq", 5)
    yq, yk = ops.qk_norm_rope_fwd(q, k, gq, gk)
    qkv = torch.full((B, S, 3 * H, dh), 7.0, device="cuda", dtype=torch.float16)
    ops.qk_norm_rope_fwd(q, k, gq, gk, out=(qkv[:, :, :H], qkv[:, :, H:2 * H]))
    assert torch.equal(qkv[:, :, :H], yq) and torch.equal(qkv[:, :, H:2 * H], yk)
    assert bool((qkv[:, :, 2 * H:] == 7.0).all())
    dq, dk, _, _ = ops.qk_norm_rope_bwd(dyq, dyk, q, k, gq, gk)
    d1, d2 = dyq.clone(), dyk.clone()
    ops.qk_norm_rope_bwd(d1, d2, q, k, gq, gk, out=(d1, d2))
    assert torch.equal(d1, dq) and torch.equal(d2, dk)
    q1, k1 = q.clone(), k.clone()
    ops.qk_norm_rope_fwd(q1, k1, gq, gk, out=(q1, k1))
    assert torch.equal(q1, yq) and torch.equal(k1, yk)


def test_zero_rows_and_what_is_not_finite(ops):
    """A head of zeros gives zeros and finite gradients; a head with an infinity or a NaN spoils itself only."""
    B, S, H, dh, rot = 1, 9, 4, 64, 32
    q, k, gq, gk, dyq, dyk, _ = case(B, S, H, H, dh, rot, False, "rows", "seq", 7)
    clean, _ = ops.qk_norm_rope_fwd(q, k, gq, gk, rot=rot)
    q = q.clone()
    q[0, 3, 1] = 0
    q[0, 5, 2, 7] = float("inf")
    q[0, 6, 0, 63] = float("nan")
    yq, _ = ops.qk_norm_rope_fwd(q, k, gq, gk, rot=rot)
    assert bool((yq[0, 3, 1] == 0).all())
    spoilt = torch.zeros(B, S, H, dtype=torch.bool, device="cuda")
    spoilt[0, 5, 2] = spoilt[0, 6, 0] = True
    same = ~spoilt
    same[0, 3, 1] = False
    assert torch.equal(yq[same], clean[same])
    # the infinity's own channel and its rotated partner are not numbers; the row's other channels are x / inf = 0
    row = yq[0, 5, 2]
    bad = torch.zeros(dh, dtype=torch.bool, device="cuda")
    bad[7] = bad[7 + rot // 2] = True
    assert bool(row[bad].isnan().all()) and bool((row[~bad] == 0).all())
    assert bool(yq[0, 6, 0].isnan().all())
    dq, _, _, _ = ops.qk_norm_rope_bwd(dyq, dyk, q, k, gq, gk, rot=rot)
    assert bool(dq[~spoilt].isfinite().all())


@pytest.mark.parametrize("B,S", [(0, 4), (3, 0)])
def test_no_tokens(ops, B, S):
    q = torch.empty(B, S, 2, 64, device="cuda", dtype=torch.float16)
    yq, yk = ops.qk_norm_rope_fwd(q, q)
    assert yq.shape == q.shape and yk.shape == q.shape
    _, _, dgq, dgk = ops.qk_norm_rope_bwd(q, q, q, q)
    assert bool((dgq == 0).all()) and bool((dgk == 0).all())


def test_offsets_beyond_32_bits(ops):
    """Two tokens of one sequence 2^31 elements apart."""
    far = 2 ** 31 + 64
    buf = torch.zeros(far + 128, device="cuda", dtype=torch.float16)
    x = torch.randn(2, 64, device="cuda").half()
    buf[:64], buf[far:far + 64] = x[0], x[1]
    q = torch.as_strided(buf, (1, 2, 1, 64), (0, far, 64, 1))
    y, _ = ops.qk_norm_rope_fwd(q, None)
    want, _ = ops.qk_norm_rope_fwd(x.view(1, 2, 1, 64), None)
    assert torch.equal(y, want)
    ops.qk_norm_rope_fwd(q, None, out=(q, None))
    assert torch.equal(buf[far:far + 64], want[0, 1, 0]) and bool((buf[64:far] == 0).all())


def test_repeats_bits_on_streams_and_in_graphs(ops):
    """The same bits again, on another stream, and from two graphs replayed at the same time."""
    c = (4, 300, 6, 3, 64, 64, False, "rows", "far")
    q, k, gq, gk, dyq, dyk, positions = case(*c, seed=11)

    def both():
        return ops.qk_norm_rope_fwd(q, k, gq, gk, positions) + ops.qk_norm_rope_bwd(dyq, dyk, q, k, gq, gk, positions)

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
    for _ in range(5):
        for side, gr, out in graphs:
            with torch.cuda.stream(side):
                for t in out:
                    t.zero_()
                gr.replay()
    torch.cuda.synchronize()
    for _, _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refused_tensors(ops):
    q = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q.float(), q)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q, q.cpu())
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q, q[:, :3])
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q.transpose(2, 3), None)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q, q, positions=torch.zeros(1, 4, device="cuda", dtype=torch.int64))
    with pytest.raises(RuntimeError, match="zero stride"):
        ops.qk_norm_rope_fwd(q, None, out=(q[:, :1].expand(1, 4, 2, 64), None))
    with pytest.raises(RuntimeError, match="rot"):
        ops.qk_norm_rope_fwd(q, None, rot=24)


def test_strides_of_axes_of_size_one(ops):
    """Nothing is read by the stride of an axis of size 1, so any will do: torch gives such axes what it likes."""
    x = torch.randn(3, 64, device="cuda").half()
    g = (1 + torch.randn(64, device="cuda")).half()
    for shape, rows in (((1, 3, 1, 64), (0, 64, 0)), ((1, 1, 3, 64), (0, 0, 64)), ((3, 1, 1, 64), (64, 0, 0))):
        strides = [s if n > 1 else 13 for s, n in zip(rows, shape)] + [1]
        odd = torch.as_strided(x, shape, strides)
        y, dq = torch.as_strided(torch.zeros_like(x), shape, strides), torch.as_strided(torch.zeros_like(x), shape, strides)
        plain = x.view(shape)
        want, _ = ops.qk_norm_rope_fwd(plain, None, g)
        ops.qk_norm_rope_fwd(odd, None, g, out=(y, None))
        assert torch.equal(y, want)
        wdq, _, wg, _ = ops.qk_norm_rope_bwd(plain, None, plain, None, g)
        _, _, dg, _ = ops.qk_norm_rope_bwd(odd, None, odd, None, g, out=(dq, None))
        assert torch.equal(dq, wdq) and torch.equal(dg, wg)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        ops.qk_norm_rope_fwd(torch.as_strided(x, (1, 2, 1, 64), (0, 65, 0, 1)), None)


def test_as_many_tokens_as_are_taken(ops):
    """2^31 - 1 tokens of one head of 8, two tokens a warp, with listed positions: the last tokens are those of a short
    call, the rest (zeros) stays zero."""
    n, last = 2 ** 31 - 1, 300
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs 43 GB")
    q = torch.zeros(1, n, 1, 8, device="cuda", dtype=torch.float16)
    q[0, -last:] = torch.randn(last, 1, 8, device="cuda").half()
    pos = torch.arange(n, device="cuda", dtype=torch.int32).view(1, n)
    g = (1 + torch.randn(8, device="cuda")).half()
    want, _ = ops.qk_norm_rope_fwd(q[:, -last:].clone(), None, g, positions=pos[:, -last:].clone(), rot=8, interleaved=True)
    ops.qk_norm_rope_fwd(q, None, g, positions=pos, rot=8, interleaved=True, out=(q, None))
    assert torch.equal(q[:, -last:], want)
    for part in q.view(-1)[:-8 * last].split(1 << 30):
        assert not bool(part.any())
    del q, pos, part
    torch.cuda.empty_cache()
