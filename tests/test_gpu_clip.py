"""rbk_clip_grad_norm against float64.

Tolerances, E = 2^-24: the squares are summed in FP64 (n 2^-53, below E for every n here); eight squares of
halves are first added in FP32, at most 8 E of their sum and 4 E of the norm.  The norm is rounded to FP32: 5 E
(with halves) or 2 E.  The factor takes the norm's error in FP64 and one rounding, the product one more: 7 E,
then for a half its own rounding, 2^-11 of the value (2^-25 among the subnormals).
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from rbk import ops as o
    torch.cuda.set_device(0)
    return o


def tensors(sizes, types, shift=0, sigma=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(sizes))
    out = []
    for i, n in enumerate(sizes):
        dt = {"f32": torch.float32, "f16": torch.float16, "mixed": (torch.float32, torch.float16)[i % 2]}[types]
        s = (shift * (i + 1)) % 11
        out.append((sigma * torch.randn(n + s, device="cuda", generator=g)).to(dt)[s:])
    return out


def check(grads, out, norm, max_norm, scale=1.0):
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads)) / scale
    assert abs(float(norm) - want) <= 5 * E * want, (float(norm), want)
    coef = min(1.0, max_norm / want) if want > 0 and max_norm > 0 else 1.0
    for g, o in zip(grads, out):
        if o is None:
            continue
        v = g.double() * coef
        lim = (7 * E + (2.0 ** -11 if g.dtype == torch.float16 else 0)) * v.abs()
        lim = lim + (2.0 ** -25 if g.dtype == torch.float16 else 2.0 ** -149)
        assert bool(((o.double() - v).abs() <= lim).all())


SIZES = [[1], [3], [5, 1, 2], [0, 7, 0], [8191, 8192, 8193], [4096, 16384, 16385, 16383], [100003],
         [1, 2, 3, 4, 5, 6, 7, 8, 9, 10] * 13, [700001, 3, 50000, 12345, 1, 999]]


@pytest.mark.parametrize("types", ["f32", "f16", "mixed"])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:6])))
def test_norm_and_clipped(ops, sizes, types, shift):
    grads = tensors(sizes, types, shift)
    n = max(1, sum(sizes))
    for max_norm in (0.1 * math.sqrt(n), 10 * math.sqrt(n)):          # clips, does not clip
        out = [torch.full_like(g, 77.0) for g in grads]
        norm = ops.clip_grad_norm(grads, max_norm, out=out)
        check(grads, out, norm, max_norm)
        own = [g.clone() for g in grads]
        norm2 = ops.clip_grad_norm(own, max_norm)
        assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(own, out))


def test_neighbours_stay(ops):
    """Out of place at another alignment than the gradients': the elements around every range stay as they were."""
    for dt in (torch.float32, torch.float16):
        for n in (1, 5, 8, 33, 8192 * 2 + 1):
            for off in (0, 1, 2, 3, 5, 7):
                g = torch.randn(n + 3, device="cuda").to(dt)[3:]
                buf = torch.full((n + 32,), 5.0, device="cuda", dtype=dt)
                out = buf[8 + off:8 + off + n]
                norm = ops.clip_grad_norm([g], 0.01, out=[out])
                check([g], [out], norm, 0.01)
                assert bool((buf[:8 + off] == 5).all()) and bool((buf[8 + off + n:] == 5).all())


def test_loss_scale_and_tensors_that_are_only_counted(ops):
    grads = tensors([1000, 33, 20000], "f32", sigma=300.0)
    sc = ops.new_scaler(scale=1024.0)
    out = [torch.empty_like(grads[0]), None, torch.empty_like(grads[2])]
    keep = grads[1].clone()
    norm = ops.clip_grad_norm(grads, 1.0, scaler=sc, out=out)
    check(grads, out, norm, 1.0, 1024.0)
    assert torch.equal(grads[1], keep)
    norm2 = ops.clip_grad_norm(grads, 0.0, scaler=sc)                 # the norm alone
    assert torch.equal(norm, norm2) and torch.equal(grads[1], keep)


def test_many_tensors(ops):
    """More tensors than one launch takes (900), and more than two."""
    for count in (121, 901, 2000):
        grads = tensors([(37 * i) % 300 for i in range(count)], "mixed", 1)
        out = [torch.empty_like(g) for g in grads]
        norm = ops.clip_grad_norm(grads, 3.0, out=out)
        check(grads, out, norm, 3.0)


def test_nothing_to_clip(ops):
    assert float(ops.clip_grad_norm([], 1.0)) == 0.0
    z = torch.zeros(100, device="cuda")
    assert float(ops.clip_grad_norm([z, z[:0]], 1.0)) == 0.0 and bool((z == 0).all())


def test_extreme_values(ops):
    """Squares beyond FP32's range on both sides; FP16's largest values; subnormals."""
    for v, dt in ((3e38, torch.float32), (1e-30, torch.float32), (65504.0, torch.float16), (2.0 ** -24, torch.float16)):
        g = torch.full((1000,), v, device="cuda", dtype=dt)
        out = [torch.empty_like(g)]
        m = min(float(g[0]) * 3, 1e38)
        norm = ops.clip_grad_norm([g], m, out=out)
        want = float(g[0]) * math.sqrt(1000)
        assert abs(float(norm) - want) <= 5 * E * want if want < 3.4e38 else math.isinf(float(norm))
        v = g.double() * (m / want)
        half = dt == torch.float16
        assert bool(((out[0].double() - v).abs() <= 7 * E * v + (2.0 ** -11 * v + 2.0 ** -25 if half else 0)).all())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_is_not_finite_passes_unchanged(ops, bad):
    """The tail must still find the overflow, and find the other gradients as they were."""
    for types in ("f32", "f16"):
        grads = tensors([1000, 20, 30000], types)
        grads[2][12345] = bad
        own, out = [g.clone() for g in grads], [torch.empty_like(g) for g in grads]
        n1 = ops.clip_grad_norm(own, 1.0)
        n2 = ops.clip_grad_norm(grads, 1.0, out=out)
        assert not math.isfinite(float(n1)) and not math.isfinite(float(n2))
        for g, a, b in zip(grads, own, out):
            assert torch.equal(g.nan_to_num(1.5), a.nan_to_num(1.5)) and torch.equal(g.nan_to_num(1.5), b.nan_to_num(1.5))


def test_before_the_optimizer_tail(ops):
    """Clip, then rbk_adam_tail: a clean step moves the masters, an overflow is skipped and counted."""
    n = 5000
    p32 = torch.randn(n, device="cuda")
    m, v, p16 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), p32.half()
    sc = ops.new_scaler(scale=256.0)
    g = 256.0 * torch.randn(n, device="cuda")
    before = p32.clone()
    parts = [g[:1024], g[1024:1027], g[1027:]]
    norm = ops.clip_grad_norm(parts, 0.5, scaler=sc)
    want = 0.5 * g.double() / g.double().norm()            # what the tail sees, divided by the scale
    ops.adam_tail(p32, g.clone(), m, v, p16, sc, lr=1e-3)
    assert float(norm) > 50 and torch.allclose(m.double(), 0.1 * want, rtol=1e-5, atol=1e-9)
    assert not torch.equal(p32, before)
    held = p32.clone()
    g = 256.0 * torch.randn(n, device="cuda")
    g[7] = float("inf")
    ops.clip_grad_norm([g], 0.5, scaler=sc)
    ops.adam_tail(p32, g, m, v, p16, sc, lr=1e-3)
    st = ops.read_scaler(sc)
    assert st.skipped == 1 and st.overflow_steps == 1 and torch.equal(p32, held)


def test_repeats_bits_on_streams_and_in_graphs(ops):
    grads = tensors([70001, 333, 1 << 20, 8], "mixed", 1)

    def once():
        out = [torch.empty_like(g) for g in grads]
        return [ops.clip_grad_norm(grads, 2.0, out=out)] + out

    want = once()
    assert all(torch.equal(a, b) for a, b in zip(once(), want))
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                out = once()
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
    g = torch.zeros(8, 8, device="cuda")
    for grads, kw in (([g.T[1:]], {}), ([g.cpu()], {}), ([g.double()], {}), ([g], dict(out=[])),
                      ([g], dict(out=[g.half()])), ([g], dict(out=[g[:4]])),
                      ([g], dict(scaler=torch.zeros(8, device="cuda")))):
        with pytest.raises(ValueError):
            ops.clip_grad_norm(grads, 1.0, **kw)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grad_norm([g, g], 1.0)


def test_factors_below_the_normal_range(ops):
    """max_norm / norm below 2^-126, and below the smallest subnormal: large gradients keep all their bits.  The factor
    is then two, each right to E, the first product to E (2^-150 among the subnormals, times a factor of at most 1), the
    second to E (2^-150): 7 E as before, and 2^-149."""
    for v, max_norm, scale in ((3e38, 1e-3, 1.0), (3e38, 1e-7, 1.0), (1e30, 1e-12, 1.0), (3e38, 1e-30, 2.0 ** -20),
                               (1e20, 1e-38, 1.0)):
        max_norm = float(torch.tensor(max_norm, dtype=torch.float32))
        half = float(torch.tensor(max_norm / math.sqrt(2), dtype=torch.float32))
        g = torch.full((70001,), v, device="cuda")
        g[::3] = 1.0
        g[1::7] = -v / 7
        h = torch.full((33,), 2.0, device="cuda").half()
        sc = ops.new_scaler(scale=scale)
        want = math.sqrt(float((g.double() ** 2).sum()) + 33 * 4.0)
        f = max_norm / (want / scale)
        assert f < 2.0 ** -126
        out = [torch.empty_like(g), torch.ones_like(h), torch.full((g.numel() + 9,), 5.0, device="cuda")[9:]]
        ops.clip_grad_norm([g, h, g], half, scaler=sc, out=[out[0], out[1], None])
        ops.clip_grad_norm([g, h], max_norm, scaler=sc, out=[out[2], None])
        lim = 7 * E * (g.double() * f).abs() + 2.0 ** -149
        f2 = half / (math.sqrt(2 * float((g.double() ** 2).sum()) + 33 * 4.0) / scale)
        assert bool(((out[0].double() - g.double() * f2).abs() <= lim).all()) and bool((out[1] == 0).all())
        assert bool(((out[2].double() - g.double() * f).abs() <= lim).all())


def test_model_step_clipped_by_the_global_norm(ops):
    """Between a model's backward and its optimizer step, by public means: the arena's gradients, the model's scaler.
    The step is the one of gradients scaled by hand: m = 0.1 g / scale * factor, the factor right to 7 E, the tail's
    division and product to 3 E more."""
    from rbk.model import ModelConfig, RubidiumTransformer
    m = RubidiumTransformer(ModelConfig(V=512, T=64, D=128, H=2, L=2, FF=256), max_batch=2, max_seq=64)
    m.init_weights(seed=5)
    tok = torch.randint(0, 512, (2, 64), device="cuda", dtype=torch.int32)
    m.forward(tok, tok, 2, 64)
    m.backward(tok, tok, 2, 64)
    g, scale = m.grad.double(), m.loss_scale
    want = float(g.norm()) / scale
    norm = ops.clip_grad_norm([m.grad], want / 4, scaler=m.scaler_buffer)
    assert abs(float(norm) - want) <= 2 * E * want
    m.optimizer_step(1, 1e-3)
    got, v = m._bufs[3].double(), 0.1 * g / scale / 4
    assert bool(((got - v).abs() <= 10 * E * v.abs() + 2.0 ** -149).all()) and float(got.norm()) > 0
    assert m.scaler().skipped == 0


def test_more_elements_than_32_bits_count(ops):
    """A tensor of 2^32 + 5 halves, clipped in place: its ends count and are scaled, its neighbours stay."""
    n = 2 ** 32 + 5
    buf = torch.zeros(n + 16, device="cuda", dtype=torch.float16)
    g = buf[3:3 + n]
    at = [0, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, n - 1]
    g[at] = 16.0
    buf[:3], buf[3 + n:] = 5.0, 5.0
    want = 16.0 * math.sqrt(len(at))
    norm = ops.clip_grad_norm([g], want / 4)
    assert abs(float(norm) - want) <= 5 * E * want
    assert bool((g[at] == 4.0).all()) and int(torch.count_nonzero(g)) == len(at)
    assert bool((buf[:3] == 5).all()) and bool((buf[3 + n:] == 5).all())
    del buf, g
    torch.cuda.empty_cache()
