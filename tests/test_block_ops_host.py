"""Argument checks and references of the decoder-block operators that need no GPU: a call is refused for its
arguments before it looks at its context or a device."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import ffn_ref   # noqa: E402
import qk_ref   # noqa: E402

P = 1 << 20     # an aligned address that no refused call reads


def refused(name, args, match):
    from rbk import lib
    st = getattr(lib(), name)(None, C.byref(args), None)
    msg = lib().rbk_last_error().decode()
    assert st == -1 and match in msg, (st, msg)


def qk(**kw):
    from rbk._lib import Heads, QkArgs
    a = QkArgs()
    a.B, a.S, a.Hq, a.Hk, a.dh, a.rot, a.eps, a.theta = 2, 4, 3, 1, 64, 64, 1e-6, 1e4
    for n in ("q", "k", "oq", "ok", "dyq", "dyk"):
        setattr(a, n, Heads(P, 1024, 256, 64))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("name", ["rbk_qk_norm_rope_fwd", "rbk_qk_norm_rope_bwd"])
def test_qk_refusals(name):
    from rbk._lib import Heads
    for kw, match in [
        (dict(B=-1), "negative"), (dict(Hk=-1), "negative"), (dict(B=65536, S=65536), "tokens"),
        (dict(Hq=(1 << 20) + 1), "heads"), (dict(q=Heads(P, 1 << 35, 256, 64)), "2^34"),
        (dict(oq=Heads(P, 1024, -(1 << 35), 64)), "2^34"),
        (dict(dh=0, rot=0), "dh"), (dict(dh=60, rot=0), "dh"), (dict(dh=264, rot=0), "dh"),
        (dict(rot=80), "rot"), (dict(rot=-16), "rot"), (dict(rot=24), "rot"), (dict(rot=4, interleaved=1), "rot"),
        (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(theta=0.0), "theta"),
        (dict(theta=float("inf")), "theta"), (dict(gq=P + 2), "gains"), (dict(gk=P + 8), "gains"),
        (dict(q=Heads(None, 1024, 256, 64)), "q is NULL"), (dict(k=Heads(P + 2, 1024, 256, 64)), "k must be 16-byte"),
        (dict(q=Heads(P, 1024, 252, 64)), "strides of q"), (dict(ok=Heads(P, 1024, 256, 63)), "strides of ok"),
        (dict(pos0=2 ** 31 - 3), "2^31 - 1"),
        (dict(oq=Heads(P, 1024, 256, 0)), "zero stride"), (dict(oq=Heads(P, 0, 256, 64)), "zero stride"),
    ]:
        refused(name, qk(**kw), match)
    freq = (C.c_double * 32)(*([0.5] * 31 + [float("inf")]))
    refused(name, qk(inv_freq=C.cast(freq, C.c_void_p)), "inv_freq[31]")
    refused(name, qk(pos0=2 ** 31 - 4), "ctx is NULL")       # positions up to 2^31 - 1
    refused(name, qk(pos0=-2 ** 31), "ctx is NULL")
    refused(name, qk(), "ctx is NULL")                       # nothing else is wrong with these arguments
    refused(name, qk(Hk=0, k=Heads(), ok=Heads(), dyk=Heads()), "ctx is NULL")


def test_qk_bwd_refusals():
    from rbk._lib import Heads
    refused("rbk_qk_norm_rope_bwd", qk(dyq=Heads(None, 0, 0, 0)), "dyq is NULL")
    refused("rbk_qk_norm_rope_bwd", qk(ws=P + 4), "ws")


def test_qk_gradient_formula_against_differences():
    """The reference's gradient, in float64, against central differences of its forward."""
    torch.manual_seed(0)
    B, S, H, dh = 1, 2, 2, 16
    for rot, inter in ((16, False), (8, True)):
        x, dy = (torch.randn(B, S, H, dh, dtype=torch.float64) for _ in range(2))
        gain = 1 + 0.3 * torch.randn(dh, dtype=torch.float64)
        ang = qk_ref.angles(B, S, rot, 100.0, None, 3)

        def f(x, gain):
            return float((qk_ref.fwd(x, gain, ang, rot, inter, 1e-3)[0] * dy).sum())

        dx, dg, _, _ = qk_ref.bwd(dy, x, gain, ang, rot, inter, 1e-3)
        step = 1e-6                                          # truncation ~ step^2, cancellation ~ 1e-16 / step
        for t, d in ((x, dx), (gain, dg)):
            for i in range(0, t.numel(), 7):
                e = torch.zeros_like(t)
                e.view(-1)[i] = step
                lo, hi = (f(x - e, gain), f(x + e, gain)) if t is x else (f(x, gain - e), f(x, gain + e))
                assert abs((hi - lo) / (2 * step) - float(d.view(-1)[i])) < 1e-7


def ffn(**kw):
    from rbk._lib import FfnArgs
    a = FfnArgs()
    a.N, a.D, a.F, a.ldx, a.ldy, a.ldr = 4, 64, 128, 64, 64, 64
    a.x = a.wgu = a.bgu = a.wd = a.bd = a.residual = a.y = a.gu = a.h = P
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_ffn_fwd_refusals():
    n = "rbk_gated_ffn_fwd"
    for kw, match in [
        (dict(N=-1), "negative"), (dict(D=0), "multiples of 8"), (dict(D=60), "multiples of 8"),
        (dict(N=2 ** 30 + 1), "2^30 rows"), (dict(D=2 ** 29 + 8, ldx=2 ** 29 + 8), "2^29"), (dict(F=2 ** 29 + 8), "2^29"),
        (dict(F=-8), "multiples of 8"), (dict(F=12), "multiples of 8"), (dict(act=2), "act"), (dict(act=-1), "act"),
        (dict(x=None), "x is NULL"), (dict(wgu=None), "wgu is NULL"), (dict(wd=None), "wd is NULL"),
        (dict(y=None), "y is NULL"), (dict(h=None), "h is NULL"), (dict(x=P + 2), "x must be 16-byte"),
        (dict(bgu=P + 8), "bgu must be"), (dict(bd=P + 8), "bd must be"), (dict(gu=P + 8), "gu must be"),
        (dict(residual=P + 4), "residual must be"), (dict(ldx=56), "stride of x"), (dict(ldx=68), "stride of x"),
        (dict(ldy=0), "stride of y"), (dict(ldr=8), "stride of residual"),
    ]:
        refused(n, ffn(**kw), match)
    refused(n, ffn(), "ctx is NULL")
    refused(n, ffn(bgu=None, bd=None, residual=None, ldr=0, gu=None), "ctx is NULL")


def test_ffn_bwd_refusals():
    from rbk._lib import FfnBwdArgs

    def args(**kw):
        a = FfnBwdArgs()
        a.N, a.D, a.F, a.lddy, a.ldx, a.lddx = 4, 64, 128, 64, 64, 64
        for k in ("dy", "x", "gu", "wgu", "wd", "h", "dgu", "dx", "dwgu", "dbgu", "dwd", "dbd"):
            setattr(a, k, P)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    n = "rbk_gated_ffn_bwd"
    for kw, match in [
        (dict(N=-2), "negative"), (dict(D=4), "multiples of 8"), (dict(act=7), "act"), (dict(dwgu=None), "dbgu needs"),
        (dict(dwd=None), "dbd needs"), (dict(dy=None), "dy is NULL"), (dict(x=None), "x is NULL"),
        (dict(gu=None), "gu is NULL"), (dict(wgu=None), "wgu is NULL"), (dict(wd=None), "wd is NULL"),
        (dict(h=None), "h is NULL"), (dict(dgu=None), "dgu is NULL"), (dict(dgu=P + 8), "dgu must be"),
        (dict(lddy=60), "stride of dy"), (dict(lddx=32), "stride of dx"), (dict(dwgu=P + 4), "dwgu must be"),
    ]:
        refused(n, args(**kw), match)
    refused(n, args(), "ctx is NULL")
    refused(n, args(dwgu=None, dbgu=None, dwd=None, dbd=None, dx=None, x=None, wgu=None, h=None), "ctx is NULL")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_ffn_gradient_formula_against_differences(act):
    """The reference's gradient, in float64, against central differences of its forward."""
    torch.manual_seed(1)
    N, D, F = 3, 8, 16
    x, wgu, wd, dy = (torch.randn(*s, dtype=torch.float64) for s in ((N, D), (2 * F, D), (D, F), (N, D)))

    def y(x, wgu, wd):
        return float((ffn_ref.fwd(x, wgu, wd, None, None, None, act)["y"][0] * dy).sum())

    g = ffn_ref.bwd(dy, x, x @ wgu.T, wgu, wd, act)
    args = [x, wgu, wd]
    for i, name in enumerate(("dx", "dwgu", "dwd")):
        for j in range(0, args[i].numel(), 5):
            e = torch.zeros_like(args[i])
            e.view(-1)[j] = 1e-6
            up = [t + e if k == i else t for k, t in enumerate(args)]
            lo = [t - e if k == i else t for k, t in enumerate(args)]
            want = (y(*up) - y(*lo)) / 2e-6
            assert abs(want - float(g[name][0].reshape(-1)[j])) < 1e-6 * (1 + abs(want))


def clip(tensors, max_norm=1.0, norm=P, ws=P, count=None):
    from rbk import lib
    from rbk._lib import Grad
    arr = (Grad * max(1, len(tensors)))(*[Grad(*t) for t in tensors])
    st = lib().rbk_clip_grad_norm(None, C.cast(arr, C.c_void_p), len(tensors) if count is None else count, max_norm,
                                  None, norm, ws, None)
    return st, lib().rbk_last_error().decode()


@pytest.mark.parametrize("tensors,kw,match", [
    ([], dict(count=-1), "negative count"), ([], dict(norm=None), "norm is NULL"), ([], dict(ws=P + 8), "ws"),
    ([], dict(max_norm=float("nan")), "max_norm"), ([(P, P, -1, 0)], {}, "negative size"),
    ([(P, P, 4, 2)], {}, "half must"), ([(None, None, 4, 0)], {}, "tensor 0 is NULL"),
    ([(P, P, 4, 0), (P + 66, P + 66, 4, 0)], {}, "tensor 1 is not aligned"), ([(P, P + 101, 4, 1)], {}, "not aligned"),
    ([(P, P, 1 << 41, 0)], {}, "too large"),
    ([(P, P, 100, 0), (P, P, 100, 0)], {}, "overlaps"),                       # the same tensor twice
    ([(P, P, 100, 0), (P + 396, P + 396, 9, 0)], {}, "overlaps"),             # one element shared
    ([(P, P + 4, 100, 0)], {}, "overlaps"),                                   # shifted over itself
    ([(P + 4000, P, 100, 0), (P + 300, None, 10, 1)], {}, "overlaps"),        # written over a tensor that is read
    ([(P, None, 10, 0), (P + 4000, P + 2000, 9, 0), (P + 8000, P + 2032, 9, 0)], {}, "overlaps"),
])
def test_clip_refusals(tensors, kw, match):
    st, msg = clip(tensors, **kw)
    assert st == -1 and match in msg, (st, msg)


@pytest.mark.parametrize("tensors", [
    [], [(None, None, 0, 0)], [(P, P, 100, 0), (P + 400, P + 400, 7, 0)], [(P + 400, P + 400, 7, 1), (P, P, 100, 0)],
    [(P, None, 100, 0), (P, None, 100, 0)], [(P, P + 400, 100, 0)], [(P + 2, P + 202, 100, 1)],
])
def test_clip_accepts(tensors):
    """What is not refused for its tensors is refused for the missing context only."""
    st, msg = clip(tensors)
    assert st == -1 and "ctx is NULL" in msg


def test_clip_counts_chunks_in_32_bits():
    """Tensors that are only counted may be given more than once: 2^27 chunks of 16 KB each here, fewer than 2^30 in all."""
    one = (P, None, (1 << 39) - 65536, 0)
    st, msg = clip([one] * 8)
    assert st == -1 and "ctx is NULL" in msg
    st, msg = clip([(P, None, 1 << 39, 0)] * 8)
    assert st == -1 and "too large" in msg


def test_packed_args_are_the_structs():
    """The packed forms that the ops pass have the structs' bytes."""
    from rbk import _lib
    for cls, pack in ((_lib.QkArgs, _lib.QK_PACK), (_lib.FfnArgs, _lib.FFN_PACK), (_lib.FfnBwdArgs, _lib.FFN_BWD_PACK)):
        flat, n = [], 0

        def fill(s):
            nonlocal n
            for f, ty in s._fields_:
                if issubclass(ty, C.Structure):
                    fill(getattr(s, f))
                    continue
                n += 1
                setattr(s, f, n)
                flat.append(n)

        s = cls()
        fill(s)
        assert pack.pack(*flat) + bytes(C.sizeof(cls) - pack.size) == bytes(s)


def test_workspace_sizes_match_header():
    import os
    import re

    from rbk import ops
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rbk.h")).read()
    for name in ("RBK_QK_BWD_WS_BYTES", "RBK_CLIP_WS_BYTES"):
        expr = re.search(rf"#define {name} \((.*)\)", src).group(1)
        assert eval(expr) == getattr(ops, name), name


def test_ffn_ws_bytes_refusals():
    from rbk import lib
    for args in ((-1, 64, 128, 0), (4, 60, 128, 1), (4, 64, 0, 0), (64, 64, 128, 0)):
        assert lib().rbk_gated_ffn_ws_bytes(None, *args) == -1


def test_args_layouts_match_header(tmp_path):
    """The ctypes mirrors of the block operators' argument structs have the C compiler's field offsets."""
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    from rbk import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = [("rbk_heads", _lib.Heads), ("rbk_qk_args", _lib.QkArgs), ("rbk_ffn_args", _lib.FfnArgs),
               ("rbk_ffn_bwd_args", _lib.FfnBwdArgs), ("rbk_grad", _lib.Grad)]
    lines, want = [], []
    for cname, cls in structs:
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {f}));')
            want.append(getattr(cls, f).offset)
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(C.sizeof(cls))
    src = tmp_path / "off.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rbk.h"\nint main(void) {\n' +
                   "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-I/usr/local/cuda/include", str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


FFN_SIZES = r"""
import ctypes as C, sys
from rbk import lib
ctx = (C.c_int * 1024)(0, 148)          # a context of a device with 148 SMs: nothing else of it is looked at
for n, d, f, back in eval(sys.argv[1]):
    print(lib().rbk_gated_ffn_ws_bytes(ctx, n, d, f, back), lib().rbk_last_error().decode())
"""


def test_ffn_sizes_at_the_ends_of_their_range():
    """A query with sizes of the documented range answers or refuses, and divides by no product that has wrapped to 0."""
    import subprocess
    import sys
    from rbk._lib import PKG_ROOT
    # (N, D, F, backward): more tiles than an int counts
    refused = [(2 ** 30, 2 ** 29, 8, 0), (2 ** 30, 2 ** 29, 8, 1), (2 ** 30, 2 ** 29, 2 ** 29, 0), (2 ** 24, 2 ** 24, 8, 0),
               (8, 2 ** 29, 2 ** 29, 1), (2 ** 30, 8, 2 ** 29, 0), (2 ** 22, 2 ** 23, 8, 0)]      # 2^15 * 2^16 tiles
    taken = [(2 ** 30, 8, 8, 0), (2 ** 30, 8, 8, 1), (2 ** 22, 2 ** 22, 2 ** 21, 1), (8, 2 ** 29, 256, 1),
             (2 ** 22, 2 ** 23 - 128, 8, 0)]
    r = subprocess.run([sys.executable, "-c", FFN_SIZES, str(refused + taken)], cwd=PKG_ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.returncode
    lines = r.stdout.splitlines()
    assert all(x.startswith("-1 ") and "tiles" in x for x in lines[:len(refused)]), lines
    assert all(int(x.split()[0]) >= 0 for x in lines[len(refused):]), lines


def test_ffn_timeout_test_refusals():
    from rbk import lib
    ctx = (C.c_int * 1024)(0, 148)
    for c, limit, match in ((None, 1e-3, "null ctx"), (ctx, 1e-5, "limit_s"), (ctx, 3.0, "limit_s"),
                            (ctx, float("nan"), "limit_s")):
        assert lib().rbk_ctx_arm_ffn_timeout_test(c, limit) == -1 and match in lib().rbk_last_error().decode()


def ffn_plan(N, D, F, back):
    """The kernels of a call on 148 SMs, as rbk_gated_ffn_plan gives them."""
    from rbk import lib
    ctx, plan = (C.c_int * 1024)(0, 148), (C.c_int * 6)()
    assert lib().rbk_gated_ffn_plan(ctx, N, D, F, back, plan) == 0, lib().rbk_last_error()
    return tuple(plan[:3]), tuple(plan[3:])


def ffn_kernels(N, D, F):
    """The kernel instances and configurations that a forward and a backward of these sizes run."""
    out = set()
    for back in (0, 1):
        for i, (kernel, cols, parts) in enumerate(ffn_plan(N, D, F, back)):
            if kernel == 0:                                 # rows: by the rows' multiple of 8 too
                parts = 1 if N <= 8 else 2 if N <= 16 else 4 if N <= 32 else 8
            elif kernel == 2:
                parts = parts > 1
            out.add((back, i, kernel, cols, parts))
    return out


def test_ffn_tests_reach_every_kernel():
    """Whatever kernel a call of 1 to 5000 rows and widths up to 5632 chooses, some size of the GPU tests chooses too."""
    import random

    import test_gpu_ffn as t
    tested = set().union(*(ffn_kernels(*s) for s in t.SIZES + t.MIDDLE + t.REST + t.PAIRS))
    r = random.Random(0)
    for _ in range(60000):
        n, d, f = (int(2 ** r.uniform(0, 12.3)), 8 * int(2 ** r.uniform(0, 9.46)), 8 * int(2 ** r.uniform(0, 9.46)))
        missing = ffn_kernels(n, d, f) - tested
        assert not missing, (n, d, f, missing)


def test_ffn_plan():
    from rbk import lib
    rows, pairs = 0, 2
    assert ffn_plan(1, 2048, 5632, 0) == ((rows, 0, 1), (rows, 1, 1))
    assert ffn_plan(8192, 2048, 5632, 0) == ((pairs, 256, 1), (pairs, 256, 1))
    for size in ((1999, 776, 2056), (600, 264, 8712)):
        for back in (0, 1):
            (k0, _, _), (k1, _, parts) = ffn_plan(*size, back)
            assert k0 == k1 == pairs and parts > 1
            ctx = (C.c_int * 1024)(0, 148)
            assert lib().rbk_gated_ffn_ws_bytes(ctx, *size, back) == 4 * parts * size[0] * size[1]
    plan, ctx = (C.c_int * 6)(), (C.c_int * 1024)(0, 148)
    for args, match in (((None, 4, 64, 128, 0, plan), "NULL"), ((ctx, 4, 64, 128, 0, None), "NULL"),
                        ((ctx, 0, 64, 128, 0, plan), "no rows"), ((ctx, 4, 60, 128, 0, plan), "multiples")):
        assert lib().rbk_gated_ffn_plan(*args) == -1 and match in lib().rbk_last_error().decode()


def test_import_without_a_cuda_build_of_torch():
    """The package's operators import where torch has none of its CUDA functions."""
    import subprocess
    import sys
    from rbk._lib import PKG_ROOT
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_get')]:\n    delattr(torch._C, n)\n"
            "import rbk.ops, rbk.model, rbk.tokenizer\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=PKG_ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
