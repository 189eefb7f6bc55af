"""The norms around a block (csrc/blocknorm.hip, block_hip.norm_before / norm_after / norm_between) against the formulas in
64 bits.

Tolerances, set before the first run.  u = half a step of the element type (bf16 2^-8, fp16 2^-11, fp32 2^-24).  Between
loads and stores everything is float32, so a 16-bit result is off by its one rounding, u / sqrt(3) of it in the 2-norm at
most, and float32 sums of c terms (c 2^-24 at the very most, 1e-5 for c = 8192 with pairwise sums): u + 1e-5.  Float32
results and the parameters' gradients: 1e-5 in the 2-norm."""
import ctypes as C

import pytest
import torch

from tests.helpers import new_graph, record, rel_err
from video_diffusion_amd import _lib

gpu = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.bfloat16: 2.0 ** -8 + 1e-5, torch.float16: 2.0 ** -11 + 1e-5, torch.float32: 1e-5}
NAMES = ("x", "h", "post_weight", "gate", "weight", "scale", "shift")


def unit(t, kind, eps):
    if kind is None:
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)


def reference(p, alpha, kind, post_kind, eps, want_y=True):
    """(out, y) by autograd-capable torch operations in float64."""
    x, h, pw, gate, w, scale, shift = (p[k] for k in NAMES)
    row = lambda t: t if t.dim() == 1 else t.reshape(t.shape[0], *([1] * (x.dim() - 2)), t.shape[1])
    out = x
    if h is not None:
        t = unit(h, post_kind, eps)
        t = t if pw is None else t * pw
        out = alpha * x + (t if gate is None else t * row(gate))
    y = None
    if want_y:
        y = unit(out, kind, eps)
        y = y if w is None else y * w
        y = y if scale is None else y * (1 + row(scale))
        y = y if shift is None else y + row(shift)
    return (None if h is None else out), y


def make(shape, dtype, seed, absent=(), per_sample=("gate", "scale", "shift")):
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, c = shape[0], shape[-1]
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    p = {"x": (1.5 * rnd(*shape) + 0.3).to(dtype), "h": (0.7 * rnd(*shape) - 0.2).to(dtype),
         "post_weight": 1 + 0.3 * rnd(c), "weight": 1 + 0.3 * rnd(c)}
    for k in ("gate", "scale", "shift"):
        v = 0.5 * rnd(b, c)
        p[k] = v if k in per_sample else v[:1] if b % 2 else v[0].clone()
    for k in absent:
        p[k] = None
    return p, [rnd(*shape).to(dtype) for _ in range(2)]


def call(B, p, alpha, kind, post_kind, eps, want_y):
    if p["h"] is None:
        return None, B.norm_before(p["x"], p["weight"], p["scale"], p["shift"], kind=kind, eps=eps)
    if not want_y:
        return B.norm_after(p["x"], p["h"], p["post_weight"], p["gate"], alpha=alpha, kind=post_kind, eps=eps), None
    return B.norm_between(*(p[k] for k in NAMES), alpha=alpha, kind=kind, post_kind=post_kind, eps=eps)


def check(name, p, ups, alpha=1.0, kind="rms", post_kind="rms", eps=1e-5, want_y=True):
    from video_diffusion_amd import block_hip as B
    tol = TOL[p["x"].dtype]
    used = [k for k in NAMES if p[k] is not None and (want_y or k in ("x", "h", "post_weight", "gate"))]
    lv = {k: p[k].detach().requires_grad_() if k in used else None for k in NAMES}
    ref = {k: None if v is None else v.detach().double().requires_grad_() for k, v in lv.items()}
    got, want = call(B, lv, alpha, kind, post_kind, eps, want_y), reference(ref, alpha, kind, post_kind, eps, want_y)
    sel = [i for i in range(2) if got[i] is not None]
    assert sel == [i for i in range(2) if want[i] is not None]
    for i in sel:
        assert got[i].dtype == p["x"].dtype and got[i].shape == p["x"].shape
        err = record(f"norm.{name}.{('out', 'y')[i]}", rel_err(got[i].detach(), want[i].detach()), tol)
        assert err < tol, (name, i, err)
    grads = torch.autograd.grad([got[i] for i in sel], [lv[k] for k in used], [ups[i] for i in sel])
    refs = torch.autograd.grad([want[i] for i in sel], [ref[k] for k in used], [ups[i].double() for i in sel])
    for k, a, b in zip(used, grads, refs):
        t = tol if k in ("x", "h") else 1e-5
        assert a.shape == b.shape
        err = record(f"norm.{name}.d{k}", rel_err(a, b), t)
        assert err < t, (name, k, err)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("c", [1, 3, 8, 30, 64, 72, 128, 200, 256, 384, 512, 520, 1000, 1024, 1181, 1536, 2048, 2055, 4096, 5000, 8192])
def test_widths(c, dtype):
    """Every arrangement of lanes and pieces, with and without wide loads.  (One column: the layer norm is constant zero, and
    the gradient of the other kind is the share eps has of the mean square: a large one, for its relative error to say
    something.)"""
    kind = "rms" if c == 1 or c % 3 else "layer"
    check(f"c{c}.{dtype}", *make((3, 11, c), dtype, c), alpha=0.7, kind=kind, post_kind=kind, eps=0.5 if c == 1 else 1e-5)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", [2, 5, 7, 9, 15, 17, 63, 65, 127, 129, 255, 257, 511, 513, 1023, 1025, 2047, 2049, 4095, 4097, 8191])
def test_odd_widths(c, dtype):
    """Rows whose last piece overlaps the one before, or that are shorter than a piece."""
    check(f"odd{c}.{dtype}", *make((2, 37, c), dtype, c + 1), alpha=0.7, kind="layer" if c > 8 else "rms", eps=0.5 if c < 8 else 1e-5)


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post_kind", ["rms", "layer", None])
@pytest.mark.parametrize("shape", [(1, 1, 64), (2, 1, 64), (5, 333, 64), (2, 3, 5, 7, 96), (4, 2500, 32), (7, 512)])
def test_kinds_and_row_counts(shape, post_kind, kind):
    check(f"{shape}.{kind}.{post_kind}", *make(shape, torch.bfloat16, 1), kind=kind, post_kind=post_kind)


@gpu
@pytest.mark.parametrize("absent", [("post_weight",), ("gate",), ("weight",), ("scale",), ("shift",), ("gate", "scale", "shift"),
                                    ("post_weight", "gate", "weight", "scale", "shift")])
@pytest.mark.parametrize("per_sample", [("gate", "scale", "shift"), ("gate",), ("shift",), ()])
@pytest.mark.parametrize("b", [1, 2, 3])
def test_absent_and_shared_parameters(absent, per_sample, b):
    """Gradients of parameters that belong to samples, to all rows ([c] and [1, c]), or are not there."""
    check(f"absent{absent}.{per_sample}.{b}", *make((b, 70, 128), torch.float32, 2, absent, per_sample), kind="layer")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", [64, 100, 1024])
def test_before_and_after_alone(c, dtype):
    p, ups = make((2, 50, c), dtype, 3)
    check(f"after.{c}.{dtype}", p, ups, alpha=-0.5, post_kind="layer", want_y=False)
    check(f"after_plain.{c}.{dtype}", p, ups, post_kind=None, want_y=False)
    for k in ("h", "post_weight", "gate"):
        p[k] = None
    check(f"before.{c}.{dtype}", p, ups, kind="layer")
    check(f"before_rms.{c}.{dtype}", p, ups, kind="rms", eps=1e-2)


@gpu
def test_strides_and_alignment():
    """Rows inside wider ones, rows at odd addresses and pitches, transposed and expanded tensors; gradients of such
    layouts."""
    g = torch.Generator(device=DEV).manual_seed(4)
    wide = torch.randn(2, 40, 300, generator=g, device=DEV).to(torch.bfloat16)
    p, ups = make((2, 40, 64), torch.bfloat16, 4)
    for name, x in (("pitch", wide[..., 8:72]), ("odd", wide[..., 3:67]), ("turned", wide[..., :64].transpose(0, 1).contiguous().transpose(0, 1)),
                    ("columns", torch.randn(2, 64, 40, generator=g, device=DEV).to(torch.bfloat16).transpose(1, 2)),
                    ("expanded", wide[:, :1, :64].expand(2, 40, 64))):
        for k in ("x", "h"):
            check(f"stride.{name}.{k}", dict(p, **{k: x}), ups)
        check(f"stride.{name}.up", p, [x, ups[1]])
        check(f"stride.{name}.up2", p, [ups[0], x])


@gpu
def test_gradient_against_differences():
    """Directional derivatives of a fixed functional by central differences of the float64 formula."""
    from video_diffusion_amd import block_hip as B
    p, ups = make((2, 9, 72), torch.float32, 5)
    lv = {k: v.detach().requires_grad_() for k, v in p.items()}
    got = call(B, lv, 0.9, "layer", "rms", 1e-5, True)
    grads = dict(zip(NAMES, torch.autograd.grad(got, [lv[k] for k in NAMES], ups)))
    g = torch.Generator(device=DEV).manual_seed(6)
    for k in NAMES:
        d = torch.randn(p[k].shape, generator=g, device=DEV, dtype=torch.float64)
        val = []
        for e in (1e-5, -1e-5):
            q = {n: v.double() for n, v in p.items()}
            q[k] = q[k] + e * d
            val.append(sum(float((o * u.double()).sum()) for o, u in zip(reference(q, 0.9, "layer", "rms", 1e-5), ups)))
        slope = (val[0] - val[1]) / 2e-5
        assert abs(float((grads[k].double() * d).sum()) - slope) < 1e-5 * float(grads[k].double().norm() * d.norm()), k


@gpu
def test_partial_gradients():
    """Some inputs only; one of the two results unused; parameters of the unused one get zeros."""
    from video_diffusion_amd import block_hip as B
    p, ups = make((2, 33, 128), torch.bfloat16, 7)
    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    out, y = reference(ref, 1.0, "rms", "rms", 1e-5)
    for i, r in ((0, out), (1, y)):
        want = dict(zip(NAMES, torch.autograd.grad(r, [ref[k] for k in NAMES], ups[i].double(), retain_graph=True, allow_unused=True)))
        for k in NAMES:
            lv = dict(p)
            lv[k] = p[k].detach().requires_grad_()
            got = call(B, lv, 1.0, "rms", "rms", 1e-5, True)[i]
            (gk,) = torch.autograd.grad(got, lv[k], ups[i])
            if want[k] is None:
                assert not gk.any()
            else:
                assert rel_err(gk, want[k]) < (TOL[torch.bfloat16] if k in ("x", "h") else 1e-5), (i, k)


@gpu
def test_rows_of_zeros_and_rows_that_are_not_finite():
    """A row of zeros has the norm zero; a NaN stays in its row (forward, dx, dh)."""
    from video_diffusion_amd import block_hip as B
    p, ups = make((2, 8, 64), torch.bfloat16, 8)
    p["x"][0, 0] = p["h"][0, 0] = 0
    check("zeros", p, ups)
    lv = {k: v.detach().requires_grad_() for k, v in p.items()}
    clean = call(B, lv, 1.0, "rms", "layer", 1e-5, True)
    cg = torch.autograd.grad(clean, [lv["x"], lv["h"]], ups)
    q = dict(p, x=p["x"].clone(), h=p["h"].clone())
    q["x"][1, 3, 5], q["h"][0, 6, 9] = float("nan"), float("inf")
    lv = {k: v.detach().requires_grad_() for k, v in q.items()}
    bad = call(B, lv, 1.0, "rms", "layer", 1e-5, True)
    bg = torch.autograd.grad(bad, [lv["x"], lv["h"]], ups)
    keep = torch.ones(2, 8, dtype=torch.bool, device=DEV)
    keep[1, 3] = keep[0, 6] = False
    for a, b in zip((*clean, *cg), (*bad, *bg)):
        assert torch.equal(a[keep], b[keep])
    assert not torch.isfinite(bad[1][~keep]).any()


@gpu
def test_same_bits_streams_and_graph():
    from video_diffusion_amd import block_hip as B
    p, ups = make((3, 1000, 256), torch.bfloat16, 9)

    def run():
        lv = {k: v.detach().requires_grad_() for k, v in p.items()}
        got = call(B, lv, 1.0, "layer", "rms", 1e-5, True)
        return [*(t.detach() for t in got), *torch.autograd.grad(got, [lv[k] for k in NAMES], ups)]

    want = run()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    res = []
    for s in streams:
        with torch.cuda.stream(s):
            res.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in res for a, b in zip(r, want))
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = new_graph()
    with torch.cuda.graph(graph):
        outs = run()
    g = torch.Generator(device=DEV).manual_seed(10)
    for _ in range(3):
        for t in (p["x"], p["h"], *ups, p["gate"]):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


@gpu
def test_no_rows():
    from video_diffusion_amd import block_hip as B
    x = torch.zeros(2, 0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out, y = B.norm_between(x, x)
    assert out.shape == x.shape and y.shape == x.shape
    assert B.norm_before(x).shape == x.shape and B.norm_after(x, x).shape == x.shape


@gpu
def test_parameters_of_calls_without_rows():
    from video_diffusion_amd import block_hip as B
    x = torch.zeros(2, 0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    p = [torch.randn(64, device=DEV, requires_grad=True) for _ in range(5)]
    for res, used in ((B.norm_between(x, x, *p), p), (B.norm_between(x, x, *p)[:1], p[:2]), ([B.norm_before(x, *p[:3])], p[:3])):
        assert not any(g.any() for g in torch.autograd.grad([r.sum() for r in res], used))


@gpu
def test_many_samples():
    """More samples than one grid dimension of 16 bits holds, each with its own parameters."""
    p, ups = make((70001, 1, 8), torch.bfloat16, 6)
    check("many", p, ups, alpha=0.9, post_kind="layer")


@gpu
def test_offsets_beyond_32_bits():
    """5.1e9 elements: the first and last rows against the same rows by themselves."""
    from video_diffusion_amd import block_hip as B
    rows, c = 620000, 8192
    w = 1 + 0.3 * torch.randn(c, device=DEV)
    x = torch.zeros(rows, c, device=DEV, dtype=torch.bfloat16)
    ends = torch.randn(64, c, device=DEV).to(torch.bfloat16)
    x[:32], x[-32:] = ends[:32], ends[32:]
    y = B.norm_before(x, w)
    assert torch.equal(torch.cat((y[:32], y[-32:])), B.norm_before(ends, w))
    assert not y[32:40].any()
    del y
    x.requires_grad_()
    ends.requires_grad_()
    dy = torch.zeros_like(x)
    dy[:32], dy[-32:] = 1.5, -0.5
    (dx,) = torch.autograd.grad(B.norm_before(x, w), x, dy)
    (want,) = torch.autograd.grad(B.norm_before(ends, w), ends, torch.cat((dy[:32], dy[-32:])))
    assert torch.equal(torch.cat((dx[:32], dx[-32:])), want)


@gpu
def test_no_second_derivative():
    from video_diffusion_amd import block_hip as B
    x = torch.randn(2, 5, 64, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(B.norm_before(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def _args(**kw):
    a = _lib.BlockNormArgs()
    a.c, a.rows, a.rows_per_sample, a.eps, a.alpha = 64, 20, 10, 1e-5, 1.0
    for f in ("x", "h", "out", "y", "post_weight", "gate", "weight", "scale", "shift"):
        setattr(a, f, 256)
    for f in ("ldx", "ldh", "ldo", "ldy", "lddo", "lddy", "lddx", "lddh"):
        setattr(a, f, 64)
    a.gate_stride = a.scale_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_entry_points_refuse_bad_arguments():
    lib = _lib.lib()
    E_ARG, E_SHAPE, E_ALIGN = -1, -2, -3
    fwd = lambda **kw: lib.vdmi_block_norm_fwd(C.byref(_args(**kw)), None)
    grads = dict(dout=256, dy=256, dx=256, dh=256, dweight=256)
    bwd = lambda **kw: lib.vdmi_block_norm_bwd(C.byref(_args(**{**grads, **kw})), None)
    need = lambda **kw: lib.vdmi_block_norm_bwd_workspace_bytes(C.byref(_args(**{**grads, **kw})))
    assert lib.vdmi_block_norm_fwd(None, None) == E_ARG and lib.vdmi_block_norm_bwd(None, None) == E_ARG
    for f in (fwd, bwd):
        assert f(x=None) == E_ARG and f(dtype=3) == E_ARG and f(kind=-1) == E_ARG and f(post_kind=2) == E_ARG
        assert f(eps=-1.0) == E_ARG and f(eps=float("nan")) == E_ARG and f(alpha=float("inf")) == E_ARG
        assert f(c=0) == E_SHAPE and f(c=8193) == E_SHAPE and f(rows=0) == E_SHAPE and f(rows=21) == E_SHAPE
        assert f(gate_stride=32) == E_SHAPE and f(ldx=63) == E_SHAPE and f(ldh=8) == E_SHAPE
        assert f(x=257) == E_ALIGN and f(dtype=2, h=258) == E_ALIGN
        assert f(h=None, out=None, dh=None) == E_ARG                    # a gate without a block
    assert fwd(out=None) == E_ARG and fwd(y=None, out=None, h=None, gate=None, post_weight=None) == E_ARG
    assert fwd(ldo=60) == E_SHAPE and fwd(ldy=60) == E_SHAPE
    assert bwd(dout=None, dy=None) == E_ARG and bwd(dweight=256, weight=None) == E_ARG and bwd(dgate=256, gate=None) == E_ARG
    assert bwd(lddx=63) == E_SHAPE and bwd() == E_ARG                   # no workspace
    assert need() > 0 and bwd(workspace=256, workspace_bytes=need() - 1) == E_ARG
    assert bwd(workspace=264, workspace_bytes=need()) == E_ALIGN
    assert need(dweight=None) == 0                                      # no parameter's gradient: no sums


@gpu
def test_python_entry_points_refuse():
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    x = torch.zeros(2, 4, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV)
    for f, what in [(lambda: B.norm_before(x.double()), "bfloat16"), (lambda: B.norm_before(x, w[:32]), "weight"),
                    (lambda: B.norm_before(x, w.half()), "weight"), (lambda: B.norm_before(x, w, torch.ones(3, 64, device=DEV)), "scale"),
                    (lambda: B.norm_before(x, kind="batch"), "kind"), (lambda: B.norm_before(x, kind=None), "kind"),
                    (lambda: B.norm_before(x, eps=-1), "eps"), (lambda: B.norm_after(x, x[:, :2]), "alike"),
                    (lambda: B.norm_after(x, x.float()), "alike"), (lambda: B.norm_after(x, x, alpha=float("nan")), "alpha"),
                    (lambda: B.norm_before(x[0, 0]), "rows are"), (lambda: B.norm_before(torch.zeros(2, 9000, device=DEV)), "8192"),
                    (lambda: B.norm_after(x, None), "missing"), (lambda: B.norm_between(x, None), "missing"),
                    (lambda: B.norm_before(x, w.cpu()), "no CPU path")]:
        with pytest.raises(VdmiError, match=what):
            f()


def test_no_cpu_path():
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    with pytest.raises(VdmiError, match="no CPU path"):
        B.norm_before(torch.zeros(2, 8))


@gpu
def test_more_samples_than_one_launch_takes():
    """A launch has less than 2^32 threads: 2^24 workgroups of 256 and 2^22 of 1024 are more.  Samples at the borders of
    launches against the same samples by themselves; the weight's gradient, which 64 threads add up one sample after the
    other, is off by 2^-24 sqrt(n / 128) of it: 2.2e-5."""
    from video_diffusion_amd import block_hip as B
    n, c = (1 << 24) + 5, 8
    g = torch.Generator(device=DEV).manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    p = {"x": rnd(n, c).to(torch.bfloat16), "h": rnd(n, c).to(torch.bfloat16), "post_weight": None, "gate": None, "weight": 1 + 0.3 * rnd(c),
         "scale": 0.5 * rnd(n, c), "shift": rnd(n, c)}
    dy = rnd(n, c).to(torch.bfloat16)

    def run(rows):
        lv = {k: v if v is None else (v if v.dim() == 1 else v[rows]).detach().requires_grad_() for k, v in p.items()}
        out, y = B.norm_between(*(lv[k] for k in NAMES))
        return out.detach(), y.detach(), *torch.autograd.grad(y, [lv[k] for k in ("x", "h", "scale", "shift", "weight")], dy[rows])

    *got, dw = run(slice(None))
    for at in (0, 1 << 21, 1 << 22, 1 << 23, 1 << 24):
        rows = slice(max(at - 40, 0), at + 40)
        for a, b in zip(got, run(rows)):
            assert torch.equal(a[rows], b)
    s1 = got[4].double() / p["weight"].double()                             # dscale = weight * sum dy n
    assert record("norm.launches.dweight", rel_err(dw, ((1 + p["scale"].double()) * s1).sum(0)), 5e-5) < 5e-5
