"""Activations kept in 8 bits (csrc/rows8.hip; block_hip.pack_rows8, rows8_wgrad, linear_rows8).

Codes and unpacked values are held to equality with a restatement in 64 bits.  The weight gradient is a float32 sum of exact
products: 1e-5 in the 2-norm.  linear_rows8 (bf16 operands, float32 sums, one rounding of the result): u = 2^-8 of the
2-norm for the rounded weights and as much for the result, 2 u."""
import ctypes as C

import pytest
import torch

from tests.helpers import new_graph, record, rel_err
from video_diffusion_amd import _lib

gpu = pytest.mark.gpu
DEV = "cuda:0"


def kept_values(x):
    """(values, exponents) in float64 on the CPU: e the least power of two whose 448 2^e holds the group's largest finite
    magnitude, -118 <= e <= 119; steps of an eighth of the power of two below a value, at least 2^-9 2^e, ties to even."""
    x = x.detach().double().cpu()
    r, c = x.shape
    t = torch.zeros(r, -(-c // 32) * 32, dtype=torch.float64)
    t[:, :c] = x
    t = t.view(r, -1, 32)
    fin = torch.isfinite(t)
    top = torch.where(fin, t.abs(), torch.zeros_like(t)).amax(-1)
    e = torch.full(top.shape, -118, dtype=torch.float64)
    for k in range(-117, 120):
        e = torch.where(top > 448 * 2.0 ** (k - 1), torch.full_like(e, float(k)), e)
    u = torch.exp2(e).unsqueeze(-1)
    a = torch.where(fin, t, torch.zeros_like(t)) / u
    _, ex = torch.frexp(a.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((ex - 4).double())
    v = (torch.round(a / step) * step).clamp(-448, 448) * u             # the clamp: magnitudes beyond 448 2^119
    v = torch.where(fin, v, torch.full_like(v, float("nan")))
    return v.view(r, -1)[:, :c], e


def sample(r, c, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(r, c, generator=g, device=DEV) * torch.exp(2 * torch.randn(c, generator=g, device=DEV))
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("r,c", [(1, 8), (3, 24), (7, 32), (5, 40), (1000, 72), (33, 256), (2, 1000), (129, 2048)])
def test_codes_and_values(r, c, dtype):
    from video_diffusion_amd import block_hip as B
    x = sample(r, c, dtype, r + c)
    kept = B.pack_rows8(x)
    want, e = kept_values(x)
    assert torch.equal(kept.exps.cpu().double() - 127, e)
    assert kept.codes.shape == (r, c) and kept.exps.shape == (r, -(-c // 32))
    assert torch.equal(kept.unpack(torch.float32).cpu().double(), want)
    back = kept.unpack()
    assert back.dtype == dtype and torch.equal(back.cpu(), want.to(dtype))
    assert torch.equal(kept.unpack(torch.bfloat16).cpu().double(), want)        # every code times 2^e is a bfloat16
    # what is kept of a value: half a step of three fraction bits, or of the least code
    assert ((want - x.double().cpu()).abs() <= torch.maximum(x.double().abs().cpu() * 2.0 ** -4,
                                                             2.0 ** (e - 10).repeat_interleave(32, 1)[:, :c])).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_special_values(dtype):
    """Zeros, the largest and least magnitudes of the type, subnormals, infinities, NaN, exact ties, values at the border
    between two exponents."""
    from video_diffusion_amd import block_hip as B
    f = torch.finfo(dtype)
    rows = torch.zeros(12, 64, dtype=torch.float64)
    rows[1, 3] = f.max
    rows[2, 5], rows[2, 40] = -f.max, f.tiny
    rows[3, 0] = f.smallest_normal / 4
    rows[4, 1:4] = torch.tensor([float("inf"), 1.0, -3.0])
    rows[5, 33:36] = torch.tensor([float("nan"), -0.5, 7.0])
    rows[6, :32] = float("-inf")
    rows[7, :16] = torch.arange(16).double() / 16 + 1            # ties between codes of a step of 1/8
    rows[8, 0], rows[8, 32] = 448.0, 449.0 if dtype == torch.float32 else 450.0
    rows[9, 0], rows[9, 1], rows[9, 2] = 448.0, 2.0 ** -10, 3 * 2.0 ** -10      # half steps of the least code
    rows[10, :8] = -0.0
    rows[11, :] = 2.0 ** -125
    x = rows.to(dtype).to(DEV)
    kept = B.pack_rows8(x)
    want, e = kept_values(x)
    assert torch.equal(kept.exps.cpu().double() - 127, e)
    got = kept.unpack(torch.float32).cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0).float().double())


@gpu
def test_layouts():
    from video_diffusion_amd import block_hip as B
    x = sample(60, 320, torch.bfloat16, 1).view(3, 20, 320)
    for name, t in (("pitch", x[..., 8:200]), ("odd", x[..., 3:67]), ("turned", x[..., :64].transpose(0, 1)),
                    ("columns", x[..., :64].transpose(1, 2)[..., :16]), ("expanded", x[:, :1].expand(3, 9, 320))):
        kept = B.pack_rows8(t)
        flat = t.reshape(-1, t.shape[-1])
        assert kept.shape == tuple(t.shape)
        assert torch.equal(kept.unpack().cpu(), kept_values(flat)[0].to(torch.bfloat16).view(t.shape)), name
    empty = B.pack_rows8(x[:0])
    assert empty.unpack().shape == (0, 20, 320)
    assert not B.rows8_wgrad(empty, torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16)).any()


@gpu
@pytest.mark.parametrize("r,c,o", [(1, 8, 8), (5, 40, 16), (63, 128, 128), (64, 136, 64), (65, 64, 264), (1000, 72, 200), (4097, 512, 384),
                                   (300000, 64, 32), (20000, 1000, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weight_and_bias_gradient(r, c, o, dtype):
    from video_diffusion_amd import block_hip as B
    x = sample(r, c, dtype, r)
    dy = sample(r, o, torch.bfloat16, r + 1)
    kept = B.pack_rows8(x)
    dw, db = B.rows8_wgrad(kept, dy, bias=True)
    want = dy.double().t() @ kept.unpack(torch.float32).double()
    assert dw.shape == (o, c) and dw.dtype == torch.float32
    # a bias gradient is a sum of r values that mostly cancel: held against the sum of magnitudes, r 2^-24 of it at most
    assert record(f"rows8.wgrad.{r}x{c}x{o}.{dtype}", rel_err(dw, want), 1e-5) < 1e-5
    slack = (db.double() - dy.double().sum(0)).abs() - 1e-6 * dy.double().abs().sum(0)
    assert float(slack.max()) <= 0
    assert torch.equal(dw, B.rows8_wgrad(kept, dy))
    pitched = torch.zeros(r, o + 24, device=DEV, dtype=torch.bfloat16)
    pitched[:, 8:8 + o] = dy
    assert torch.equal(dw, B.rows8_wgrad(kept, pitched[:, 8:8 + o]))
    pitched[:, 3:3 + o] = dy
    assert torch.equal(dw, B.rows8_wgrad(kept, pitched[:, 3:3 + o]))


@gpu
@pytest.mark.parametrize("shape,o", [((2, 50, 64), 128), ((3, 7, 96), 32), ((4, 33, 17, 128), 384), ((1, 256), 32)])
def test_linear(shape, o):
    """The layer against float64: output, input gradient, weight gradient from the kept values, bias gradient."""
    from video_diffusion_amd import block_hip as B
    g = torch.Generator(device=DEV).manual_seed(o)
    x = torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    w = (torch.randn(o, shape[-1], generator=g, device=DEV) * shape[-1] ** -0.5).requires_grad_()
    b = torch.randn(o, generator=g, device=DEV).requires_grad_()
    dy = torch.randn(*shape[:-1], o, generator=g, device=DEV).to(torch.bfloat16)
    y = B.linear_rows8(x, w, b)
    want = x.detach().double() @ w.detach().double().t() + b.detach().double()
    assert y.dtype == torch.bfloat16 and rel_err(y.detach(), want) < 2 * 2.0 ** -8
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert rel_err(dx, dy.double() @ w.detach().double()) < 2 * 2.0 ** -8
    kept = B.pack_rows8(x).unpack(torch.float32).double().reshape(-1, shape[-1])
    d2 = dy.double().reshape(-1, o)
    assert rel_err(dw, d2.t() @ kept) < 1e-5 and rel_err(db, d2.sum(0)) < 1e-5
    # 8 bits against the rows themselves: a value is off by 2^-4 of itself at most, 2^-4 / sqrt(3) evenly spread
    assert rel_err(dw, d2.t() @ x.detach().double().reshape(-1, shape[-1])) < 2.0 ** -4 / 3 ** 0.5
    (only,) = torch.autograd.grad(B.linear_rows8(x.detach(), w, None), w, dy)
    assert torch.equal(only, dw)


@gpu
def test_what_a_linear_keeps():
    """Memory held between forward and backward: codes and exponents in place of the rows."""
    from video_diffusion_amd import block_hip as B
    x = torch.randn(65536, 512, device=DEV).to(torch.bfloat16)
    w = torch.randn(64, 512, device=DEV, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = B.linear_rows8(x, w)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= 65536 * (512 + 16) + (1 << 16)
    y.sum().backward()


@gpu
def test_graph_and_streams():
    from video_diffusion_amd import block_hip as B
    x, dy = sample(3000, 128, torch.bfloat16, 2), sample(3000, 256, torch.bfloat16, 3)

    def run():
        k = B.pack_rows8(x)
        return [k.unpack(), *B.rows8_wgrad(k, dy, bias=True)]

    want = run()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    res = []
    for s in streams:
        with torch.cuda.stream(s):
            res.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in res for a, b in zip(r, want))
    graph = new_graph()
    with torch.cuda.graph(graph):
        outs = run()
    for seed in range(3):
        x.copy_(sample(3000, 128, torch.bfloat16, 10 + seed))
        dy.copy_(sample(3000, 256, torch.bfloat16, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


@gpu
def test_offsets_beyond_32_bits():
    """5.1e9 elements: the first and last rows against the same rows by themselves."""
    from video_diffusion_amd import block_hip as B
    rows, c = 620000, 8192
    x = torch.zeros(rows, c, device=DEV, dtype=torch.bfloat16)
    ends = sample(64, c, torch.bfloat16, 4)
    x[:32], x[-32:] = ends[:32], ends[32:]
    kept, want = B.pack_rows8(x), B.pack_rows8(ends)
    del x
    at = lambda t: torch.cat((t[:32], t[-32:]))
    assert torch.equal(at(kept.codes), want.codes) and torch.equal(at(kept.exps), want.exps)
    assert torch.equal(at(kept.unpack()), want.unpack())
    dy = torch.zeros(rows, 32, device=DEV, dtype=torch.bfloat16)
    dy[:32] = 1
    dy[-32:] = torch.randn(32, 32, device=DEV).to(torch.bfloat16)
    dw = B.rows8_wgrad(kept, dy)
    assert rel_err(dw, at(dy).double().t() @ want.unpack(torch.float32).double()) < 1e-5


@gpu
def test_no_second_derivative():
    from video_diffusion_amd import block_hip as B
    x = torch.randn(5, 64, device=DEV).to(torch.bfloat16).requires_grad_()
    (g,) = torch.autograd.grad(B.linear_rows8(x, torch.randn(32, 64, device=DEV)).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


def test_entry_points_refuse_bad_arguments():
    lib = _lib.lib()
    E_ARG, E_SHAPE, E_ALIGN = -1, -2, -3
    for f, p in ((lib.vdmi_rows8_pack, lambda x, l, c, e, *r: (x, l, c, e, *r)), (lib.vdmi_rows8_unpack, lambda x, l, c, e, *r: (c, e, x, l, *r))):
        assert f(*p(None, 64, 16, 16, 0, 10, 64), None) == E_ARG
        assert f(*p(16, 64, None, 16, 0, 10, 64), None) == E_ARG
        assert f(*p(16, 64, 16, 16, 3, 10, 64), None) == E_ARG
        assert f(*p(16, 64, 16, 16, 0, 0, 64), None) == E_SHAPE
        assert f(*p(16, 64, 16, 16, 0, 10, 60), None) == E_SHAPE
        assert f(*p(16, 56, 16, 16, 0, 10, 64), None) == E_SHAPE
        assert f(*p(16, 68, 16, 16, 0, 10, 64), None) == E_SHAPE
        assert f(*p(16, 64, 16, 16, 0, 1 << 40, 64), None) == E_SHAPE
        assert f(*p(24, 64, 16, 16, 0, 10, 64), None) == E_ALIGN
        assert f(*p(16, 64, 20, 16, 0, 10, 64), None) == E_ALIGN
    assert lib.vdmi_rows8_wgrad_workspace_bytes(60, 64, 100) == 0 and lib.vdmi_rows8_wgrad_workspace_bytes(64, 64, 0) == 0
    assert lib.vdmi_rows8_wgrad_workspace_bytes(64, 64, 100) > 0
    w = lambda *a: lib.vdmi_rows8_wgrad(*a, None)
    assert w(None, 16, 16, 64, 16, None, 64, 64, 100, 16) == E_ARG
    assert w(16, 16, 16, 64, 16, None, 64, 64, 100, None) == E_ARG
    assert w(16, 16, 16, 64, 16, None, 60, 64, 100, 16) == E_SHAPE
    assert w(16, 16, 16, 56, 16, None, 64, 64, 100, 16) == E_SHAPE
    assert w(16, 16, 24, 64, 16, None, 64, 64, 100, 16) == E_ALIGN
    assert w(16, 16, 16, 64, 16, None, 64, 64, 100, 24) == E_ALIGN


@gpu
def test_python_entry_points_refuse():
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    kept = B.pack_rows8(x)
    w = torch.zeros(32, 64, device=DEV)
    for f, what in [(lambda: B.pack_rows8(x.double()), "bfloat16"), (lambda: B.pack_rows8(x[:, :60]), "multiple of 8"),
                    (lambda: B.pack_rows8(x.cpu()), "no CPU path"), (lambda: kept.unpack(torch.int8), "bfloat16"),
                    (lambda: B.rows8_wgrad(kept, x.float()), "dy is bfloat16"), (lambda: B.rows8_wgrad(kept, x[:3]), "a row for each"),
                    (lambda: B.rows8_wgrad(kept, x[:, :60]), "multiple of 8"), (lambda: B.linear_rows8(x.float(), w), "x is bfloat16"),
                    (lambda: B.linear_rows8(x, w.half()), "weight float32"), (lambda: B.linear_rows8(x, w[:, :32]), "cin"),
                    (lambda: B.linear_rows8(x, w, w[0]), "bias"), (lambda: B.linear_rows8(x, w[:20]), "multiples of 32"),
                    # shapes that the row GEMMs do not take, forward (cout) or towards the input (cin)
                    (lambda: B.linear_rows8(torch.zeros(3, 7, 72, device=DEV, dtype=torch.bfloat16), torch.zeros(40, 72, device=DEV)),
                     "multiples of 32"),
                    (lambda: B.linear_rows8(torch.zeros(1, 256, device=DEV, dtype=torch.bfloat16), torch.zeros(8, 256, device=DEV)),
                     "multiples of 32")]:
        with pytest.raises(VdmiError, match=what):
            f()


@gpu
def test_the_largest_halfs():
    """Rows of finite halfs come back finite: what their codes stand for, at most 65504; infinities and NaN as NaN."""
    from video_diffusion_amd import block_hip as B
    x = torch.tensor([[65504.0, 63488.0, 63456.0, 61440.0, 3.0, 0.0, -1e-7, 448.0], [-65504.0, -63488.0, -63456.0, 57344.0, 2.0, 1.0, 0.5, 0.25],
                      [float("inf"), 65504.0, float("nan"), -65504.0, 1.0, 2.0, 3.0, 4.0]], device=DEV).half()
    kept = B.pack_rows8(x)
    values = kept_values(x)[0]
    assert float(values.abs().nan_to_num().max()) == 65536.0                # the code next to the largest half
    assert torch.equal(torch.nan_to_num(kept.unpack(torch.float32).cpu().double(), nan=7e7), torch.nan_to_num(values, nan=7e7))
    got, want = kept.unpack().cpu().double(), values.clamp(-65504, 65504)
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x.cpu()))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))
    fin = torch.isfinite(x.cpu())
    assert ((got - x.cpu().double()).abs()[fin] <= (x.cpu().double().abs() * 2.0 ** -4).clamp(min=2.0 ** -2)[fin]).all()


@gpu
def test_what_is_lost_of_the_smallest_values():
    """The documented bound: 2^-4 of a value, or under 2^-17 of its group's largest (2^-128 where that is below 224 2^-118)."""
    from video_diffusion_amd import block_hip as B
    x = torch.zeros(64, 32, dtype=torch.float64)
    for r in range(64):
        x[r, 0] = 224.0 * (1 + 2.0 ** -7) * 2.0 ** (r - 40)             # just above the border to the next exponent
        x[r, 1:] = x[r, 0] * 2.0 ** -17.8 * torch.linspace(0.2, 1.2, 31, dtype=torch.float64)
    x[:8] *= 2.0 ** -100
    x = x.float()
    got, want = B.pack_rows8(x.to(DEV)).unpack().cpu().double(), x.double()
    top = want.abs().amax(1, keepdim=True)
    off = (got - want).abs()
    assert (off <= torch.maximum(want.abs() * 2.0 ** -4, torch.maximum(top * 2.0 ** -17, torch.tensor(2.0 ** -128)))).all()
    assert (off > torch.maximum(want.abs() * 2.0 ** -4, top * 2.0 ** -18)).any()            # 2^-18 would not hold


@gpu
@pytest.mark.parametrize("n", [64, 96])
def test_a_weight_and_its_transpose_within_fixed_weights(n):
    """One square parameter as w and as w.t(): the same memory and shape, two weight sets."""
    from video_diffusion_amd import block_hip as B, train_hip as T
    g = torch.Generator(device=DEV).manual_seed(n)
    w = (torch.randn(n, n, generator=g, device=DEV) * n ** -0.5).requires_grad_()
    x = torch.randn(50, n, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(50, n, generator=g, device=DEV).to(torch.bfloat16)
    want = [(y, *torch.autograd.grad(y, (x, w), dy)) for y in (B.linear_rows8(x, w), B.linear_rows8(x, w.t()))]
    with T.fixed_weights(T.PackStore()):
        got = [(y, *torch.autograd.grad(y, (x, w), dy)) for y in (B.linear_rows8(x, w), B.linear_rows8(x, w.t()))]
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert rel_err(got[1][0].detach(), x.detach().double() @ w.detach().double()) < 2 * 2.0 ** -8


@gpu
@pytest.mark.parametrize("start", [1, 3, 8])
def test_linear_of_rows_at_any_address(start):
    """Input, weight, bias and gradient that begin `start` elements into their memory."""
    from video_diffusion_amd import block_hip as B

    def at(t):
        m = torch.zeros(t.numel() + start, device=DEV, dtype=t.dtype)
        m[start:] = t.reshape(-1)
        return m[start:].view(t.shape)

    g = torch.Generator(device=DEV).manual_seed(start)
    x = torch.randn(5, 11, 64, generator=g, device=DEV).to(torch.bfloat16)
    w, b = torch.randn(96, 64, generator=g, device=DEV) / 8, torch.randn(96, generator=g, device=DEV)
    dy = torch.randn(5, 11, 96, generator=g, device=DEV).to(torch.bfloat16)

    def run(*ts):
        ins = [t.detach().requires_grad_() for t in ts[:3]]
        y = B.linear_rows8(*ins)
        return (y.detach(), *torch.autograd.grad(y, ins, ts[3]))

    for a, e in zip(run(at(x), at(w), at(b), at(dy)), run(x, w, b, dy)):
        assert torch.equal(a, e)


@gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_packed_where_no_backward_can_follow(mode, monkeypatch):
    """Parameters ask for gradients while a model samples, too."""
    from video_diffusion_amd import block_hip as B
    x = torch.randn(40, 64, device=DEV).to(torch.bfloat16)
    w, b = (torch.randn(96, 64, device=DEV) / 8).requires_grad_(), torch.randn(96, device=DEV).requires_grad_()
    packs = []
    real = B.pack_rows8
    monkeypatch.setattr(B, "pack_rows8", lambda t: packs.append(t.shape) or real(t))
    want = B.linear_rows8(x, w, b)
    assert len(packs) == 1 and want.requires_grad
    with mode():
        got = B.linear_rows8(x, w, b)
    assert len(packs) == 1 and not got.requires_grad and torch.equal(got, want)
    assert B.linear_rows8(x.requires_grad_(), w.detach()).requires_grad and len(packs) == 1


def test_calls_beyond_one_launch_are_refused():
    """2^32 threads of eight channels each, or of the shares' sums: refused on the host."""
    lib = _lib.lib()
    assert lib.vdmi_rows8_pack(16, 64, 16, 16, 0, 1 << 29, 64, None) == -2
    assert lib.vdmi_rows8_unpack(16, 16, 16, 64, 0, 1 << 29, 64, None) == -2
    assert lib.vdmi_rows8_pack(16, 8, 16, 16, 0, 1 << 30, 8, None) == -2       # three of four threads of a group are idle
    assert lib.vdmi_rows8_wgrad_workspace_bytes(1 << 16, 1 << 16, 64) == 0
    assert lib.vdmi_rows8_wgrad(16, 16, 16, 1 << 16, 16, None, 1 << 16, 1 << 16, 64, 16, None) == -2
    assert lib.vdmi_rows8_wgrad_workspace_bytes(1 << 15, 1 << 15, 64) > 0


@gpu
@pytest.mark.parametrize("rows,o", [(40, 64), (200000, 256), (300000, 32)])
def test_bias_gradient_of_a_frozen_weight(rows, o):
    """The bias gradient alone, eager and from a graph that is replayed with eager work in between."""
    from video_diffusion_amd import block_hip as B
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, w = torch.randn(rows, 64, generator=g, device=DEV).to(torch.bfloat16), torch.randn(o, 64, generator=g, device=DEV) / 8
    b = torch.randn(o, generator=g, device=DEV).requires_grad_()
    dy = torch.randn(rows, o, generator=g, device=DEV).to(torch.bfloat16)

    def run():
        return torch.autograd.grad(B.linear_rows8(x, w, b), b, dy)[0]

    def check(db):
        slack = (db.double() - dy.double().sum(0)).abs() - 1e-6 * dy.double().abs().sum(0)
        assert float(slack.max()) <= 0

    check(run())
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = new_graph()
    with torch.cuda.graph(graph):
        db = run()
    for _ in range(4):
        dy.copy_(torch.randn(rows, o, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        check(db)
        assert torch.equal(db, run())


@gpu
def test_tensors_without_dimensions_are_refused():
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    one = torch.zeros((), device=DEV, dtype=torch.bfloat16)
    kept = B.pack_rows8(torch.zeros(1, 8, device=DEV, dtype=torch.bfloat16))
    for f in (lambda: B.pack_rows8(one), lambda: B.rows8_wgrad(kept, one), lambda: B.linear_rows8(one, torch.zeros(32, 32, device=DEV))):
        with pytest.raises(VdmiError, match=r"\(\)|no dimensions"):
            f()
