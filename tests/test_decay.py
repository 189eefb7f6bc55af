"""Attention over time with a decay per head (csrc/decay.hip, block_hip.decay_attention / decay_attention_step) against the
definition in 64 bits.

Tolerances, set before the first run.  u = half a step of the element type (bf16 2^-8, fp16 2^-11).  A kernel rounds the
weighted pairs (or the state) once as a matrix operand and the result once, so an output element is off by at most
u (A + |o|), A the same sum with absolute values; 2^-16 A more covers float32 sums.  In the 2-norm the roundings are
independent, each u / sqrt(3) of what it rounds at most: 1.25 u.  A state sees products of sums of 16-bit operands (2^-16
of them may be lost) and float32 sums: 1e-5 in the 2-norm."""
import ctypes as C

import pytest
import torch

from tests.helpers import new_graph, record, rel_err
from video_diffusion_amd import _lib

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(q, k, v, g, s0, lengths, scale, do=None, ds=None):
    """(o, last state[, dq, dk, dv, ds0]) in float64 by pairs over the whole sequence, and the bounds A of o, dq, dk, dv.
    q, k, v [B, n, h, d]."""
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))              # [B, h, n, d]
    B, h, n, d = q.shape
    g = g.double()
    t = torch.arange(n, dtype=torch.float64, device=q.device)
    L = torch.full((B,), n, dtype=torch.float64, device=q.device) if lengths is None else lengths.reshape(-1).double().clamp(0, n)
    live = (t[None] < L[:, None]).double()[:, None, :, None]
    gap = t[:, None] - t[None, :]
    D = torch.where(gap >= 0, torch.exp(g.view(h, 1, 1) * gap.clamp(min=0)), torch.zeros((), dtype=torch.float64, device=q.device))
    into = torch.exp(g.view(h, 1) * (t + 1))[None, :, :, None]
    left = (torch.exp(g.view(1, h, 1) * (L[:, None] - 1 - t).clamp(min=0)[:, None]))[..., None] * live
    whole = torch.exp(g.view(1, h) * L[:, None])[..., None, None]
    s = torch.zeros(B, h, d, d, dtype=torch.float64, device=q.device) if s0 is None else s0.double().reshape(B, h, d, d)
    q, k, v = (torch.where(live > 0, x, torch.zeros_like(x)) for x in (q, k, v))

    def attn(q, k, v, s):
        return scale * live * (((q @ k.mT) * D) @ v + into * (q @ s))

    back = lambda x: x.transpose(1, 2)
    res = [back(attn(q, k, v, s)), whole * s + (left * k).mT @ v]
    bound = [back(attn(q.abs(), k.abs(), v.abs(), s.abs())).abs()]
    if do is not None:
        e = scale * live * torch.where(live > 0, do.double().transpose(1, 2), torch.zeros_like(q))
        r = torch.zeros_like(s) if ds is None else ds.double().reshape(B, h, d, d)

        def grads(q, k, v, e, s, r):
            a, p = (e @ v.mT) * D, (q @ k.mT) * D
            return a @ k + into * (e @ s.mT), a.mT @ q + left * (v @ r.mT), p.mT @ e + left * (k @ r)

        res += [back(x) for x in grads(q, k, v, e, s, r)] + [whole * r + (into * q).mT @ e]
        ab = torch.abs
        # with absolute values all the way down the pairs' sums stay above the kernel's roundings of them
        bound += [back(x).abs() for x in grads(ab(q), ab(k), ab(v), ab(e), ab(s), ab(r))]
    return res, bound


def close(name, got, want, A, u):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), name
    slack = (got.detach() - want).abs() - (u * (A + want.abs()) + 2.0 ** -16 * A + 1e-30)
    assert float(slack.max()) <= 0, (name, float(slack.max()))
    if want.norm() > 0:
        err = record("decay." + name, rel_err(got, want), 1.25 * u)
        assert err < 1.25 * u, (name, err)


def inputs(b, s, n, h, d, dtype, seed, state=False, ragged=False, layout="rows"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *sh: torch.randn(*sh, generator=g, device=DEV)
    if layout == "rows":            # (batch, time, site) rows of a qkv projection
        qkv = rnd(b, n, s, 3, h, d).to(dtype)
        q, k, v = (t.permute(0, 2, 1, 3, 4) for t in qkv.unbind(3))
        do = rnd(b, n, s, h, d).to(dtype).permute(0, 2, 1, 3, 4)
    elif layout == "heads":         # heads before time, as softmax attention cores take them
        q, k, v, do = (rnd(b, s, h, n, d).to(dtype).transpose(2, 3) for _ in range(4))
    elif layout == "odd":           # rows of an odd pitch: read from a copy
        q, k, v, do = (rnd(b, s, n, h, d + 1).to(dtype)[..., 1:] for _ in range(4))
    else:                           # one value for all sites and heads
        q, do = (rnd(b, s, n, h, d).to(dtype) for _ in range(2))
        k, v = (rnd(b, 1, n, 1, d).to(dtype).expand(b, s, n, h, d) for _ in range(2))
    decay = torch.log1p(-torch.exp2(-torch.linspace(1, 9, h, device=DEV)))
    st = rnd(b, s, h, d, d) if state else None
    ds = rnd(b, s, h, d, d) if state else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, n + 1, (b, s), generator=g, device=DEV, dtype=torch.int32)
        lengths.view(-1)[0] = n
        lengths.view(-1)[-1] = 0
    return q, k, v, do, decay, st, ds, lengths


def check_all(case, q, k, v, do, decay, st, ds, lengths, scale=None):
    from video_diffusion_amd import block_hip as B
    b, s, n, h, d = q.shape
    u = U[q.dtype]
    m = d ** -0.5 if scale is None else scale
    flat = lambda t: None if t is None else t.reshape(b * s, *t.shape[2:])
    (o, last, dq, dk, dv, ds0), bd = reference(flat(q), flat(k), flat(v), decay, flat(st), lengths, m, flat(do), flat(ds))
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    s0 = None if st is None else st.detach().requires_grad_()
    kw = dict(scale=scale, initial_state=s0, lengths=lengths)
    if st is None:
        got = B.decay_attention(*ins, decay, **kw)
        grads = torch.autograd.grad(got, ins, do)
    else:
        got, gl = B.decay_attention(*ins, decay, return_state=True, **kw)
        *grads, gs = torch.autograd.grad((got, gl), (*ins, s0), (do, ds))
        assert record(f"decay.{case}.state", rel_err(flat(gl), last), 1e-5) < 1e-5
        assert record(f"decay.{case}.dstate", rel_err(flat(gs), ds0), 1e-5) < 1e-5
    assert got.shape == q.shape and got.dtype == q.dtype
    for name, x, w, A in zip(("o", "dq", "dk", "dv"), (got, *grads), (o, dq, dk, dv), bd):
        close(f"{case}.{name}", flat(x), w, A, u)
    if lengths is not None:
        pad = torch.arange(n, device=DEV)[None] >= lengths.reshape(-1, 1)
        for x in (got, *grads):
            assert not flat(x)[pad].any()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 5, 10, 16, 17, 31, 32])
def test_short_sequences(n, d, dtype):
    """Sequences that share a tile of 32 rows (forward and the one-launch backward); counts that leave the last tile
    partly empty."""
    check_all(f"short.n{n}.d{d}.{dtype}", *inputs(2, 7, n, 3, d, dtype, 10 * n + d))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 100, 300])
def test_states_in_and_out(n, d, dtype):
    check_all(f"states.n{n}.d{d}.{dtype}", *inputs(2, 1, n, 3, d, dtype, n + d, state=True))


@gpu
@pytest.mark.parametrize("n", [33, 129])
@pytest.mark.parametrize("layout", ["rows", "heads", "odd", "expanded"])
@pytest.mark.parametrize("state", [False, True])
def test_layouts(layout, n, state):
    check_all(f"layout.{layout}.n{n}.{state}", *inputs(2, 3, n, 2, 32, torch.bfloat16, n, state=state, layout=layout))
    check_all(f"layout.{layout}.n9.{state}", *inputs(2, 3, 9, 2, 64, torch.bfloat16, n, state=state, layout=layout))


@gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n,state", [(12, False), (32, False), (70, False), (70, True), (1100, True)])
def test_ragged_batches(n, state, d):
    """lengths from zero to n in a padded batch whose padding holds NaN: never read, outputs and gradients zero there."""
    q, k, v, do, decay, st, ds, lengths = inputs(3, 2, n, 2, d, torch.bfloat16, n + d, state=state, ragged=True)
    pad = (torch.arange(n, device=DEV)[None, None] >= lengths[..., None])
    for t in (q, k, v, do):
        t.masked_fill_(pad[..., None, None], float("nan"))
    check_all(f"ragged.n{n}.d{d}.{state}", q, k, v, do, decay, st, ds, lengths)


@gpu
@pytest.mark.parametrize("d,n", [(32, 2048), (32, 2047), (64, 4000), (128, 3001)])
@pytest.mark.parametrize("state,ragged", [(False, False), (True, False), (True, True)])
def test_segments(d, n, state, ragged):
    """Few long sequences: the time axis is cut into segments."""
    a = _lib.DecayArgs()
    a.b, a.inner, a.n, a.heads, a.d, a.scale, a.log_decay = 2, 1, n, 2, d, 1.0, 16
    for f in ("q", "k", "v"):
        setattr(a, f, _lib.Rows4(16, 0, 0, d * 2, d))
    assert _lib.lib().vdmi_decay_attn_workspace_bytes(C.byref(a)) > 0
    check_all(f"segments.n{n}.d{d}.{state}.{ragged}", *inputs(2, 1, n, 2, d, torch.bfloat16, n, state=state, ragged=ragged))


@gpu
@pytest.mark.parametrize("n", [8, 200])
def test_extreme_decays_and_scales(n):
    """No decay at all, decays that underflow within a tile, an infinite one (only the token itself is seen), scales."""
    q, k, v, do, _, st, ds, _ = inputs(1, 3, n, 4, 32, torch.bfloat16, 5, state=True)
    decay = torch.tensor([0.0, -3.0, -200.0, float("-inf")], device=DEV)
    ref = decay.clone()
    ref[3] = -1e4                               # exp(-1e4) is zero in 64 bits too, without 0 * inf at a token's own place
    for scale in (1.0, -0.25, 3.0):
        from video_diffusion_amd import block_hip as B
        got, last = B.decay_attention(q, k, v, decay, scale=scale, initial_state=st, return_state=True)
        same, last2 = B.decay_attention(q, k, v, ref, scale=scale, initial_state=st, return_state=True)
        assert torch.equal(got, same) and torch.equal(last, last2)
        check_all(f"extreme.n{n}.{scale}", q, k, v, do, ref, st, ds, None, scale)
        check_all(f"extreme.short.n{n}.{scale}", q, k, v, do, ref, None, None, None, scale)


@gpu
def test_rows_that_are_not_finite_stay_in_their_sequence():
    """Sequences that share a tile: an infinity or NaN in one of them does not reach the others, forward or backward, and
    later tokens do not reach the pairs of earlier ones through the mask."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, *_ = inputs(2, 9, 6, 2, 32, torch.bfloat16, 3)
    clean = [t.clone() for t in (q, k, v, do)]

    def run(q, k, v, do):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        o = B.decay_attention(*ins, decay)
        return [o, *torch.autograd.grad(o, ins, do)]

    want = run(*clean)
    others = torch.ones(2, 9, dtype=torch.bool, device=DEV)
    others[0, 3] = others[1, 8] = False
    for which in range(4):
        bad = [t.clone() for t in clean]
        bad[which][0, 3, 5] = float("nan")
        bad[which][1, 8, 2, 1, 7] = float("inf")
        for got, w in zip(run(*bad), want):
            assert torch.equal(got[others], w[others])
    bad = [t.clone() for t in clean]
    bad[1][0, 3, 5] = float("nan")              # a key of the last token: no pair of an earlier query is touched
    o = run(*bad)[0]
    assert torch.equal(o[0, 3, :5], want[0][0, 3, :5]) and torch.isnan(o[0, 3, 5]).all()


@gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead", [(1,), (3,), (5, 7), ()])
def test_step(lead, d, dtype):
    """A step against the definition; then a whole sequence as steps against the scan (outputs and state)."""
    from video_diffusion_amd import block_hip as B
    g = torch.Generator(device=DEV).manual_seed(d)
    h = 3
    decay = torch.tensor([-0.3, -0.01, 0.0], device=DEV)
    state = torch.randn(*lead, h, d, d, generator=g, device=DEV)
    qkv = torch.randn(*lead, 3, h, d, generator=g, device=DEV).to(dtype)
    q, k, v = qkv.unbind(-3)
    want_s = torch.exp(decay.double())[:, None, None] * state.double() + k.double()[..., :, None] * v.double()[..., None, :]
    want = (q.double()[..., None, :] @ want_s)[..., 0, :] * d ** -0.5
    A = (q.double().abs()[..., None, :] @ want_s.abs())[..., 0, :] * d ** -0.5
    o = B.decay_attention_step(q, k, v, decay, state)
    assert rel_err(state, want_s) < 2.0 ** -21                  # one product and one sum in float32
    # the result is rounded once, a sum of d float32 products (d 2^-24 A) before it
    assert ((o.double() - want).abs() <= U[dtype] * want.abs() + d * 2.0 ** -23 * A).all()


@gpu
def test_steps_follow_a_sequence():
    from video_diffusion_amd import block_hip as B
    q, k, v, _, decay, *_ = inputs(2, 3, 40, 2, 64, torch.bfloat16, 8)
    o, last = B.decay_attention(q, k, v, decay, return_state=True)
    first, state = B.decay_attention(q[:, :, :33], k[:, :, :33], v[:, :, :33], decay, return_state=True)
    # a piece's outputs do not depend on what follows it
    assert torch.equal(first, o[:, :, :33])
    (want, _), (A,) = reference(*(t.flatten(0, 1) for t in (q, k, v)), decay, None, None, 64 ** -0.5)
    for t in range(33, 40):
        got = B.decay_attention_step(q[:, :, t], k[:, :, t], v[:, :, t], decay, state)
        close(f"step{t}", got.flatten(0, 1), want[:, t], A[:, t], U[torch.bfloat16])
    assert rel_err(state, last) < 1e-5
    # the rest of the sequence from the state, as one piece
    _, mid = B.decay_attention(q[:, :, :33], k[:, :, :33], v[:, :, :33], decay, return_state=True)
    rest, end = B.decay_attention(q[:, :, 33:], k[:, :, 33:], v[:, :, 33:], decay, initial_state=mid, return_state=True)
    close("pieces", rest.flatten(0, 1), want[:, 33:], A[:, 33:], U[torch.bfloat16])
    assert rel_err(end, last) < 1e-5


@gpu
@pytest.mark.parametrize("n,state", [(9, False), (40, True)])
def test_gradients_against_differences(n, state):
    """Directional derivative of a fixed functional against central differences of the float64 definition (whose slope is
    exact up to 1e-6): the gradient's roundings give at most 1.25 u of the norms' product."""
    q, k, v, do, decay, st, ds, _ = inputs(1, 2, n, 2, 32, torch.float16, 4, state=state)
    from video_diffusion_amd import block_hip as B
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = B.decay_attention(*ins, decay, initial_state=st, return_state=False)
    grads = torch.autograd.grad(o, ins, do)
    flat = lambda t: None if t is None else t.flatten(0, 1).double()
    g = torch.Generator(device=DEV).manual_seed(1)
    for i in range(3):
        p = torch.randn(q.shape, generator=g, device=DEV, dtype=torch.float64)
        val = []
        for e in (1e-4, -1e-4):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + e * p
            (y, _), _ = reference(*(flat(t) for t in x), decay, flat(st), None, 32 ** -0.5)
            val.append(float((y * flat(do)).sum()))
        slope = (val[0] - val[1]) / 2e-4
        assert abs(float((grads[i].double() * p).sum()) - slope) < 1.25 * U[torch.float16] * float(grads[i].double().norm() * p.norm())


@gpu
def test_gradient_forms():
    """Gradients of some inputs only, of the state alone, of an output nobody uses; a gradient of another dtype or
    broadcast strides."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(2, 1, 45, 2, 32, torch.bfloat16, 6, state=True)
    (_, _, dq, dk, dv, ds0), _ = reference(*(t[:, 0] for t in (q, k, v)), decay, st[:, 0], None, 32 ** -0.5, torch.ones_like(do[:, 0]))
    kr = k.detach().requires_grad_()
    B.decay_attention(q, kr, v, decay, initial_state=st).sum().backward()             # an expanded gradient of ones
    assert rel_err(kr.grad[:, 0], dk) < 1.25 * 2.0 ** -8
    sr = st.detach().requires_grad_()
    B.decay_attention(q, k, v, decay, initial_state=sr)[:, :, :, :].float().sum().backward()
    assert rel_err(sr.grad[:, 0], ds0) < 1e-5
    vr = v.detach().requires_grad_()
    _, last = B.decay_attention(q, k, vr, decay, return_state=True)
    (got,) = torch.autograd.grad(last, vr, ds)
    (_, _, _, _, want, _), _ = reference(*(t[:, 0] for t in (q, k, v)), decay, None, None, 32 ** -0.5, torch.zeros_like(do[:, 0]), ds[:, 0])
    assert rel_err(got[:, 0], want) < 1.25 * 2.0 ** -8


@gpu
def test_same_bits_and_other_streams():
    """Repeated calls give the same bits (no atomics); calls on a side stream after an event, two at once."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 1, 3000, 2, 64, torch.bfloat16, 2, state=True)

    def run():
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        o, s = B.decay_attention(*ins, decay, initial_state=st, return_state=True)
        return [o, s, *torch.autograd.grad((o, s), ins, (do, ds))]

    want = run()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))


@gpu
@pytest.mark.parametrize("n,state", [(10, False), (1500, True)])
def test_captured_and_replayed(n, state):
    """Forward, backward and a step in one graph, replayed with eager work in between and new inputs."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 2, n, 2, 32, torch.bfloat16, 12, state=state)
    q, k, v, do = (t.contiguous() for t in (q, k, v, do))
    step_state = torch.randn(2, 2, 32, 32, device=DEV)

    def run():
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        o = B.decay_attention(*ins, decay, initial_state=st)
        x = B.decay_attention_step(q[0, :, 0], k[0, :, 0], v[0, :, 0], decay, step_state)
        return [o.detach(), x, *torch.autograd.grad(o, ins, do)]

    run()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = new_graph()
    with torch.cuda.graph(graph):
        outs = run()
    g = torch.Generator(device=DEV).manual_seed(77)
    for _ in range(3):
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        start = step_state.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in outs], step_state.clone()
        step_state.copy_(start)
        want = run()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(after, step_state)


@gpu
def test_offsets_beyond_32_bits():
    """Token rows whose offsets pass 2^31 elements (4.4 GB of rows)."""
    pitch, n = 1 << 20, 2100
    big = torch.zeros(n * pitch, device=DEV, dtype=torch.bfloat16)
    rows = big.view(n, pitch)
    g = torch.Generator(device=DEV).manual_seed(9)
    rows[:, :192] = torch.randn(n, 192, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = (rows[:, 64 * i:64 * i + 64].view(1, 1, n, 2, 32) for i in range(3))
    assert q.data_ptr() == big.data_ptr()
    from video_diffusion_amd import block_hip as B
    decay = torch.tensor([-0.01, -0.2], device=DEV)
    o = B.decay_attention(q, k, v, decay)
    (want, _), (A,) = reference(*(t[0] for t in (q, k, v)), decay, None, None, 32 ** -0.5)
    close("offsets", o[0], want, A, 2.0 ** -8)


@gpu
@pytest.mark.parametrize("inner", [1, 2, 3, 7, 64, 1000, 4097])
def test_many_sites(inner):
    """Short sequences find their rows by a division by the number of sites."""
    q, k, v, do, decay, *_ = inputs(3, inner, 5, 1, 32, torch.bfloat16, inner)
    check_all(f"sites.{inner}", q, k, v, do, decay, None, None, None)


@gpu
def test_pitches_beyond_the_kernels():
    """Token strides of more than 2^25 elements are read from a copy."""
    big = torch.zeros(3 * (1 << 25) + 3 * 4096, device=DEV, dtype=torch.bfloat16)
    t = big.as_strided((1, 1, 3, 2, 32), (0, 0, (1 << 25) + 1024, 32, 1))
    t.copy_(torch.randn(1, 1, 3, 2, 32, device=DEV))
    check_all("pitch", t, t, t, t, torch.tensor([-0.1, -0.5], device=DEV), None, None, None)


@gpu
def test_no_tokens_and_no_sequences():
    from video_diffusion_amd import block_hip as B
    decay = torch.zeros(2, device=DEV)
    q = torch.zeros(3, 0, 2, 32, device=DEV, dtype=torch.bfloat16)
    s0 = torch.randn(3, 2, 32, 32, device=DEV)
    o, s = B.decay_attention(q, q, q, decay, initial_state=s0, return_state=True)
    assert o.shape == q.shape and torch.equal(s, s0) and s.data_ptr() != s0.data_ptr()
    q = torch.zeros(0, 5, 2, 32, device=DEV, dtype=torch.bfloat16)
    o, s = B.decay_attention(q, q, q, decay, return_state=True)
    assert o.shape == q.shape and s.shape == (0, 2, 32, 32)
    assert B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], decay, s).shape == (0, 2, 32)


@gpu
def test_state_of_a_call_without_tokens():
    from video_diffusion_amd import block_hip as B
    q = torch.zeros(3, 0, 2, 32, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    s0 = torch.randn(3, 2, 32, 32, device=DEV, requires_grad=True)
    dq, ds = torch.autograd.grad(B.decay_attention(q, q, q, torch.zeros(2, device=DEV), initial_state=s0).sum(), (q, s0))
    assert dq.shape == q.shape and not ds.any()


@gpu
def test_a_state_kept_for_the_backward_and_stepped():
    """decay_attention_step writes the state: a backward that kept it raises."""
    from video_diffusion_amd import block_hip as B
    q = torch.randn(1, 3, 2, 32, device=DEV).to(torch.bfloat16).requires_grad_()
    dec, s = torch.full((2,), -0.1, device=DEV), torch.zeros(1, 2, 32, 32, device=DEV)
    o = B.decay_attention(q, q, q, dec, initial_state=s)
    with torch.no_grad():
        B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():
        s = torch.zeros(1, 2, 32, 32, device=DEV)
        B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, s)
        assert s.any()


@gpu
def test_no_second_derivative():
    from video_diffusion_amd import block_hip as B
    q = torch.randn(1, 40, 2, 32, device=DEV).to(torch.bfloat16).requires_grad_()
    o = B.decay_attention(q, q, q, torch.full((2,), -0.1, device=DEV))
    (g,) = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


def _args(**kw):
    a = _lib.DecayArgs()
    a.dtype, a.b, a.inner, a.n, a.heads, a.d, a.scale, a.log_decay = 0, 2, 3, 10, 2, 32, 0.2, 16
    for f in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        setattr(a, f, _lib.Rows4(256, 64 * 30, 64, 64 * 3, 32))
    for k, x in kw.items():
        if "_" in k and k.split("_")[0] in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
            f, sub = k.split("_")
            r = getattr(a, f)
            setattr(r, sub, x)
        else:
            setattr(a, k, x)
    return a


def test_entry_points_refuse_bad_arguments():
    """Checked on the host before anything is launched."""
    lib = _lib.lib()
    E_ARG, E_SHAPE, E_ALIGN = -1, -2, -3
    fwd = lambda **kw: lib.vdmi_decay_attn_fwd(C.byref(_args(**kw)), None)
    bwd = lambda **kw: lib.vdmi_decay_attn_bwd(C.byref(_args(**kw)), None)
    assert lib.vdmi_decay_attn_fwd(None, None) == E_ARG and lib.vdmi_decay_attn_bwd(None, None) == E_ARG
    for f in (fwd, bwd):
        assert f(dtype=2) == E_ARG and f(log_decay=None) == E_ARG and f(q_p=None) == E_ARG
        assert f(scale=0.0) == E_ARG and f(scale=float("inf")) == E_ARG and f(scale=float("nan")) == E_ARG
        assert f(n=0) == E_SHAPE and f(b=0) == E_SHAPE and f(d=48) == E_SHAPE and f(heads=1 << 17) == E_SHAPE
        assert f(b=1 << 30, inner=1 << 4) == E_SHAPE
        assert f(q_p=264) == E_ALIGN and f(k_n=100) == E_ALIGN and f(v_h=33) == E_ALIGN
    assert fwd(o_p=None) == E_ARG and fwd(o_b=4) == E_ALIGN
    assert bwd(dout_p=None) == E_ARG and bwd(dk_p=None) == E_ARG and bwd(dv_p=8) == E_ALIGN
    # few long sequences need a workspace
    assert lib.vdmi_decay_attn_workspace_bytes(C.byref(_args())) == 0
    long = dict(b=1, inner=1, n=8192, d=64)
    need = lib.vdmi_decay_attn_workspace_bytes(C.byref(_args(**long)))
    assert need > 0 and need % (2 * 64 * 64 * 4) == 0
    assert fwd(**long) == E_ARG and fwd(**long, workspace=256, workspace_bytes=need - 1) == E_ARG
    assert bwd(**long, workspace=256, workspace_bytes=need - 1, fwd_workspace=256) == E_ARG
    assert bwd(**long, workspace=256, workspace_bytes=need) == E_ARG            # the forward's states
    full = dict(**long, workspace_bytes=need)
    assert fwd(**full, workspace=264) == E_ALIGN and bwd(**full, workspace=264, fwd_workspace=256) == E_ALIGN
    assert bwd(**full, workspace=256, fwd_workspace=260) == E_ALIGN
    assert bwd(state_in=264) == E_ALIGN
    for f, r in ((fwd, "q_n"), (fwd, "o_n"), (bwd, "v_n"), (bwd, "dk_n")):
        assert f(**{r: (1 << 25) + 8}) == E_SHAPE and f(**{r: -8}) == E_SHAPE
    assert lib.vdmi_decay_attn_workspace_bytes(C.byref(_args(d=48))) == 0
    st = (C.c_int64 * 8)(*[64, 32] * 4)
    step = lambda *a: lib.vdmi_decay_attn_step(*a, None)
    assert step(None, 16, 16, 16, st, 16, 16, 0, 1, 2, 32, 0.2) == E_ARG
    assert step(16, 16, 16, 16, st, 16, None, 0, 1, 2, 32, 0.2) == E_ARG
    assert step(16, 16, 16, 16, st, 16, 16, 2, 1, 2, 32, 0.2) == E_ARG
    assert step(16, 16, 16, 16, st, 16, 16, 0, 1, 2, 32, 0.0) == E_ARG
    assert step(16, 16, 16, 16, st, 16, 16, 0, 0, 2, 32, 0.2) == E_SHAPE
    assert step(16, 16, 16, 16, st, 16, 16, 0, 1, 2, 40, 0.2) == E_SHAPE
    assert step(16, 16, 16, 16, st, 16, 24, 0, 1, 2, 32, 0.2) == E_ALIGN


def test_python_entry_points_refuse():
    """No CPU path, and calls that do not fit together, raise VdmiError."""
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    q = torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(VdmiError, match="no CPU path"):
        B.decay_attention(q, q, q, torch.zeros(2))
    with pytest.raises(VdmiError, match="no CPU path"):
        B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 32, 32))
    with pytest.raises(VdmiError, match="dimensions"):
        B.decay_attention(q[0], q[0], q[0], torch.zeros(2))


@gpu
def test_python_entry_points_refuse_on_the_gpu():
    from video_diffusion_amd import block_hip as B
    from video_diffusion_amd._lib import VdmiError
    q = torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16, device=DEV)
    dec = torch.zeros(2, device=DEV)
    st = torch.zeros(1, 2, 32, 32, device=DEV)
    bad = [
        (lambda: B.decay_attention(q.float(), q.float(), q.float(), dec), "bfloat16 or float16"),
        (lambda: B.decay_attention(q, q.half(), q, dec), "one dtype"),
        (lambda: B.decay_attention(q, q[:, :3], q, dec), "one shape"),
        (lambda: B.decay_attention(q, q, q[:, :, :1], dec), "one shape"),
        (lambda: B.decay_attention(q[..., :16], q[..., :16], q[..., :16], dec), "32, 64 or 128"),
        (lambda: B.decay_attention(q, q, q, dec[:1]), "log_decay"),
        (lambda: B.decay_attention(q, q, q, dec.double()), "log_decay"),
        (lambda: B.decay_attention(q, q, q, dec.clone().requires_grad_()), "constant"),
        (lambda: B.decay_attention(q, q, q, dec, initial_state=st[:, :1]), "state"),
        (lambda: B.decay_attention(q, q, q, dec, initial_state=st.half()), "state"),
        (lambda: B.decay_attention(q, q, q, dec, initial_state=st.cpu()), "no CPU path"),
        (lambda: B.decay_attention(q, q, q, dec, scale=0.0), "scale"),
        (lambda: B.decay_attention(q, q, q, dec, scale=float("nan")), "scale"),
        (lambda: B.decay_attention(q, q, q, dec, lengths=torch.tensor([4], device=DEV)), "lengths"),
        (lambda: B.decay_attention(q, q, q, dec, lengths=torch.tensor([4, 4], device=DEV, dtype=torch.int32)), "lengths"),
        (lambda: B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, st.transpose(-1, -2)), "contiguous"),
        (lambda: B.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, st.clone().requires_grad_()), "no gradients"),
    ]
    for call, what in bad:
        with pytest.raises(VdmiError, match=what):
            call()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n,state", [(20, False), (20, True), (33, False), (300, True), (2500, False)])
def test_results_are_rounded_once(n, state, d, dtype):
    """What is stored is as near to the definition as its rounding allows, at any length: pairs and states enter their
    products as two 16-bit operands (2^-17 of them lost in bfloat16, 2^-22 in half), under a hundredth of the result's own
    rounding in the 2-norm; 1.05 leaves room for the float32 sums."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 1, n, 3, d, dtype, n + d, state=state)
    flat = lambda t: None if t is None else t[0]
    (o, last, *want), _ = reference(flat(q), flat(k), flat(v), decay, flat(st), None, d ** -0.5, flat(do), flat(ds))
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    if state:
        got, gl = B.decay_attention(*ins, decay, initial_state=st, return_state=True)
        grads = torch.autograd.grad((got, gl), ins, (do, ds))
    else:
        got = B.decay_attention(*ins, decay)
        grads = torch.autograd.grad(got, ins, do)
    for name, x, w in zip(("o", "dq", "dk", "dv"), (got.detach(), *grads), (o, *want)):
        once = rel_err(w.to(dtype), w)
        err = record(f"decay.once.n{n}.d{d}.{dtype}.{state}.{name}", rel_err(flat(x), w), 1.05 * once)
        assert err < 1.05 * once, (name, err, once)


@gpu
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("n", [6, 10, 17, 24, 31, 32])
def test_a_neighbour_that_is_not_finite(n, ragged):
    """Sequences of every length that leaves rows of a tile over: an infinity or NaN in the first token of one of them does
    not reach the ones beside it, forward or backward."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, *_ = inputs(2, 9, n, 2, 32, torch.bfloat16, n)
    lengths = torch.full((2, 9), n, device=DEV, dtype=torch.int32) if ragged else None
    clean = [t.clone() for t in (q, k, v, do)]

    def run(q, k, v, do):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        o = B.decay_attention(*ins, decay, lengths=lengths)
        return [o, *torch.autograd.grad(o, ins, do)]

    want = run(*clean)
    others = torch.ones(2, 9, dtype=torch.bool, device=DEV)
    others[0, 3] = others[1, 8] = False
    for which in range(4):
        for value in (float("nan"), float("inf")):
            bad = [t.clone() for t in clean]
            bad[which][0, 3, 0] = value
            bad[which][1, 8, 0, 1, 7] = value
            for got, w in zip(run(*bad), want):
                assert torch.equal(got[others], w[others])


@gpu
@pytest.mark.parametrize("n", [5, 12, 20, 32, 70])
def test_padding_behind_a_token_that_is_not_finite(n):
    """Outputs and gradients behind lengths are zeros whatever the tokens before them hold."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, *_ = inputs(2, 3, n, 2, 32, torch.bfloat16, n)
    lengths = torch.full((2, 3), n - 2, device=DEV, dtype=torch.int32)
    for which in range(4):
        bad = [t.clone() for t in (q, k, v, do)]
        bad[which][:, :, 1] = float("nan")
        ins = [t.detach().requires_grad_() for t in bad[:3]]
        o = B.decay_attention(*ins, decay, lengths=lengths)
        for x in (o.detach(), *torch.autograd.grad(o, ins, bad[3])):
            assert torch.equal(x[:, :, n - 2:], torch.zeros_like(x[:, :, n - 2:]))


@gpu
@pytest.mark.parametrize("qk,up", [(1e-2, 1e-4), (1.0, 1e-5), (1e-3, 1.0), (1e-4, 1e-6)])
@pytest.mark.parametrize("n,d,state", [(9, 64, False), (24, 32, True), (33, 64, False), (300, 128, False), (3000, 64, True)])
def test_small_halfs(n, d, state, qk, up):
    """Halfs whose pairs, states or own values lie below the type's normal range count in full: every result is as near to
    the definition as its rounding to half allows (1.05 of that, as for values near one)."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 1, n, 2, d, torch.float32, n + d, state=state)
    q, k, v, do = (qk * q).half(), (qk * k).half(), v.half(), (up * do).half()
    if state:
        st, ds = qk * st, up * ds
    flat = lambda t: None if t is None else t[0]
    (o, last, dq, dk, dv, ds0), _ = reference(flat(q), flat(k), flat(v), decay, flat(st), None, d ** -0.5, flat(do), flat(ds))
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    if state:
        got, gl = B.decay_attention(*ins, decay, initial_state=st, return_state=True)
        grads = torch.autograd.grad((got, gl), ins, (do, ds))
        assert rel_err(flat(gl), last) < 1e-5
    else:
        got = B.decay_attention(*ins, decay)
        grads = torch.autograd.grad(got, ins, do)
    for name, x, w in zip(("o", "dq", "dk", "dv"), (got.detach(), *grads), (o, dq, dk, dv)):
        once = rel_err(w.half(), w)
        err = record(f"decay.small.n{n}.d{d}.{qk}.{up}.{state}.{name}", rel_err(flat(x), w), 1.05 * once)
        assert err < 1.05 * once, (name, err, once)


@gpu
@pytest.mark.parametrize("n,state", [(9, False), (9, True), (70, False), (3000, True)])
def test_a_decay_that_is_not_a_number(n, state):
    """NaN in log_decay makes everything of its head NaN, and nothing of another head."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 1, n, 3, 32, torch.bfloat16, n, state=state)
    bad = decay.clone()
    bad[1] = float("nan")

    def run(decay):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        if not state:
            o = B.decay_attention(*ins, decay)
            return [o.detach(), *torch.autograd.grad(o, ins, do)], []
        o, s = B.decay_attention(*ins, decay, initial_state=st, return_state=True)
        step = s.detach()[:, 0].clone()
        x = B.decay_attention_step(q[:, 0, 0], k[:, 0, 0], v[:, 0, 0], decay, step)
        return [o.detach(), *torch.autograd.grad((o, s), ins, (do, ds))], [s.detach()[:, 0], step, x]

    (rows, states), (rows0, states0) = run(bad), run(decay)
    for x, w in zip(rows, rows0):
        assert torch.isnan(x[..., 1, :]).all()
        assert torch.equal(x[..., 0::2, :], w[..., 0::2, :])
    for x, w in zip(states, states0):
        assert torch.isnan(x[:, 1]).all() and torch.equal(x[:, 0::2], w[:, 0::2])


@gpu
@pytest.mark.parametrize("wanted,n,state", [(w, n, n > 9) for n in (9, 45, 3000) for w in ("q", "k", "v", "s", "qs", "kv", "qk")
                                            if n > 9 or "s" not in w])
def test_only_the_gradients_that_are_asked_for(wanted, n, state, monkeypatch):
    """They are those of a call that asks for all, and nothing else is computed."""
    from video_diffusion_amd import block_hip as B
    q, k, v, do, decay, st, ds, _ = inputs(1, 2, n, 2, 64, torch.bfloat16, n, state=state)
    asked = []
    real = _lib.lib().vdmi_decay_attn_bwd
    monkeypatch.setattr(_lib.lib(), "vdmi_decay_attn_bwd",
                        lambda a, s: asked.append((bool(a.dq.p), bool(a.dk.p), bool(a.dv.p), bool(a.dstate_out))) or real(a, s))

    def run(names):
        t = {"q": q, "k": k, "v": v, "s": st}
        t = {i: x if x is None else x.detach().requires_grad_(i in names) for i, x in t.items()}
        o, s = B.decay_attention(t["q"], t["k"], t["v"], decay, initial_state=t["s"], return_state=True)
        return dict(zip(names, torch.autograd.grad((o, s), [t[i] for i in names], (do, torch.zeros_like(s) if ds is None else ds))))

    full, got = run("qkvs" if state else "qkv"), run(wanted)
    for i in wanted:
        assert torch.equal(got[i], full[i])
    both = wanted != "q"                     # one walk computes dk, dv and the state's gradient
    assert asked[1] == ("q" in wanted, both, both, "s" in wanted)


def test_gradients_that_nobody_wants():
    """The library takes a null dq, or null dk and dv without the state's gradient; not one of dk and dv alone, nor none."""
    lib = _lib.lib()
    bwd = lambda **kw: lib.vdmi_decay_attn_bwd(C.byref(_args(**kw)), None)
    none = dict(dk_p=None, dv_p=None)
    assert bwd(dv_p=None) == -1 and bwd(dq_p=None, **none) == -1 and bwd(dstate_out=256, **none) == -1
    # the rest is still checked, up to here without a launch
    assert bwd(dq_p=None, dk_b=4) == -3 and bwd(dq_p=8, **none) == -3 and bwd(dq_p=None, v_p=None) == -1


def test_results_of_a_broadcast_operand_stay_within_the_kernels_pitch():
    """A result lies in memory in its operand's order, but never with tokens further apart than the kernels take: sites that
    share one row do not become the fastest dimension of 2^26 elements."""
    from video_diffusion_amd import block_hip as B
    for shape, strides in (((2, 1 << 19, 4, 2, 64), (1024, 0, 128, 64, 1)), ((2, 1 << 19, 4, 2, 64), (0, 0, 0, 0, 1)),
                           ((1, 1 << 19, 4, 2, 64), (0, 64, 1 << 25, 1 << 27, 1))):
        q = torch.empty(0, device="meta", dtype=torch.bfloat16).new_empty_strided(shape, strides)
        t = B._empty_like_rows(q)
        assert t.shape == q.shape and t.stride(2) <= _lib.DECAY_MAX_PITCH and t.stride(4) == 1
        assert t.untyped_storage().nbytes() == 2 * q.numel()


def test_scales_without_a_reciprocal_are_refused():
    """The backward divides by the scale: one whose reciprocal is not a finite float32 is refused on the host."""
    lib = _lib.lib()
    for s in (1e-39, -1e-39, 1e-45, 3e38, -3e38):
        assert lib.vdmi_decay_attn_fwd(C.byref(_args(scale=s)), None) == -1
        assert lib.vdmi_decay_attn_bwd(C.byref(_args(scale=s)), None) == -1
    from video_diffusion_amd import block_hip as B
    for s in (1e-39, -1e-39, 1e-46, 3e38, float("inf"), float("nan"), 0.0):
        with pytest.raises(_lib.VdmiError, match="scale"):
            B._scale(s, 32)
    assert B._scale(2.0 ** -126, 32) == 2.0 ** -126 and B._scale(-(2.0 ** 126), 32) == -(2.0 ** 126)


def test_calls_beyond_one_launch_are_refused():
    """2^32 threads, of operands that all sequences may share: refused on the host, before anything is launched."""
    lib = _lib.lib()
    rows = lambda: _lib.Rows4(256, 0, 0, 32, 32)
    for n in (32, 40):
        a = _args(b=1 << 15, inner=1 << 15, n=n, heads=1, d=128, q=rows(), k=rows(), v=rows(), o=rows(), dout=rows(), dq=rows(), dk=rows(),
                  dv=rows())
        assert lib.vdmi_decay_attn_fwd(C.byref(a), None) == -2 and lib.vdmi_decay_attn_bwd(C.byref(a), None) == -2
    st = (C.c_int64 * 8)(*[0, 0] * 4)
    assert lib.vdmi_decay_attn_step(16, 16, 16, 16, st, 16, 16, 0, 1 << 26, 1, 32, 0.2, None) == -2
