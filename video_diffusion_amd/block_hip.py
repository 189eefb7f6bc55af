"""Operators of a causal layer over time, in training and one frame at a time, on the HIP kernels:

  decay_attention, decay_attention_step   linear attention with a decay per head over whole sequences / one more token
                                          (csrc/decay.hip)
  norm_before, norm_after, norm_between   the norms before and after a block with its gate, scale, shift and residual scale
                                          (csrc/blocknorm.hip)
  pack_rows8, rows8_wgrad, linear_rows8   activations kept for the backward pass in 8 bits, and a Linear whose weight
                                          gradient reads them (csrc/rows8.hip)

They stand beside the layers of train_hip.py: its attention is a softmax over all frames at once and keeps no state, its
LayerNorm has no scale, shift or gate, its saved rows are bfloat16 (train_hip.rows8_checkpoints() keeps its ResnetBlocks'
in 8 bits).  Element types go by the tensors (bfloat16, float16, float32 for the norms and the kept rows; states and
parameters float32) whatever VDMI_PRECISION says.  Calls run on the current stream of the tensors' device.  There is no
fallback: tensors that are not on a GPU and shapes that the kernels do not take raise VdmiError.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import VdmiError, check
from .train_hip import _plain

_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}


def _stream_of(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _require(ok, what: str):
    if not ok:
        raise VdmiError(what)


def _on_gpu(*ts):
    first = next(t for t in ts if t is not None)
    for t in ts:
        if t is None:
            continue
        _require(t.is_cuda, "the block operators need CUDA (HIP) tensors; there is no CPU path")
        _require(t.device == first.device, f"tensors on different devices: {t.device} and {first.device}")


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------------------
# attention over time with a decay per head
# ---------------------------------------------------------------------------------------------------------------------
def _rows4(t: torch.Tensor) -> "_lib.Rows4":
    """t: [b, inner, n, heads, d]"""
    return _lib.Rows4(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), t.stride(3))


def _row_operand(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it - 16-byte pieces of d contiguous features at any non-negative strides - or a copy that is."""
    pieces = all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
    if t.stride(-1) == 1 and pieces and t.data_ptr() % 16 == 0:
        if all(n > 1 or s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
            return t
        # a dimension of one element may have any stride; the library is told 0
        return t.as_strided(t.shape, [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1])] + [1])
    return t.contiguous()


def _empty_like_rows(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised dense tensor of t's shape whose dimensions lie in memory in t's order: the sites of a frame stay
    next to each other where t is a permuted view of (batch, frame, site) rows.  Broadcast dimensions of t become real."""
    order = sorted(range(t.dim() - 1), key=lambda i: (-t.stride(i), i)) + [t.dim() - 1]
    out = torch.empty([t.shape[i] for i in order], device=t.device, dtype=t.dtype)
    return out.permute([order.index(i) for i in range(t.dim())])


def _decay_args(q, k, v, log_decay, lengths, state, scale) -> "_lib.DecayArgs":
    a = _lib.DecayArgs()
    a.dtype = _DTYPES[q.dtype]
    a.b, a.inner, a.n, a.heads, a.d = q.shape
    a.scale = scale
    a.q, a.k, a.v = _rows4(q), _rows4(k), _rows4(v)
    a.log_decay, a.lengths, a.state_in = log_decay.data_ptr(), _ptr(lengths), _ptr(state)
    return a


def _run_decay(fn: str, a, device, stream):
    lib = _lib.lib()
    a.workspace_bytes = lib.vdmi_decay_attn_workspace_bytes(C.byref(a))
    ws = torch.empty(a.workspace_bytes, device=device, dtype=torch.uint8) if a.workspace_bytes else None
    a.workspace = _ptr(ws)
    check(getattr(lib, fn)(C.byref(a), stream), fn)


class DecayAttnFn(torch.autograd.Function):
    """o (and the state after the last token) of q, k, v [b, inner, n, heads, d] and a first state; constants log_decay,
    lengths, scale."""

    @staticmethod
    @_plain
    def forward(ctx, q, k, v, state, log_decay, lengths, scale, return_state):
        q, k, v = _row_operand(q), _row_operand(k), _row_operand(v)
        with torch.cuda.device(q.device):
            o = _empty_like_rows(q)
            b, inner, n, h, d = q.shape
            last = torch.empty(b, inner, h, d, d, device=q.device, dtype=torch.float32) if return_state else None
            a = _decay_args(q, k, v, log_decay, lengths, state, scale)
            a.o, a.state_out = _rows4(o), _ptr(last)
            _run_decay("vdmi_decay_attn_fwd", a, q.device, _stream_of(q))
        ctx.save_for_backward(q, k, v, state, log_decay, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @_plain
    def backward(ctx, do, dlast):
        q, k, v, state, log_decay, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        if do is None and dlast is None:
            return (None,) * 8
        with torch.cuda.device(q.device):
            do = torch.zeros_like(q) if do is None else do
            do = _row_operand(do.to(q.dtype))
            dlast = None if dlast is None else dlast.to(torch.float32).contiguous()
            dq, dk, dv = _empty_like_rows(q), _empty_like_rows(k), _empty_like_rows(v)
            dstate = torch.empty_like(state) if need[3] and state is not None else None
            a = _decay_args(q, k, v, log_decay, lengths, state, ctx.scale)
            a.dout, a.dq, a.dk, a.dv = _rows4(do), _rows4(dq), _rows4(dk), _rows4(dv)
            a.dstate_in, a.dstate_out = _ptr(dlast), _ptr(dstate)
            _run_decay("vdmi_decay_attn_bwd", a, q.device, _stream_of(q))
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dstate, None, None, None, None)


def _check_decay(q, k, v, log_decay, state, lead, heads, d):
    _on_gpu(q, k, v, log_decay, state)
    _require(q.dtype in (torch.bfloat16, torch.float16), f"q, k, v are bfloat16 or float16 (got {q.dtype})")
    _require(k.dtype == q.dtype and v.dtype == q.dtype, f"q, k, v have one dtype (got {q.dtype}, {k.dtype}, {v.dtype})")
    _require(k.shape == q.shape and v.shape == q.shape,
             f"q, k, v have one shape (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    _require(d in (32, 64, 128), f"heads of 32, 64 or 128 features (got {d})")
    _require(log_decay.dtype == torch.float32 and log_decay.shape == (heads,),
             f"log_decay is float32 [{heads}] (got {log_decay.dtype} {tuple(log_decay.shape)})")
    _require(not log_decay.requires_grad, "log_decay is a constant of the layer: no gradient is computed for it")
    if state is not None:
        _require(state.dtype == torch.float32 and tuple(state.shape) == (*lead, heads, d, d),
                 f"the state is float32 {(*lead, heads, d, d)} (got {state.dtype} {tuple(state.shape)})")


def _scale(scale, d):
    scale = d ** -0.5 if scale is None else float(scale)
    _require(scale != 0 and abs(scale) < 3e38, f"scale is finite and not zero (got {scale})")
    return scale


def decay_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """Linear attention over time whose memory of a token fades by exp(log_decay[head]) per step:
    S_t = exp(log_decay) S_(t-1) + k_t v_t^T, o_t = scale * q_t S_t.  Differentiable in q, k, v and initial_state.

    q, k, v: bfloat16 or float16 [b, n, heads, d] or, for the sequences of many sites, [b, sites, n, heads, d]; any strides
    (views of qkv rows are read in place where their rows are 16-byte aligned).  d is 32, 64 or 128.  log_decay: float32
    [heads], at most 0, a constant.  scale: d^-0.5 by default.  initial_state: float32 [b(, sites), heads, d, d], S before
    the first token (zeros by default).  lengths: int32 [b(, sites)] - tokens from there on are padding: they are not read,
    their outputs and gradients are zeros.  return_state: also return S after the last token, for decay_attention_step or
    the next piece of the sequence.  Returns o like q (in q's order of dimensions in memory), or (o, state)."""
    _require(q.dim() in (4, 5), f"q is [b, n, heads, d] or [b, sites, n, heads, d] (got {q.dim()} dimensions)")
    lead, (n, heads, d) = tuple(q.shape[:-3]), q.shape[-3:]
    _check_decay(q, k, v, log_decay, initial_state, lead, heads, d)
    scale = _scale(scale, d)
    if lengths is not None:
        _on_gpu(q, lengths)
        _require(lengths.dtype == torch.int32 and tuple(lengths.shape) == lead,
                 f"lengths is int32 {lead} (got {lengths.dtype} {tuple(lengths.shape)})")
        lengths = lengths.contiguous()
    if q.numel() == 0:
        # no sequences, or sequences of no tokens: the state stays
        o = q * k * v
        if not return_state:
            return o
        return o, (torch.zeros(*lead, heads, d, d, device=q.device) if initial_state is None else initial_state.clone())
    four = q.dim() == 4
    if four:
        q, k, v = q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1)
    b, inner = q.shape[:2]
    state = None if initial_state is None else initial_state.reshape(b, inner, heads, d, d).contiguous()
    if state is not None and state.data_ptr() % 16:
        state = state.clone()
    o, last = DecayAttnFn.apply(q, k, v, state, log_decay.contiguous(), lengths, scale, bool(return_state))
    o = o.squeeze(1) if four else o
    return (o, last.view(*lead, heads, d, d)) if return_state else o


def decay_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One more token of every sequence: state (float32 [..., heads, d, d], contiguous) is updated in place to
    exp(log_decay) state + k v^T, and scale * q state is returned.  q, k, v: bfloat16 or float16 [..., heads, d].  For
    sampling: no gradients."""
    _require(q.dim() >= 2, f"q is [..., heads, d] (got {q.dim()} dimensions)")
    lead, (heads, d) = tuple(q.shape[:-2]), q.shape[-2:]
    _check_decay(q, k, v, log_decay, state, lead, heads, d)
    scale = _scale(scale, d)
    _require(state.is_contiguous() and state.data_ptr() % 16 == 0, "the state is contiguous and 16-byte aligned")
    _require(not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state))),
             "decay_attention_step computes no gradients: call it under torch.no_grad(), or decay_attention")
    o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if q.numel() == 0:
        return o

    def flat(t):
        t = t.reshape(-1, heads, d)
        return t if t.stride(-1) == 1 else t.contiguous()

    ops = [flat(q), flat(k), flat(v), o.view(-1, heads, d)]
    strides = (C.c_int64 * 8)(*[s for t in ops for s in t.stride()[:2]])
    with torch.cuda.device(q.device):
        check(_lib.lib().vdmi_decay_attn_step(*[t.data_ptr() for t in ops], strides, log_decay.contiguous().data_ptr(),
                                              state.data_ptr(), _DTYPES[q.dtype], ops[0].shape[0], heads, d, scale,
                                              _stream_of(q)), "vdmi_decay_attn_step")
    return o


# ---------------------------------------------------------------------------------------------------------------------
# the norms before and after a block
# ---------------------------------------------------------------------------------------------------------------------
def _rows2(t: torch.Tensor) -> torch.Tensor:
    """t [..., c] as [rows][c] with contiguous columns: a view where the rows have one pitch, else a copy."""
    r = t.reshape(-1, t.shape[-1])
    return r if r.stride(1) == 1 and (r.shape[0] == 1 or r.stride(0) >= r.shape[1]) else r.contiguous()


def _pitch(r: torch.Tensor) -> int:
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


class BlockNormFn(torch.autograd.Function):
    """(out, y) of rows x, h and parameters; out None without h, y None unless want_y."""

    @staticmethod
    @_plain
    def forward(ctx, x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y):
        params = [None if p is None else p.detach().contiguous() for p in (post_weight, gate, weight, scale, shift)]
        xr, hr = _rows2(x), None if h is None else _rows2(h)
        with torch.cuda.device(x.device):
            out = None if h is None else torch.empty(x.shape, device=x.device, dtype=x.dtype)
            y = torch.empty(x.shape, device=x.device, dtype=x.dtype) if want_y else None
            a = _norm_args(xr, hr, params, x.shape[0], alpha, kind, post_kind, eps)
            a.out, a.y, a.ldo, a.ldy = _ptr(out), _ptr(y), x.shape[-1], x.shape[-1]
            check(_lib.lib().vdmi_block_norm_fwd(C.byref(a), _stream_of(x)), "vdmi_block_norm_fwd")
        ctx.save_for_backward(xr, hr, *params)
        ctx.meta = (tuple(x.shape), alpha, kind, post_kind, eps)
        ctx.set_materialize_grads(False)
        return out, y

    @staticmethod
    @_plain
    def backward(ctx, dout, dy):
        xr, hr, *params = ctx.saved_tensors
        shape, alpha, kind, post_kind, eps = ctx.meta
        need = ctx.needs_input_grad
        if dout is None and dy is None:
            return (None,) * 12
        with torch.cuda.device(xr.device):
            dout, dy = (None if g is None else _rows2(g.to(xr.dtype)) for g in (dout, dy))
            dx = torch.empty(shape, device=xr.device, dtype=xr.dtype) if need[0] else None
            dh = torch.empty(shape, device=xr.device, dtype=xr.dtype) if need[1] else None
            grads = [torch.empty_like(p) if n and p is not None else None for n, p in zip(need[2:7], params)]
            if dy is None:              # nothing is learnt about the second norm's parameters
                grads[2:] = [None if g is None else g.zero_() for g in grads[2:]]
            a = _norm_args(xr, hr, params, shape[0], alpha, kind, post_kind, eps)
            a.dout, a.dy, a.dx, a.dh = _ptr(dout), _ptr(dy), _ptr(dx), _ptr(dh)
            a.lddo, a.lddy = (shape[-1] if g is None else _pitch(g) for g in (dout, dy))
            a.lddx = a.lddh = shape[-1]
            a.dpost_weight, a.dgate = _ptr(grads[0]), _ptr(grads[1])
            if dy is not None:
                a.dweight, a.dscale, a.dshift = (_ptr(g) for g in grads[2:])
            lib = _lib.lib()
            a.workspace_bytes = lib.vdmi_block_norm_bwd_workspace_bytes(C.byref(a))
            ws = torch.empty(a.workspace_bytes, device=xr.device, dtype=torch.uint8) if a.workspace_bytes else None
            a.workspace = _ptr(ws)
            check(lib.vdmi_block_norm_bwd(C.byref(a), _stream_of(xr)), "vdmi_block_norm_bwd")
        return (dx, dh, *grads, None, None, None, None, None)


def _norm_args(xr, hr, params, samples, alpha, kind, post_kind, eps) -> "_lib.BlockNormArgs":
    a = _lib.BlockNormArgs()
    a.dtype, a.c, a.kind, a.post_kind = _DTYPES[xr.dtype], xr.shape[1], _lib.NORM_KINDS[kind], _lib.NORM_KINDS[post_kind]
    a.rows, a.rows_per_sample = xr.shape[0], xr.shape[0] // samples
    a.eps, a.alpha = eps, alpha
    a.x, a.ldx = xr.data_ptr(), _pitch(xr)
    if hr is not None:
        a.h, a.ldh = hr.data_ptr(), _pitch(hr)
    a.post_weight, a.gate, a.weight, a.scale, a.shift = (_ptr(p) for p in params)
    a.gate_stride, a.scale_stride, a.shift_stride = (
        a.c if p is not None and p.dim() == 2 and p.shape[0] > 1 else 0 for p in (params[1], params[3], params[4]))
    return a


def _block_norm(x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y):
    _on_gpu(x, h, post_weight, gate, weight, scale, shift)
    _require(x.dtype in _DTYPES, f"rows are bfloat16, float16 or float32 (got {x.dtype})")
    _require(x.dim() >= 2 and 1 <= x.shape[-1] <= 8192, f"rows are [samples, ..., c] with c from 1 to 8192 (got {tuple(x.shape)})")
    _require(h is None or (h.dtype == x.dtype and h.shape == x.shape),
             None if h is None else f"x and h are alike (got {x.dtype} {tuple(x.shape)}, {h.dtype} {tuple(h.shape)})")
    b, c = x.shape[0], x.shape[-1]
    for name, p in (("post_weight", post_weight), ("weight", weight)):
        _require(p is None or (p.dtype == torch.float32 and tuple(p.shape) == (c,)), f"{name} is float32 [{c}]")
    for name, p in (("gate", gate), ("scale", scale), ("shift", shift)):
        _require(p is None or (p.dtype == torch.float32 and tuple(p.shape) in ((c,), (1, c), (b, c))),
                 f"{name} is float32 [{c}], [1, {c}] or [{b}, {c}]")
    _require(kind in ("rms", "layer"), f"kind is 'rms' or 'layer' (got {kind!r})")
    _require(post_kind in ("rms", "layer", None), f"the kind of the norm after the block is 'rms', 'layer' or None (got {post_kind!r})")
    eps, alpha = float(eps), float(alpha)
    _require(0 <= eps < 1e30 and abs(alpha) < 3e38, f"eps is not negative and alpha finite (got {eps}, {alpha})")
    if x.numel() == 0:
        return (None if h is None else x + h), (x * 1 if want_y else None)
    return BlockNormFn.apply(x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y)


def norm_before(x, weight=None, scale=None, shift=None, *, kind="rms", eps=1e-5):
    """N(x) * weight * (1 + scale) + shift, the norm before a block.  x: bfloat16, float16 or float32 [samples, ..., c]; N
    over the last dimension, x / sqrt(mean x^2 + eps) (kind "rms") or (x - mean) / sqrt(var + eps) ("layer").  weight:
    float32 [c]; scale, shift: float32 [c] or one row per sample, [samples, c]; each may be absent.  Differentiable in all."""
    return _block_norm(x, None, None, None, weight, scale, shift, 1.0, kind, None, eps, True)[1]


def norm_after(x, h, weight=None, gate=None, *, alpha=1.0, kind="rms", eps=1e-5):
    """alpha x + gate * P(h) * weight: a block's output h behind its norm (kind "rms" or "layer"; None: h as it is) and
    gate (float32 [c] or [samples, c]) added to the residual x.  Differentiable in x, h and the parameters."""
    return _block_norm(x, h, weight, gate, None, None, None, alpha, "rms", kind, eps, False)[0]


def norm_between(x, h, post_weight=None, gate=None, weight=None, scale=None, shift=None, *, alpha=1.0, kind="rms",
                 post_kind="rms", eps=1e-5):
    """From one block to the next in one pass: out = norm_after(x, h, post_weight, gate) and y = norm_before of it with
    weight, scale, shift (of the sum before it is rounded to x's dtype).  Returns (out, y)."""
    return _block_norm(x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, True)


# ---------------------------------------------------------------------------------------------------------------------
# activations kept in 8 bits
# ---------------------------------------------------------------------------------------------------------------------
class Rows8:
    """Rows kept in 8 bits: codes uint8 [rows][c] (e4m3) times a power of two per 32 channels, exps uint8 [rows][ceil(c/32)].
    shape and dtype are those of the tensor that was packed."""

    __slots__ = ("codes", "exps", "shape", "dtype")

    def __init__(self, codes, exps, shape, dtype):
        self.codes, self.exps, self.shape, self.dtype = codes, exps, shape, dtype

    def unpack(self, dtype=None) -> torch.Tensor:
        """The values the codes stand for, in the packed tensor's shape."""
        dtype = self.dtype if dtype is None else dtype
        _require(dtype in _DTYPES, f"rows are bfloat16, float16 or float32 (got {dtype})")
        out = torch.empty(self.shape, device=self.codes.device, dtype=dtype)
        if out.numel():
            rows, c = self.codes.shape
            with torch.cuda.device(out.device):
                check(_lib.lib().vdmi_rows8_unpack(self.codes.data_ptr(), self.exps.data_ptr(), out.data_ptr(), c, _DTYPES[dtype],
                                                   rows, c, _stream_of(out)), "vdmi_rows8_unpack")
        return out


def pack_rows8(x: torch.Tensor) -> Rows8:
    """x [..., c] (bfloat16, float16 or float32, c a multiple of 8) in 8 bits: e4m3 codes times the least power of two per
    row and 32 channels that holds the largest magnitude.  Off by 2^-4 of a value at most (2^-18 of its group's largest for
    the smallest ones); infinities and NaN come back as NaN, magnitudes beyond 448 * 2^119 as that."""
    _on_gpu(x)
    _require(x.dtype in _DTYPES, f"rows are bfloat16, float16 or float32 (got {x.dtype})")
    _require(x.dim() >= 1 and x.shape[-1] > 0 and x.shape[-1] % 8 == 0, f"rows of a multiple of 8 channels (got {tuple(x.shape)})")
    with torch.no_grad(), torch.cuda.device(x.device):
        r = _rows2(x.detach())
        if r.data_ptr() % 16 or _pitch(r) % 8:
            r = r.contiguous().clone() if r.is_contiguous() else r.contiguous()
        rows, c = r.shape
        codes = torch.empty(rows, c, device=x.device, dtype=torch.uint8)
        exps = torch.empty(rows, (c + 31) // 32, device=x.device, dtype=torch.uint8)
        if rows:
            check(_lib.lib().vdmi_rows8_pack(r.data_ptr(), _pitch(r), codes.data_ptr(), exps.data_ptr(), _DTYPES[x.dtype], rows, c,
                                             _stream_of(x)), "vdmi_rows8_pack")
    return Rows8(codes, exps, tuple(x.shape), x.dtype)


def rows8_wgrad(kept: Rows8, dy: torch.Tensor, bias: bool = False):
    """float32 [cout][cin] weight gradient of a Linear from its input kept in 8 bits and the gradient dy [..., cout] of its
    output (bfloat16 rows); with bias also the bias gradient: (dw, db)."""
    _on_gpu(kept.codes, dy)
    rows, cin = kept.codes.shape
    cout = dy.shape[-1]
    _require(dy.dtype == torch.bfloat16, f"dy is bfloat16 (got {dy.dtype})")
    _require(cout > 0 and cout % 8 == 0, f"a multiple of 8 output channels (got {cout})")
    _require(dy.numel() == rows * cout, f"dy has a row for each of the {rows} kept rows (got {tuple(dy.shape)})")
    with torch.no_grad(), torch.cuda.device(dy.device):
        d = _rows2(dy.detach())
        if d.data_ptr() % 16 or _pitch(d) % 8:
            d = d.contiguous().clone() if d.is_contiguous() else d.contiguous()
        if rows == 0:
            dw, db = torch.zeros(cout, cin, device=dy.device), torch.zeros(cout, device=dy.device)
            return (dw, db) if bias else dw
        lib = _lib.lib()
        dw = torch.empty(cout, cin, device=dy.device, dtype=torch.float32)
        db = torch.empty(cout, device=dy.device, dtype=torch.float32) if bias else None
        ws = torch.empty(lib.vdmi_rows8_wgrad_workspace_bytes(cin, cout, rows), device=dy.device, dtype=torch.uint8)
        check(lib.vdmi_rows8_wgrad(kept.codes.data_ptr(), kept.exps.data_ptr(), d.data_ptr(), _pitch(d), dw.data_ptr(), _ptr(db),
                                   cin, cout, rows, ws.data_ptr(), _stream_of(dy)), "vdmi_rows8_wgrad")
    return (dw, db) if bias else dw


class LinearRows8Fn(torch.autograd.Function):
    """y = x weight^T + bias on the row GEMMs of train_hip.py; what is kept of x for the weight gradient is 8 bits wide."""

    @staticmethod
    @_plain
    def forward(ctx, x, weight, bias):
        from .train_hip import _linear_pack, conv_rows
        with torch.cuda.device(x.device):
            xr = x.reshape(-1, x.shape[-1]).contiguous()
            y = conv_rows(xr, _linear_pack(weight.detach(), False), None if bias is None else bias.detach().float().contiguous(),
                          1, 1, 1, xr.shape[0])
            kept = pack_rows8(xr) if ctx.needs_input_grad[1] else None
        ctx.save_for_backward(weight, *((kept.codes, kept.exps) if kept else ()))
        ctx.shape = tuple(x.shape)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @_plain
    def backward(ctx, dy):
        from .train_hip import _linear_pack, conv_rows
        weight, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        with torch.cuda.device(dy.device):
            d = dy.to(torch.bfloat16).reshape(-1, dy.shape[-1]).contiguous()
            if need[0]:
                dx = conv_rows(d, _linear_pack(weight.detach(), True), None, 1, 1, 1, d.shape[0]).view(ctx.shape)
            if need[1]:
                dw = rows8_wgrad(Rows8(*kept, ctx.shape, torch.bfloat16), d, bias=need[2])
                dw, db = dw if need[2] else (dw, None)
            elif need[2]:
                db = d.float().sum(0)
        return dx, dw, db


def linear_rows8(x: torch.Tensor, weight: torch.Tensor, bias=None) -> torch.Tensor:
    """F.linear(x, weight, bias) on the library's row GEMMs for bfloat16 x [..., cin] and float32 weight [cout, cin]
    (multiples of 32), whose input is kept for the weight gradient in 8 bits (about half of a bfloat16 copy).  Output and input gradient are exactly
    those of the bfloat16 path; only the weight gradient sees the rounding to 8 bits.  Needs the bfloat16 build."""
    _on_gpu(x, weight, bias)
    _require(_lib.PRECISION == "bf16", "the training layers exchange bfloat16 rows: VDMI_PRECISION=f16 serves sampling only")
    _require(x.dtype == torch.bfloat16 and weight.dtype == torch.float32 and weight.dim() == 2,
             f"x is bfloat16 and weight float32 [cout, cin] (got {x.dtype}, {weight.dtype} {tuple(weight.shape)})")
    _require(x.shape[-1] == weight.shape[1] and (bias is None or tuple(bias.shape) == (weight.shape[0],)),
             f"x [..., cin], weight [cout, cin], bias [cout] (got {tuple(x.shape)}, {tuple(weight.shape)})")
    _require(weight.shape[0] % 32 == 0 and weight.shape[1] % 32 == 0, f"multiples of 32 channels (got {tuple(weight.shape)})")
    if x.numel() == 0:
        return torch.nn.functional.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))
    return LinearRows8Fn.apply(x, weight, bias)
