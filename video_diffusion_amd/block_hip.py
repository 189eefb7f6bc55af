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
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import VdmiError, check
from .train_hip import _plain

_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
_FLOAT16S = (torch.bfloat16, torch.float16)
_I64x8 = C.c_int64 * 8

_current_device, _raw_stream = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream
_increment_version = torch.autograd.graph.increment_version


def _stream_of(t: torch.Tensor) -> int:
    """The handle of the current stream of t's device, which has to be the current one (_there)."""
    return _raw_stream(t.device.index)


def _there(fn):
    """fn(t, ...) with t's device as the current one."""
    @functools.wraps(fn)
    def inner(t, *args):
        if t.device.index == _current_device():
            return fn(t, *args)
        with torch.cuda.device(t.device):
            return fn(t, *args)
    return inner


def _first_order(backward):
    """backward(ctx, *grads) whose own derivative raises; what that takes is only set up where a graph of it is asked for."""
    once = once_differentiable(backward)

    @functools.wraps(backward)
    def inner(ctx, *grads):
        return (once if torch.is_grad_enabled() else backward)(ctx, *grads)
    return inner


def _on_gpu(first, *ts):
    dev = first.device
    if dev.type != "cuda":
        raise VdmiError("the block operators need CUDA (HIP) tensors; there is no CPU path")
    for t in ts:
        if t is not None and t.device != dev:
            raise VdmiError("the block operators need CUDA (HIP) tensors; there is no CPU path" if not t.is_cuda else
                            f"tensors on different devices: {t.device} and {dev}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _linked(empty: torch.Tensor, *params) -> torch.Tensor:
    """A result of no elements as one of the parameters too: their gradients are zeros, not absent."""
    for p in params:
        if p is not None and _wants_grad(p):
            empty = empty + p.sum().to(empty.dtype)
    return empty


# ---------------------------------------------------------------------------------------------------------------------
# attention over time with a decay per head
# ---------------------------------------------------------------------------------------------------------------------
def _row_operand(t: torch.Tensor) -> torch.Tensor:
    """t [b, inner, n, heads, d] as the kernels read it - 16-byte pieces of d contiguous features at any non-negative
    strides - or a copy that is."""
    s = t.stride()
    if s[4] == 1 and not ((s[0] | s[1] | s[2] | s[3]) & 7) and s[2] <= _lib.DECAY_MAX_PITCH and not t.data_ptr() & 15:
        return t
    # a dimension of one element may have any stride: the library is told 0
    fixed = [x if n > 1 else 0 for x, n in zip(s[:4], t.shape[:4])]
    if s[4] == 1 and not any(x & 7 for x in fixed) and fixed[2] <= _lib.DECAY_MAX_PITCH and not t.data_ptr() & 15:
        return t.as_strided(t.shape, fixed + [1])
    return t.clone(memory_format=torch.contiguous_format)


def _empty_like_rows(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised dense tensor of t's shape whose dimensions lie in memory in t's order: the sites of a frame stay
    next to each other where t is a permuted view of (batch, frame, site) rows.  Broadcast dimensions of t become real; where
    that would part the tokens further than the kernels go, they lie next to each other instead."""
    (b, i, n, h, d), (sb, si, sn, sh, _) = t.shape, t.stride()
    if sb >= si >= sn >= sh:
        return torch.empty((b, i, n, h, d), device=t.device, dtype=t.dtype)
    if sb >= sn >= si >= sh:                    # (batch, frame, site) rows
        strides = [n * i * h * d, h * d, i * h * d, d, 1]
    else:
        strides, pitch = [0, 0, 0, 0, 1], d
        for k in sorted(range(4), key=lambda k: (t.stride(k), -k)):
            strides[k] = pitch
            pitch *= t.shape[k]
    if strides[2] > _lib.DECAY_MAX_PITCH:
        return torch.empty((b, i, n, h, d), device=t.device, dtype=t.dtype)
    return t.new_empty_strided((b, i, n, h, d), strides)


_NO_ROWS = _lib.Rows4()


def _rows4(t) -> "_lib.Rows4":
    if t is None:
        return _NO_ROWS
    s = t.stride()
    return _lib.Rows4(t.data_ptr(), s[0], s[1], s[2], s[3])


def _decay_workspace(a, like):
    size = _lib.lib().vdmi_decay_attn_workspace_bytes(a)
    if not size:
        return None
    ws = torch.empty(size, device=like.device, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    return ws


@_there
def _decay_forward(q, k, v, state, log_decay, lengths, scale, return_state):
    """(o, last state or None, the workspace) of operands as the kernels read them."""
    b, inner, n, h, d = q.shape
    o = _empty_like_rows(q)
    last = torch.empty((b, inner, h, d, d), device=q.device, dtype=torch.float32) if return_state else None
    a = _lib.DecayArgs(_DTYPES[q.dtype], b, inner, n, h, d, scale, 0, _rows4(q), _rows4(k), _rows4(v), _rows4(o),
                       _NO_ROWS, _NO_ROWS, _NO_ROWS, _NO_ROWS, log_decay.data_ptr(), _ptr(lengths), _ptr(state), _ptr(last))
    ws = _decay_workspace(a, q)
    check(_lib.lib().vdmi_decay_attn_fwd(a, _stream_of(q)), "vdmi_decay_attn_fwd")
    return o, last, ws


@_there
def _decay_backward(q, k, v, state, log_decay, lengths, fwd_ws, scale, do, dlast, need):
    """The gradients that need (of q, k, v, the state) asks for; dk and dv come together."""
    do = torch.zeros_like(q) if do is None else _row_operand(do if do.dtype == q.dtype else do.to(q.dtype))
    if dlast is not None:
        dlast = dlast.to(torch.float32).contiguous()
    dq = _empty_like_rows(q) if need[0] else None
    dk, dv = (_empty_like_rows(k), _empty_like_rows(v)) if any(need[1:4]) else (None, None)
    dstate = torch.empty_like(state) if need[3] else None
    b, inner, n, h, d = q.shape
    a = _lib.DecayArgs(_DTYPES[q.dtype], b, inner, n, h, d, scale, 0, _rows4(q), _rows4(k), _rows4(v), _NO_ROWS,
                       _rows4(do), _rows4(dq), _rows4(dk), _rows4(dv), log_decay.data_ptr(), _ptr(lengths), _ptr(state), None,
                       _ptr(dlast), _ptr(dstate), None, 0, _ptr(fwd_ws))
    ws = _decay_workspace(a, q)
    check(_lib.lib().vdmi_decay_attn_bwd(a, _stream_of(q)), "vdmi_decay_attn_bwd")
    return dq, dk, dv, dstate


def _decay_operands(q, k, v, state):
    """q, k, v [b, inner, n, heads, d] and the state as the kernels read them, of [b, n, heads, d] or the former."""
    if q.dim() == 4:
        q, k, v = q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1)
        state = None if state is None else state.unsqueeze(1)
    if state is not None:
        state = state.contiguous()
        if state.data_ptr() & 15:
            state = state.clone()
    return _row_operand(q), _row_operand(k), _row_operand(v), state


class DecayAttnFn(torch.autograd.Function):
    """o (and the state after the last token) of q, k, v [b(, sites), n, heads, d] and a first state; constants log_decay,
    lengths, scale."""

    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, lengths, scale, return_state):
        ctx.sites = q.dim() == 5
        ops = _decay_operands(q, k, v, state)
        o, last, ws = _decay_forward(*ops, log_decay, lengths, scale, return_state)
        ctx.save_for_backward(*ops, log_decay, lengths, ws)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (o, last) if ctx.sites else (o.squeeze(1), None if last is None else last.squeeze(1))

    @staticmethod
    @_first_order
    def backward(ctx, do, dlast):
        if do is None and dlast is None:
            return (None,) * 8
        need = ctx.needs_input_grad
        if not (ctx.sites or do is None):
            do = do.unsqueeze(1)
        grads = _decay_backward(*ctx.saved_tensors, ctx.scale, do, dlast, need)
        if not ctx.sites:
            grads = [None if g is None else g.squeeze(1) for g in grads]
        dq, dk, dv, dstate = grads
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dstate, None, None, None, None)


def _check_decay(q, k, v, log_decay, state, lead, heads, d):
    if (q.dtype in _FLOAT16S and k.dtype == q.dtype and v.dtype == q.dtype and k.shape == q.shape and v.shape == q.shape and
            d in (32, 64, 128) and log_decay.dtype == torch.float32 and log_decay.shape == (heads,) and not log_decay.requires_grad and
            (state is None or (state.dtype == torch.float32 and state.shape == (*lead, heads, d, d)))):
        return
    if q.dtype not in _FLOAT16S:
        raise VdmiError(f"q, k, v are bfloat16 or float16 (got {q.dtype})")
    if not (k.dtype == q.dtype and v.dtype == q.dtype):
        raise VdmiError(f"q, k, v have one dtype (got {q.dtype}, {k.dtype}, {v.dtype})")
    if not (k.shape == q.shape and v.shape == q.shape):
        raise VdmiError(f"q, k, v have one shape (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    if d not in (32, 64, 128):
        raise VdmiError(f"heads of 32, 64 or 128 features (got {d})")
    if log_decay.requires_grad:
        raise VdmiError("log_decay is a constant of the layer: no gradient is computed for it")
    if not (log_decay.dtype == torch.float32 and log_decay.shape == (heads,)):
        raise VdmiError(f"log_decay is float32 [{heads}] (got {log_decay.dtype} {tuple(log_decay.shape)})")
    raise VdmiError(f"the state is float32 {(*lead, heads, d, d)} (got {state.dtype} {tuple(state.shape)})")


def _scale(scale, d):
    if scale is None:
        return d ** -0.5
    scale = float(scale)
    if not 2.0 ** -126 <= abs(scale) <= 2.0 ** 126:
        raise VdmiError(f"scale is from 2^-126 to 2^126 in magnitude (got {scale})")
    return scale


def decay_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """Linear attention over time whose memory of a token fades by exp(log_decay[head]) per step:
    S_t = exp(log_decay) S_(t-1) + k_t v_t^T, o_t = scale * q_t S_t.  Differentiable in q, k, v and initial_state.

    q, k, v: bfloat16 or float16 [b, n, heads, d] or, for the sequences of many sites, [b, sites, n, heads, d]; any strides
    (views of qkv rows are read in place where their rows are 16-byte aligned).  d is 32, 64 or 128.  log_decay: float32
    [heads], at most 0, a constant (a NaN makes its head NaN).  scale: d^-0.5 by default, 2^-126 to 2^126 in magnitude.
    initial_state: float32 [b(, sites), heads, d, d], S before the first token (zeros by default).  lengths: int32
    [b(, sites)] - tokens from there on are padding: they do not matter, their outputs and gradients are zeros.
    return_state: also return S after the last token, for decay_attention_step or the next piece of the sequence.  Returns o
    like q (in q's order of dimensions in memory unless that parts tokens by more than 2^25 elements), or (o, state).

    Pairs scale * q_t k_j and states enter products as sums of two operands of q's dtype, so that results are rounded once,
    when they are stored: in float16 they have to stay within 65504, and 2^-36 of small ones is lost (the state that is
    returned is float32 throughout).  A token that is not finite makes the outputs from it on not finite and may make up to 31
    earlier ones of its own sequence so; other sequences and tokens behind lengths have no such effect."""
    dims = q.dim()
    if dims not in (4, 5):
        raise VdmiError(f"q is [b, n, heads, d] or [b, sites, n, heads, d] (got {dims} dimensions)")
    lead, (n, heads, d) = q.shape[:-3], q.shape[-3:]
    _on_gpu(q, k, v, log_decay, initial_state, lengths)
    _check_decay(q, k, v, log_decay, initial_state, lead, heads, d)
    scale = _scale(scale, d)
    if lengths is not None:
        if not (lengths.dtype == torch.int32 and lengths.shape == lead):
            raise VdmiError(f"lengths is int32 {tuple(lead)} (got {lengths.dtype} {tuple(lengths.shape)})")
        lengths = lengths.contiguous()
    if q.numel() == 0:
        # no sequences, or sequences of no tokens: the state stays
        o = _linked(q * k * v, initial_state)
        if not return_state:
            return o
        return o, (torch.zeros(*lead, heads, d, d, device=q.device) if initial_state is None else initial_state.clone())
    log_decay = log_decay.contiguous()
    if _wants_grad(q, k, v, initial_state):
        o, last = DecayAttnFn.apply(q, k, v, initial_state, log_decay, lengths, scale, bool(return_state))
        return (o, last) if return_state else o
    o, last, _ = _decay_forward(*_decay_operands(q, k, v, initial_state), log_decay, lengths, scale, return_state)
    if dims == 4:
        o, last = o.squeeze(1), None if last is None else last.squeeze(1)
    return (o, last) if return_state else o


def decay_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One more token of every sequence: state (float32 [..., heads, d, d], contiguous) is updated in place to
    exp(log_decay) state + k v^T, and scale * q state is returned.  q, k, v: bfloat16 or float16 [..., heads, d].  For
    sampling: no gradients."""
    if q.dim() < 2:
        raise VdmiError(f"q is [..., heads, d] (got {q.dim()} dimensions)")
    shape = q.shape
    lead, (heads, d) = shape[:-2], shape[-2:]
    _on_gpu(q, k, v, log_decay, state)
    _check_decay(q, k, v, log_decay, state, lead, heads, d)
    scale = _scale(scale, d)
    if not state.is_contiguous() or state.data_ptr() & 15:
        raise VdmiError("the state is contiguous and 16-byte aligned")
    if _wants_grad(q, k, v, state):
        raise VdmiError("decay_attention_step computes no gradients: call it under torch.no_grad(), or decay_attention")
    o = torch.empty(shape, device=q.device, dtype=q.dtype)
    if q.numel() == 0:
        return o
    if q.dim() != 3:
        q, k, v = q.reshape(-1, heads, d), k.reshape(-1, heads, d), v.reshape(-1, heads, d)
    (qb, qh, q1), (kb, kh, k1), (vb, vh, v1) = q.stride(), k.stride(), v.stride()
    if q1 != 1 or k1 != 1 or v1 != 1:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        qb = kb = vb = heads * d
        qh = kh = vh = d
    strides = _I64x8(qb, qh, kb, kh, vb, vh, heads * d, d)
    _decay_step(q, k, v, o, strides, log_decay.contiguous(), state, scale)
    if not state.is_inference():
        _increment_version((state,))            # written outside torch: a backward that kept it has to know
    return o


@_there
def _decay_step(q, k, v, o, strides, log_decay, state, scale):
    seqs, heads, d = q.shape
    check(_lib.lib().vdmi_decay_attn_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), strides, log_decay.data_ptr(),
                                          state.data_ptr(), _DTYPES[q.dtype], seqs, heads, d, scale, _stream_of(q)),
          "vdmi_decay_attn_step")


# ---------------------------------------------------------------------------------------------------------------------
# the norms before and after a block
# ---------------------------------------------------------------------------------------------------------------------
def _rows2(t: torch.Tensor) -> torch.Tensor:
    """t [..., c] as [rows][c] with contiguous columns: a view where the rows have one pitch, else a copy."""
    r = t.reshape(-1, t.shape[-1])
    rows, c = r.shape
    pitch, one = r.stride()
    return r if one == 1 and (rows == 1 or pitch >= c) else r.contiguous()


def _pitch(r: torch.Tensor) -> int:
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def _stride_of(p, c: int) -> int:
    return c if p is not None and p.dim() == 2 and p.shape[0] > 1 else 0


@_there
def _norm_forward(xr, hr, pw, gate, w, scale, shift, shape, alpha, kind, post_kind, eps, want_y):
    """(out, y) of rows xr, hr [rows][c] and contiguous parameters."""
    out = None if hr is None else xr.new_empty(shape)
    y = xr.new_empty(shape) if want_y else None
    rows, c = xr.shape
    a = _lib.BlockNormArgs(
        _DTYPES[xr.dtype], c, _lib.NORM_KINDS[kind], _lib.NORM_KINDS[post_kind], rows, rows // shape[0], eps, alpha,
        xr.data_ptr(), _ptr(hr), _ptr(out), _ptr(y), None, None, None, None,
        _pitch(xr), c if hr is None else _pitch(hr), c, c, c, c, c, c,
        _ptr(pw), _ptr(gate), _ptr(w), _ptr(scale), _ptr(shift), _stride_of(gate, c), _stride_of(scale, c), _stride_of(shift, c))
    check(_lib.lib().vdmi_block_norm_fwd(a, _stream_of(xr)), "vdmi_block_norm_fwd")
    return out, y


@_there
def _norm_backward(xr, hr, pw, gate, w, scale, shift, shape, alpha, kind, post_kind, eps, need, dout, dy):
    rows, c = xr.shape
    if dout is not None:
        dout = _rows2(dout if dout.dtype == xr.dtype else dout.to(xr.dtype))
    if dy is not None:
        dy = _rows2(dy if dy.dtype == xr.dtype else dy.to(xr.dtype))
    dx = xr.new_empty(shape) if need[0] else None
    dh = xr.new_empty(shape) if need[1] else None
    # without dy nothing is learnt about the second norm's parameters
    like = torch.empty_like if dy is not None else torch.zeros_like
    dpw, dgate = torch.empty_like(pw) if need[2] else None, torch.empty_like(gate) if need[3] else None
    dw, dscale, dshift = like(w) if need[4] else None, like(scale) if need[5] else None, like(shift) if need[6] else None
    on = dy is not None
    a = _lib.BlockNormArgs(
        _DTYPES[xr.dtype], c, _lib.NORM_KINDS[kind], _lib.NORM_KINDS[post_kind], rows, rows // shape[0], eps, alpha,
        xr.data_ptr(), _ptr(hr), None, None, _ptr(dout), _ptr(dy), _ptr(dx), _ptr(dh),
        _pitch(xr), c if hr is None else _pitch(hr), c, c, c if dout is None else _pitch(dout), _pitch(dy) if on else c, c, c,
        _ptr(pw), _ptr(gate), _ptr(w), _ptr(scale), _ptr(shift), _stride_of(gate, c), _stride_of(scale, c), _stride_of(shift, c),
        _ptr(dpw), _ptr(dgate), _ptr(dw) if on else None, _ptr(dscale) if on else None, _ptr(dshift) if on else None)
    lib = _lib.lib()
    size = lib.vdmi_block_norm_bwd_workspace_bytes(a)
    if size:
        ws = torch.empty(size, device=xr.device, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
    check(lib.vdmi_block_norm_bwd(a, _stream_of(xr)), "vdmi_block_norm_bwd")
    return dx, dh, dpw, dgate, dw, dscale, dshift


class BlockNormFn(torch.autograd.Function):
    """(out, y) of rows x, h and parameters; out None without h, y None unless want_y."""

    @staticmethod
    def forward(ctx, x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y):
        ops = _norm_operands(x, h, post_weight, gate, weight, scale, shift)
        shape = x.shape
        out, y = _norm_forward(*ops, shape, alpha, kind, post_kind, eps, want_y)
        ctx.save_for_backward(*ops)
        ctx.meta = (shape, alpha, kind, post_kind, eps)
        ctx.set_materialize_grads(False)
        return out, y

    @staticmethod
    @_first_order
    def backward(ctx, dout, dy):
        if dout is None and dy is None:
            return (None,) * 12
        return (*_norm_backward(*ctx.saved_tensors, *ctx.meta, ctx.needs_input_grad, dout, dy), None, None, None, None, None)


def _norm_operands(x, h, pw, gate, w, scale, shift):
    return (_rows2(x), None if h is None else _rows2(h), None if pw is None else pw.contiguous(),
            None if gate is None else gate.contiguous(), None if w is None else w.contiguous(),
            None if scale is None else scale.contiguous(), None if shift is None else shift.contiguous())


def _block_norm(x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y):
    _on_gpu(x, h, post_weight, gate, weight, scale, shift)
    if x.dtype not in _DTYPES:
        raise VdmiError(f"rows are bfloat16, float16 or float32 (got {x.dtype})")
    if x.dim() < 2 or not 1 <= x.shape[-1] <= 8192:
        raise VdmiError(f"rows are [samples, ..., c] with c from 1 to 8192 (got {tuple(x.shape)})")
    if h is not None and not (h.dtype == x.dtype and h.shape == x.shape):
        raise VdmiError(f"x and h are alike (got {x.dtype} {tuple(x.shape)}, {h.dtype} {tuple(h.shape)})")
    b, c = x.shape[0], x.shape[-1]
    row, one, rows, f32 = (c,), (1, c), (b, c), torch.float32
    for p in (post_weight, weight):
        if p is not None and not (p.dtype is f32 and p.shape == row):
            raise VdmiError(f"{'weight' if p is weight else 'post_weight'} is float32 [{c}]")
    for p in (gate, scale, shift):
        if p is not None and not (p.dtype is f32 and (p.shape == rows or p.shape == row or p.shape == one)):
            raise VdmiError(f"{'gate' if p is gate else 'scale' if p is scale else 'shift'} is float32 [{c}], [1, {c}] or [{b}, {c}]")
    if kind not in ("rms", "layer"):
        raise VdmiError(f"kind is 'rms' or 'layer' (got {kind!r})")
    if post_kind not in ("rms", "layer", None):
        raise VdmiError(f"the kind of the norm after the block is 'rms', 'layer' or None (got {post_kind!r})")
    eps, alpha = float(eps), float(alpha)
    if not (0 <= eps < 1e30 and abs(alpha) < 3e38):
        raise VdmiError(f"eps is not negative and alpha finite (got {eps}, {alpha})")
    if x.numel() == 0:
        out = x if h is None else _linked(x + h, post_weight, gate)
        return (None if h is None else out), (_linked(out * 1, weight, scale, shift) if want_y else None)
    if _wants_grad(x, h, post_weight, gate, weight, scale, shift):
        return BlockNormFn.apply(x, h, post_weight, gate, weight, scale, shift, alpha, kind, post_kind, eps, want_y)
    return _norm_forward(*_norm_operands(x, h, post_weight, gate, weight, scale, shift), x.shape, alpha, kind, post_kind, eps, want_y)


def norm_before(x, weight=None, scale=None, shift=None, *, kind="rms", eps=1e-5):
    """N(x) * weight * (1 + scale) + shift, the norm before a block.  x: bfloat16, float16 or float32 [samples, ..., c]; N
    over the last dimension, x / sqrt(mean x^2 + eps) (kind "rms") or (x - mean) / sqrt(var + eps) ("layer").  weight:
    float32 [c]; scale, shift: float32 [c] or one row per sample, [samples, c]; each may be absent.  Differentiable in all."""
    return _block_norm(x, None, None, None, weight, scale, shift, 1.0, kind, None, eps, True)[1]


def norm_after(x, h, weight=None, gate=None, *, alpha=1.0, kind="rms", eps=1e-5):
    """alpha x + gate * P(h) * weight: a block's output h behind its norm (kind "rms" or "layer"; None: h as it is) and
    gate (float32 [c] or [samples, c]) added to the residual x.  Differentiable in x, h and the parameters."""
    if h is None:
        raise VdmiError("h, the block's output, is missing")
    return _block_norm(x, h, weight, gate, None, None, None, alpha, "rms", kind, eps, False)[0]


def norm_between(x, h, post_weight=None, gate=None, weight=None, scale=None, shift=None, *, alpha=1.0, kind="rms",
                 post_kind="rms", eps=1e-5):
    """From one block to the next in one pass: out = norm_after(x, h, post_weight, gate) and y = norm_before of it with
    weight, scale, shift (of the sum before it is rounded to x's dtype).  Returns (out, y)."""
    if h is None:
        raise VdmiError("h, the block's output, is missing")
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
        """The values the codes stand for, in the packed tensor's shape; in float16 at most 65504, also where rows of another
        type held more."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            raise VdmiError(f"rows are bfloat16, float16 or float32 (got {dtype})")
        out = torch.empty(self.shape, device=self.codes.device, dtype=dtype)
        if out.numel():
            _unpack(self.codes, self.exps, out)
        return out


@_there
def _unpack(codes, exps, out):
    rows, c = codes.shape
    check(_lib.lib().vdmi_rows8_unpack(codes.data_ptr(), exps.data_ptr(), out.data_ptr(), c, _DTYPES[out.dtype], rows, c,
                                       _stream_of(out)), "vdmi_rows8_unpack")


@_there
def _pack(x):
    r = _aligned_rows(x)
    rows, c = r.shape
    codes = torch.empty((rows, c), device=x.device, dtype=torch.uint8)
    exps = torch.empty((rows, (c + 31) // 32), device=x.device, dtype=torch.uint8)
    if rows:
        check(_lib.lib().vdmi_rows8_pack(r.data_ptr(), _pitch(r), codes.data_ptr(), exps.data_ptr(), _DTYPES[x.dtype], rows, c,
                                         _stream_of(x)), "vdmi_rows8_pack")
    return Rows8(codes, exps, tuple(x.shape), x.dtype)


@_there
def _wgrad(dy, kept, bias):
    rows, cin = kept.codes.shape
    cout = dy.shape[-1]
    if rows == 0:
        dw, db = torch.zeros(cout, cin, device=dy.device), torch.zeros(cout, device=dy.device)
        return (dw, db) if bias else dw
    d = _aligned_rows(dy)
    lib = _lib.lib()
    dw = torch.empty((cout, cin), device=dy.device, dtype=torch.float32)
    db = torch.empty(cout, device=dy.device, dtype=torch.float32) if bias else None
    ws = torch.empty(lib.vdmi_rows8_wgrad_workspace_bytes(cin, cout, rows), device=dy.device, dtype=torch.uint8)
    check(lib.vdmi_rows8_wgrad(kept.codes.data_ptr(), kept.exps.data_ptr(), d.data_ptr(), _pitch(d), dw.data_ptr(), _ptr(db),
                               cin, cout, rows, ws.data_ptr(), _stream_of(dy)), "vdmi_rows8_wgrad")
    return (dw, db) if bias else dw


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """_rows2 of t's values, at 16-byte aligned rows."""
    r = _rows2(t.detach())
    return r.clone(memory_format=torch.contiguous_format) if r.data_ptr() & 15 or _pitch(r) % 8 or _pitch(r) > _lib.ROWS8_MAX_PITCH else r


def pack_rows8(x: torch.Tensor) -> Rows8:
    """x [..., c] (bfloat16, float16 or float32, c a multiple of 8) in 8 bits: e4m3 codes times the least power of two per
    row and 32 channels that holds the largest magnitude.  Off by 2^-4 of a value at most or, for the smallest ones, under
    2^-17 of their group's largest (2^-128 where that is below 224 * 2^-118); infinities and NaN come back as NaN, magnitudes
    beyond 448 * 2^119 as that."""
    _on_gpu(x)
    if x.dtype not in _DTYPES:
        raise VdmiError(f"rows are bfloat16, float16 or float32 (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] == 0 or x.shape[-1] % 8:
        raise VdmiError(f"rows of a multiple of 8 channels (got {tuple(x.shape)})")
    return _pack(x)


def rows8_wgrad(kept: Rows8, dy: torch.Tensor, bias: bool = False):
    """float32 [cout][cin] weight gradient of a Linear from its input kept in 8 bits and the gradient dy [..., cout] of its
    output (bfloat16 rows); with bias also the bias gradient: (dw, db)."""
    _on_gpu(kept.codes, dy)
    rows = kept.codes.shape[0]
    if dy.dim() < 1:
        raise VdmiError("dy is [..., cout] (got no dimensions)")
    cout = dy.shape[-1]
    if dy.dtype != torch.bfloat16:
        raise VdmiError(f"dy is bfloat16 (got {dy.dtype})")
    if cout == 0 or cout % 8:
        raise VdmiError(f"a multiple of 8 output channels (got {cout})")
    if dy.numel() != rows * cout:
        raise VdmiError(f"dy has a row for each of the {rows} kept rows (got {tuple(dy.shape)})")
    return _wgrad(dy, kept, bias)


class LinearRows8Fn(torch.autograd.Function):
    """y = x weight^T + bias on the row GEMMs of train_hip.py; what is kept of x for the weight gradient is 8 bits wide."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        y, kept = _linear(x, weight, bias, ctx.needs_input_grad[1])
        ctx.save_for_backward(weight, *((kept.codes, kept.exps) if kept else ()))
        ctx.shape = tuple(x.shape)
        return y

    @staticmethod
    @_first_order
    @_plain
    def backward(ctx, dy):
        weight, *kept = ctx.saved_tensors
        return _linear_backward(dy, weight, kept, ctx.shape, ctx.needs_input_grad)


def _dense(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it, contiguous and 16-byte aligned: what the row GEMMs read."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


@_plain
@_there
def _linear(x, weight, bias, keep):
    from .train_hip import _linear_pack, conv_rows
    xr = _dense(x.reshape(-1, x.shape[-1]))
    y = conv_rows(xr, _linear_pack(weight.detach(), False), None if bias is None else _dense(bias.detach().float()),
                  1, 1, 1, xr.shape[0])
    return y.view(*x.shape[:-1], weight.shape[0]), pack_rows8(xr) if keep else None


@_there
def _linear_backward(dy, weight, kept, shape, need):
    from .train_hip import _linear_pack, colsum_rows, conv_rows
    dx = dw = db = None
    d = _dense(dy.to(torch.bfloat16).reshape(-1, dy.shape[-1]))
    if need[0]:
        dx = conv_rows(d, _linear_pack(weight.detach(), True), None, 1, 1, 1, d.shape[0]).view(shape)
    if need[1]:
        dw = rows8_wgrad(Rows8(*kept, shape, torch.bfloat16), d, bias=need[2])
        dw, db = dw if need[2] else (dw, None)
    elif need[2]:
        db = colsum_rows(d)             # not torch's sum: what it clears is wrong from a graph's second replay on
    return dx, dw, db


def linear_rows8(x: torch.Tensor, weight: torch.Tensor, bias=None) -> torch.Tensor:
    """F.linear(x, weight, bias) on the library's row GEMMs for bfloat16 x [..., cin] and float32 weight [cout, cin]
    (multiples of 32), whose input is kept for the weight gradient in 8 bits (about half of a bfloat16 copy).  Output and
    input gradient are exactly those of the bfloat16 path; only the weight gradient sees the rounding to 8 bits.  Needs the
    bfloat16 build."""
    _on_gpu(x, weight, bias)
    if _lib.PRECISION != "bf16":
        raise VdmiError("the training layers exchange bfloat16 rows: VDMI_PRECISION=f16 serves sampling only")
    if not (x.dtype == torch.bfloat16 and weight.dtype == torch.float32 and weight.dim() == 2):
        raise VdmiError(f"x is bfloat16 and weight float32 [cout, cin] (got {x.dtype}, {weight.dtype} {tuple(weight.shape)})")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1] or (bias is not None and bias.shape != (weight.shape[0],)):
        raise VdmiError(f"x [..., cin], weight [cout, cin], bias [cout] (got {tuple(x.shape)}, {tuple(weight.shape)})")
    if weight.shape[0] % 32 or weight.shape[1] % 32:
        raise VdmiError(f"multiples of 32 channels (got {tuple(weight.shape)})")
    if x.numel() == 0:
        return torch.nn.functional.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))
    if not _wants_grad(x, weight, bias):        # nothing to keep: needs_input_grad does not know of no_grad
        return _linear(x, weight, bias, False)[0]
    return LinearRows8Fn.apply(x, weight, bias)
