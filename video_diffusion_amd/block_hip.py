"""Operators of a causal layer over time, in training and one frame at a time, on the HIP kernels:

  decay_attention, decay_attention_step   linear attention with a decay per head over whole sequences / one more token
                                          (csrc/decay.hip)

They stand beside the attention layers of train_hip.py, which are a softmax over all frames at once and keep no state.
Element types go by the tensors (bfloat16, float16; states float32) whatever VDMI_PRECISION says.  Calls run on the current
stream of the tensors' device.  There is no fallback: tensors that are not on a GPU and shapes that the kernels do not take
raise VdmiError.
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
