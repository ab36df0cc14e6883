"""Causal linear attention with a decay for each head on MI355X: the identity-map companion of
``identity_linear_attn`` whose earlier tokens fade, in chunks for prompts and training and one token at a
time on its state (no reference function; the reference's identity map,
benchmarks/chunked_attention_benchmark.py:81-93, is the case without decay).

With g = exp(log_decay[h]) for head h and s = ``scale``:

    y_t = s (sum_{u <= t} g^(t - u) (q_t . k_u) v_u + g^(t + 1) q_t S_in)
    S_out = g^L S_in + sum_{u < L} g^(L - 1 - u) k_u v_u^T            (L tokens)

``decay_linear_attn`` is differentiable by q, k, v and ``state_in``; the decay is a constant of the model.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .pytorch_attention import _as_kernel_input, _check_qkv, _compute_dtype

__all__ = ["decay_linear_attn", "decay_decode_step"]

_MAX_DIM = 128
_Strides = ctypes.c_longlong * 3
_KERNEL_TYPES = (torch.float32, torch.bfloat16)


def _operand(x: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """x in dtype dt with unit last stride and no negative ones; views of other strides are read in place."""
    if x.dtype != dt:
        x = x.to(dt)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _strides(x: torch.Tensor):
    """Strides of batch, head and token, or None for a contiguous tensor."""
    if x.is_contiguous():
        return None
    s = x.stride()
    return _Strides(s[0], s[1], s[2])


def _same_device(dev: int, like, *others) -> None:
    for x in others:
        if x.get_device() != dev or dev < 0:
            _lib.require_gpu(like, *others)


def _check_decay(log_decay: torch.Tensor, h: int) -> torch.Tensor:
    if log_decay.dtype != torch.float32 or log_decay.dim() != 1 or log_decay.shape[0] != h:
        raise _lib.BasedLAError(f"log_decay must be fp32 of shape ({h},)")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise _lib.BasedLAError("log_decay is a constant: there is no gradient by it (pass log_decay.detach())")
    return log_decay.contiguous()


def _check_dims(d: int, dv: int) -> None:
    if not (1 <= d <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise _lib.BasedLAError(f"the decay kernels take 1 <= d, dv <= {_MAX_DIM} (got d={d}, dv={dv})")


def _check_state(state, shape, name):
    if state.dtype != torch.float32 or state.shape != shape:
        raise _lib.BasedLAError(f"{name} must be fp32 {shape}")


def _workspace(dev, b, h, t, d, dv, backward, device):
    n = _lib.lib().la_decay_workspace_bytes(b, h, t, d, dv, backward)
    if n == 0:
        return None, 0, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt):
    b, h, t, d = q.shape
    dv, dev = v.shape[-1], q.get_device()
    cdt = _compute_dtype(q.dtype)
    kdt = odt if odt in _KERNEL_TYPES else torch.float32
    qc, kc, vc = _operand(q, cdt), _operand(k, cdt), _operand(v, cdt)
    si = None if state_in is None else _as_kernel_input(state_in, torch.float32)
    out = torch.empty((b, h, t, dv), dtype=kdt, device=q.device)
    state = torch.empty((b, h, d, dv), dtype=torch.float32, device=q.device) if return_state else None
    if t == 0 and return_state:      # nothing is launched: no token changes the state
        state.zero_() if si is None else state.copy_(si)
    ws, ws_ptr, ws_bytes = _workspace(dev, b, h, t, d, dv, 0, q.device)
    _lib.launch(dev, "la_decay_fwd", qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), _lib.dtype_code(cdt), out.data_ptr(),
                _lib.dtype_code(kdt), b, h, t, d, dv, _strides(qc), _strides(kc), _strides(vc), log_decay.data_ptr(),
                _lib.ptr(lengths), scale, _lib.ptr(si), _lib.ptr(state), ws_ptr, ws_bytes, _lib.stream_of(q))
    return (out if out.dtype == odt else out.to(odt)), state, ws


class _NoSecond(torch.autograd.Function):
    """Gradients that are taken with ``create_graph=True``: using them for second derivatives raises."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(None if x is None else x.view_as(x) for x in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("decay_linear_attn has no second derivatives")


class _DecayAttention(torch.autograd.Function):
    """The forward kernel under autograd; the backward pass is ``la_decay_bwd``."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, lengths, scale, state_in, return_state, odt):
        y, state, ctx.segments = _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
        ctx.save_for_backward(q, k, v, log_decay, lengths, state_in)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    def backward(ctx, dy, dstate):
        if torch.is_grad_enabled():
            with torch.no_grad():
                grads = _backward(ctx, dy, dstate)
            dq, dk, dv, ds = _NoSecond.apply(*(None if x is None else x.requires_grad_() for x in grads))
        else:
            dq, dk, dv, ds = _backward(ctx, dy, dstate)
        return dq, dk, dv, None, None, None, ds, None, None


def _backward(ctx, dy, dstate):
    q, k, v, log_decay, lengths, state_in = ctx.saved_tensors
    b, h, t, d = q.shape
    dv, dev, device = v.shape[-1], q.get_device(), q.device
    cdt = _compute_dtype(q.dtype)
    if dy is None:
        dy = torch.zeros((b, h, t, dv), dtype=cdt, device=device)
    qc, kc, vc, dyc = _operand(q, cdt), _operand(k, cdt), _operand(v, cdt), _operand(dy, cdt)
    si = None if state_in is None else _as_kernel_input(state_in, torch.float32)
    dso = None if dstate is None else _as_kernel_input(dstate, torch.float32)
    dq = torch.empty((b, h, t, d), dtype=cdt, device=device)
    dk = torch.empty((b, h, t, d), dtype=cdt, device=device)
    dvo = torch.empty((b, h, t, dv), dtype=cdt, device=device)
    want = state_in is not None and ctx.needs_input_grad[6]
    dsi = torch.empty((b, h, d, dv), dtype=torch.float32, device=device) if want else None
    if t == 0 and want:
        dsi.zero_() if dso is None else dsi.copy_(dso)
    seg = ctx.segments      # the forward pass's states of the segments, if it had any
    ws, ws_ptr, ws_bytes = _workspace(dev, b, h, t, d, dv, 0 if seg is not None else 1, device)
    _lib.launch(dev, "la_decay_bwd", qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), dyc.data_ptr(), _lib.dtype_code(cdt),
                dq.data_ptr(), dk.data_ptr(), dvo.data_ptr(), b, h, t, d, dv, _strides(qc), _strides(kc), _strides(vc),
                _strides(dyc), log_decay.data_ptr(), _lib.ptr(lengths), ctx.scale, _lib.ptr(si), _lib.ptr(dso),
                _lib.ptr(dsi), _lib.ptr(seg), ws_ptr, ws_bytes, _lib.stream_of(q))
    if cdt != q.dtype:
        dq, dk, dvo = dq.to(q.dtype), dk.to(q.dtype), dvo.to(q.dtype)
    return dq, dk, dvo, dsi


def decay_linear_attn(q, k, v, log_decay, scale=None, state_in=None, return_state=False, lengths=None, out_dtype=None):
    """Causal linear attention with a decay for each head, through ``la_decay_fwd`` / ``la_decay_bwd``.

    q, k: (b, h, t, d); v: (b, h, t, dv), any strides; log_decay: fp32 (h,), in general <= 0 (-inf: each token
    sees itself only).  ``scale`` defaults to 1/sqrt(d).  ``state_in``: fp32 (b, h, d, dv), an earlier call's
    state that these tokens follow; ``return_state`` also returns the state after the last token, in the
    same layout, which ``decay_decode_step`` goes on from.  ``lengths``: int32 (b,), the tokens of each
    sequence of a batch padded on the right; rows behind them are not read, their outputs and gradients
    are zeros.  Returns ``out_dtype`` (default q.dtype; bf16 and fp32 run as they are, fp16 and fp64
    through fp32).  Differentiable (once) by q, k, v and ``state_in``, through the output and the state.
    """
    _check_qkv(q, k, v)
    b, h, t, d = q.shape
    dv, dev = v.shape[3], q.get_device()
    _check_dims(d, dv)
    _same_device(dev, q, log_decay)
    log_decay = _check_decay(log_decay, h)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if lengths is not None:
        _same_device(dev, q, lengths)
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (b,):
            raise _lib.BasedLAError(f"lengths must be int32 of shape ({b},)")
        lengths = lengths.contiguous()
    if state_in is not None:
        _same_device(dev, q, state_in)
        _check_state(state_in, (b, h, d, dv), "state_in")
    odt = q.dtype if out_dtype is None else out_dtype
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state_in is not None and state_in.requires_grad)):
        y, state = _DecayAttention.apply(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
    else:
        y, state, _ = _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
    return (y, state) if return_state else y


def _kernel_row(x: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """x in dtype dt and contiguous (element loads: no alignment beyond an element's)."""
    return x if x.dtype == dt and x.is_contiguous() else x.to(dt).contiguous()


def decay_decode_step(q, k, v, log_decay, state, scale=None):
    """One token on a state of ``decay_linear_attn`` through ``la_decay_step``: ``state`` (b, h, d, dv) fp32,
    contiguous, becomes g state + k v^T in place, and scale q^T state is returned, in q.dtype.

    q, k: (b, h, d) or (b, h, 1, d); v: (b, h, dv) or (b, h, 1, dv) -- one token per head.
    """
    dims = q.dim()
    if dims not in (3, 4) or k.dim() != dims or v.dim() != dims:
        raise _lib.BasedLAError("q, k must be (b, h, d) and v (b, h, dv), or all with one token per head")
    qs, vs = q.shape, v.shape
    if dims == 4 and not (qs[2] == k.shape[2] == vs[2] == 1):
        raise _lib.BasedLAError("decode takes one token per head: shape (b, h, 1, d)")
    dev = q.get_device()
    _same_device(dev, q, k, v, state, log_decay)
    if k.shape != qs or vs[:-1] != qs[:-1]:
        raise _lib.BasedLAError("q, k must be (b, h, d) and v (b, h, dv)")
    dt = q.dtype
    if k.dtype != dt or v.dtype != dt:
        raise _lib.BasedLAError("q, k, v must share one dtype")
    b, h, d, dv = qs[0], qs[1], qs[-1], vs[-1]
    _check_dims(d, dv)
    log_decay = _check_decay(log_decay, h)
    _check_state(state, (b, h, d, dv), "state")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise _lib.BasedLAError("state must be contiguous and 16-byte aligned: it is updated in place")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise _lib.BasedLAError("decay_decode_step has no gradient: call it under torch.no_grad()")
    cdt = _compute_dtype(dt)
    kdt = dt if dt in _KERNEL_TYPES else torch.float32
    qc, kc, vc = _kernel_row(q, cdt), _kernel_row(k, cdt), _kernel_row(v, cdt)
    out = torch.empty(vs, dtype=kdt, device=q.device)
    _lib.launch(dev, "la_decay_step", qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), _lib.dtype_code(cdt), log_decay.data_ptr(),
                state.data_ptr(), out.data_ptr(), _lib.dtype_code(kdt), b, h, d, dv,
                1.0 / math.sqrt(d) if scale is None else float(scale), _lib.stream_of(q))
    if not state.is_inference():      # autograd has not seen the update in place
        torch.autograd.graph.increment_version(state)
    return out if kdt == dt else out.to(dt)
