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


def _operand(x: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """x in dtype dt with unit last stride and no negative ones; views of other strides are read in place."""
    if x.dtype != dt:
        x = x.to(dt)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _strides(x: torch.Tensor):
    return _Strides(x.stride(0), x.stride(1), x.stride(2))


def _check_decay(log_decay: torch.Tensor, like: torch.Tensor, h: int) -> torch.Tensor:
    _lib.require_gpu(like, log_decay)
    if log_decay.dtype != torch.float32 or tuple(log_decay.shape) != (h,):
        raise _lib.BasedLAError(f"log_decay must be fp32 of shape ({h},)")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise _lib.BasedLAError("log_decay is a constant: there is no gradient by it (pass log_decay.detach())")
    return log_decay.contiguous()


def _check_dims(d: int, dv: int) -> None:
    if not (1 <= d <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise _lib.BasedLAError(f"the decay kernels take 1 <= d, dv <= {_MAX_DIM} (got d={d}, dv={dv})")


def _check_state(state, like, shape, name):
    _lib.require_gpu(like, state)
    if state.dtype != torch.float32 or tuple(state.shape) != shape:
        raise _lib.BasedLAError(f"{name} must be fp32 {shape}")


def _workspace(L, b, h, t, d, dv, backward, device):
    n = int(L.la_decay_workspace_bytes(b, h, t, d, dv, backward))
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt):
    b, h, t, d = q.shape
    dv = v.shape[-1]
    cdt = _compute_dtype(q.dtype)
    kdt = odt if odt in (torch.float32, torch.bfloat16) else torch.float32
    qc, kc, vc = (_operand(x, cdt) for x in (q, k, v))
    si = None if state_in is None else _as_kernel_input(state_in, torch.float32)
    out = torch.empty(b, h, t, dv, dtype=kdt, device=q.device)
    state = torch.empty(b, h, d, dv, dtype=torch.float32, device=q.device) if return_state else None
    if t == 0 and return_state:      # nothing is launched: no token changes the state
        state.zero_() if si is None else state.copy_(si)
    L = _lib.lib()
    ws, ws_bytes = _workspace(L, b, h, t, d, dv, 0, q.device)
    rc = L.la_decay_fwd(_lib.ptr(qc), _lib.ptr(kc), _lib.ptr(vc), _lib.dtype_code(cdt), _lib.ptr(out),
                        _lib.dtype_code(kdt), b, h, t, d, dv, _strides(qc), _strides(kc), _strides(vc),
                        _lib.ptr(log_decay), _lib.ptr(lengths), scale, _lib.ptr(si), _lib.ptr(state), _lib.ptr(ws),
                        ws_bytes, _lib.stream_of(q))
    _lib.check(rc, "la_decay_fwd")
    return (out if out.dtype == odt else out.to(odt)), state


class _DecayAttention(torch.autograd.Function):
    """The forward kernel under autograd; the backward pass is ``la_decay_bwd``."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, lengths, scale, state_in, return_state, odt):
        y, state = _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
        ctx.save_for_backward(q, k, v, log_decay, lengths, state_in)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        q, k, v, log_decay, lengths, state_in = ctx.saved_tensors
        b, h, t, d = q.shape
        dv = v.shape[-1]
        cdt = _compute_dtype(q.dtype)
        if dy is None:
            dy = torch.zeros(b, h, t, dv, dtype=cdt, device=q.device)
        qc, kc, vc, dyc = (_operand(x, cdt) for x in (q, k, v, dy))
        si = None if state_in is None else _as_kernel_input(state_in, torch.float32)
        dso = None if dstate is None else _as_kernel_input(dstate, torch.float32)
        dq, dk = (torch.empty(b, h, t, d, dtype=cdt, device=q.device) for _ in range(2))
        dvo = torch.empty(b, h, t, dv, dtype=cdt, device=q.device)
        want = state_in is not None and ctx.needs_input_grad[6]
        dsi = torch.empty(b, h, d, dv, dtype=torch.float32, device=q.device) if want else None
        if t == 0 and want:
            dsi.zero_() if dso is None else dsi.copy_(dso)
        L = _lib.lib()
        ws, ws_bytes = _workspace(L, b, h, t, d, dv, 1, q.device)
        rc = L.la_decay_bwd(_lib.ptr(qc), _lib.ptr(kc), _lib.ptr(vc), _lib.ptr(dyc), _lib.dtype_code(cdt), _lib.ptr(dq),
                            _lib.ptr(dk), _lib.ptr(dvo), b, h, t, d, dv, _strides(qc), _strides(kc), _strides(vc),
                            _strides(dyc), _lib.ptr(log_decay), _lib.ptr(lengths), ctx.scale, _lib.ptr(si),
                            _lib.ptr(dso), _lib.ptr(dsi), _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
        _lib.check(rc, "la_decay_bwd")
        if cdt != q.dtype:
            dq, dk, dvo = (x.to(q.dtype) for x in (dq, dk, dvo))
        return dq, dk, dvo, None, None, None, dsi, None, None


def decay_linear_attn(q, k, v, log_decay, scale=None, state_in=None, return_state=False, lengths=None, out_dtype=None):
    """Causal linear attention with a decay for each head, through ``la_decay_fwd`` / ``la_decay_bwd``.

    q, k: (b, h, t, d); v: (b, h, t, dv), any strides; log_decay: fp32 (h,), <= 0 (-inf: each token sees
    itself only).  ``scale`` defaults to 1/sqrt(d).  ``state_in``: fp32 (b, h, d, dv), an earlier call's
    state that these tokens follow; ``return_state`` also returns the state after the last token, in the
    same layout, which ``decay_decode_step`` goes on from.  ``lengths``: int32 (b,), the tokens of each
    sequence of a batch padded on the right; rows behind them are not read, their outputs and gradients
    are zeros.  Returns ``out_dtype`` (default q.dtype; bf16 and fp32 run as they are, fp16 and fp64
    through fp32).  Differentiable by q, k, v and ``state_in``, through the output and the state.
    """
    _check_qkv(q, k, v)
    b, h, t, d = q.shape
    dv = v.shape[-1]
    _check_dims(d, dv)
    log_decay = _check_decay(log_decay, q, h)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if lengths is not None:
        _lib.require_gpu(q, lengths)
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (b,):
            raise _lib.BasedLAError(f"lengths must be int32 of shape ({b},)")
        lengths = lengths.contiguous()
    if state_in is not None:
        _check_state(state_in, q, (b, h, d, dv), "state_in")
    odt = q.dtype if out_dtype is None else out_dtype
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, state_in)):
        y, state = _DecayAttention.apply(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
    else:
        y, state = _forward(q, k, v, log_decay, lengths, scale, state_in, return_state, odt)
    return (y, state) if return_state else y


def decay_decode_step(q, k, v, log_decay, state, scale=None):
    """One token on a state of ``decay_linear_attn`` through ``la_decay_step``: ``state`` (b, h, d, dv) fp32,
    contiguous, becomes g state + k v^T in place, and scale q^T state is returned, in q.dtype.

    q, k: (b, h, d) or (b, h, 1, d); v: (b, h, dv) or (b, h, 1, dv) -- one token per head.
    """
    if q.dim() not in (3, 4) or k.dim() != q.dim() or v.dim() != q.dim():
        raise _lib.BasedLAError("q, k must be (b, h, d) and v (b, h, dv), or all with one token per head")
    if q.dim() == 4 and not (q.shape[2] == k.shape[2] == v.shape[2] == 1):
        raise _lib.BasedLAError("decode takes one token per head: shape (b, h, 1, d)")
    _lib.require_gpu(q, k, v, state)
    if k.shape != q.shape or v.shape[:-1] != q.shape[:-1]:
        raise _lib.BasedLAError("q, k must be (b, h, d) and v (b, h, dv)")
    if not (q.dtype == k.dtype == v.dtype):
        raise _lib.BasedLAError("q, k, v must share one dtype")
    b, h, d, dv = q.shape[0], q.shape[1], q.shape[-1], v.shape[-1]
    _check_dims(d, dv)
    log_decay = _check_decay(log_decay, q, h)
    _check_state(state, q, (b, h, d, dv), "state")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise _lib.BasedLAError("state must be contiguous and 16-byte aligned: it is updated in place")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v, state)):
        raise _lib.BasedLAError("decay_decode_step has no gradient: call it under torch.no_grad()")
    cdt = _compute_dtype(q.dtype)
    kdt = q.dtype if q.dtype in (torch.float32, torch.bfloat16) else torch.float32
    qc, kc, vc = (_as_kernel_input(x, cdt) for x in (q, k, v))
    out = torch.empty(v.shape, dtype=kdt, device=q.device)
    rc = _lib.lib().la_decay_step(_lib.ptr(qc), _lib.ptr(kc), _lib.ptr(vc), _lib.dtype_code(cdt), _lib.ptr(log_decay),
                                  _lib.ptr(state), _lib.ptr(out), _lib.dtype_code(kdt), b, h, d, dv,
                                  1.0 / math.sqrt(d) if scale is None else float(scale), _lib.stream_of(q))
    _lib.check(rc, "la_decay_step")
    return out if out.dtype == q.dtype else out.to(q.dtype)
