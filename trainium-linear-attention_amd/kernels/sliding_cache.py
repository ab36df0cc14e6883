"""Sliding-window softmax attention for decoding on MI355X: an 8-bit cache of keys and values, and one token
of each sequence at a time over it -- the decode form of ``sliding_window_attn`` (no reference function; the
reference has no decode path), beside ``based_decode_step`` and ``decay_decode_step`` for the linear branch.

The cache holds e4m3 codes in blocks of 64 tokens with a power-of-two scale for each block and head
(include/based_la_cache.h has the layout).  Position p of a sequence lies in block (p // 64) mod ``blocks``:
with room for the longest sequence a plain cache, with less a ring of a sequence's last blocks, which a
window of up to 64 (blocks - 1) + 1 tokens never outruns.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib
from .decay_attention import _KERNEL_TYPES, _kernel_row, _operand, _same_device, _strides
from .pytorch_attention import _compute_dtype

__all__ = ["SlidingCache", "sliding_cache", "sliding_cache_append", "sliding_decode_step"]

CACHE_BLOCK = 64
_E4M3 = torch.float8_e4m3fn


class SlidingCache(NamedTuple):
    """A cache's arrays, all contiguous: k (b, hk, blocks, 64, dp) and v (b, hk, blocks, dvp, 64) e4m3,
    k_scale and v_scale (b, hk, blocks) fp32; d and dv are the widths in use (dp, dvp: 32, 64 or 128)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    d: int
    dv: int

    @property
    def tokens(self) -> int:
        """Places for tokens of each sequence."""
        return self.k.shape[2] * CACHE_BLOCK

    def values(self):
        """The keys (b, hk, tokens, d) and values (b, hk, tokens, dv) that the codes stand for, fp32, by place."""
        k = (self.k.float() * self.k_scale[..., None, None]).flatten(2, 3)[..., :self.d]
        v = (self.v.float() * self.v_scale[..., None, None]).transpose(3, 4).flatten(2, 3)[..., :self.dv]
        return k, v


def _padded(d: int) -> int:
    if not 1 <= d <= 128:
        raise _lib.BasedLAError(f"the cache kernels take 1 <= d, dv <= 128 (got {d})")
    return 32 if d <= 32 else 64 if d <= 64 else 128


def sliding_cache(b, heads, tokens, d, dv=None, device="cuda"):
    """An empty cache for b sequences and ``heads`` key/value heads with room for ``tokens`` tokens each
    (rounded up to whole blocks).  For a window of w tokens over sequences of any length: w + 63."""
    dv = d if dv is None else dv
    dp, dvp, blocks = _padded(d), _padded(dv), -(-int(tokens) // CACHE_BLOCK)
    if blocks < 1:
        raise _lib.BasedLAError("a cache has room for at least one token")
    return SlidingCache(torch.zeros(b, heads, blocks, CACHE_BLOCK, dp, dtype=_E4M3, device=device),
                        torch.zeros(b, heads, blocks, dvp, CACHE_BLOCK, dtype=_E4M3, device=device),
                        torch.zeros(b, heads, blocks, device=device), torch.zeros(b, heads, blocks, device=device), d, dv)


def _check_cache(cache: SlidingCache, like: torch.Tensor, dev: int):
    """The cache's (b, hk, blocks), its arrays checked against each other."""
    k, v, ks, vs, d, dv = cache
    _same_device(dev, like, k, v, ks, vs)
    if k.dim() != 5:
        raise _lib.BasedLAError("cache.k must be (b, hk, blocks, 64, dp)")
    b, hk, blocks, at, dp = k.shape
    if (k.dtype != _E4M3 or v.dtype != _E4M3 or at != CACHE_BLOCK or dp != _padded(d)
            or v.shape != (b, hk, blocks, _padded(dv), CACHE_BLOCK)):
        raise _lib.BasedLAError(f"cache.k and cache.v must be float8_e4m3fn {(b, hk, blocks, CACHE_BLOCK, _padded(d))} and "
                                f"{(b, hk, blocks, _padded(dv), CACHE_BLOCK)}")
    shape = (b, hk, blocks)
    if ks.dtype != torch.float32 or vs.dtype != torch.float32 or ks.shape != shape or vs.shape != shape:
        raise _lib.BasedLAError(f"cache scales must be fp32 {shape}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise _lib.BasedLAError("the cache's arrays must be contiguous: they are updated in place")
    return shape


def _counts(x, like, dev, b, name):
    if x is None:
        return None
    _same_device(dev, like, x)
    if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != b:
        raise _lib.BasedLAError(f"{name} must be int32 of shape ({b},)")
    return x.contiguous()


def sliding_cache_append(cache, k, v, start=None, lengths=None):
    """Prompts, or pieces of them, into the cache, in place, through ``la_sliding_cache_append``: row t of sequence b at
    position start[b] + t, for t < lengths[b].

    k: (b, hk, t, d); v: (b, hk, t, dv), any strides.  ``start``: int32 (b,), default zeros (tokens before it
    have been appended before); ``lengths``: int32 (b,), default t (a batch padded on the right).
    """
    dev = k.get_device()
    b, hk, blocks = _check_cache(cache, k, dev)
    _same_device(dev, k, v)
    if k.dim() != 4 or v.dim() != 4 or k.shape[:2] != (b, hk) or v.shape[:3] != k.shape[:3] \
            or k.shape[3] != cache.d or v.shape[3] != cache.dv:
        raise _lib.BasedLAError(f"k, v must be ({b}, {hk}, t, {cache.d}) and ({b}, {hk}, t, {cache.dv})")
    if k.dtype != v.dtype:
        raise _lib.BasedLAError("k, v must share one dtype")
    start, lengths = _counts(start, k, dev, b, "start"), _counts(lengths, k, dev, b, "lengths")
    cdt = _compute_dtype(k.dtype)
    kc, vc = _operand(k.detach(), cdt), _operand(v.detach(), cdt)
    _lib.launch(dev, "la_sliding_cache_append", kc.data_ptr(), vc.data_ptr(), _lib.dtype_code(cdt), cache.k.data_ptr(),
                cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), _lib.ptr(start), _lib.ptr(lengths),
                b, hk, k.shape[2], cache.d, cache.dv, blocks, _strides(kc), _strides(vc), _lib.stream_of(k))


def sliding_decode_step(q, k, v, cache, lengths, window_size=None, scale=None):
    """One token of each sequence through ``la_sliding_decode_step``: k and v go into the cache at position
    lengths[b] - 1, and the softmax attention of q over the last ``window_size`` positions up to it is
    returned, in q.dtype.

    q: (b, h, d); k: (b, hk, d); v: (b, hk, dv) (or with one token in a third dimension of 1); h is a multiple of
    hk, and query head i reads cached head i // (h / hk).  ``lengths``: int32 (b,), tokens with this one; a
    sequence of 0 takes no part (its output is zero, its cache stays).  ``window_size`` None: every position
    that the cache holds whole blocks of, all of a sequence that fits it.  ``scale`` defaults to 1/sqrt(d).
    """
    dev = q.get_device()
    b, hk, blocks = _check_cache(cache, q, dev)
    d, dv = cache.d, cache.dv
    _same_device(dev, q, k, v)
    squeeze = q.dim() == 4
    if squeeze:
        if k.dim() != 4 or v.dim() != 4 or not (q.shape[2] == k.shape[2] == v.shape[2] == 1):
            raise _lib.BasedLAError("decode takes one token per head: shape (b, h, 1, d)")
        q, k, v = q[:, :, 0], k[:, :, 0], v[:, :, 0]
    qs = q.shape
    if len(qs) != 3 or k.shape != (b, hk, d) or v.shape != (b, hk, dv) or qs[0] != b or qs[2] != d or hk < 1 or qs[1] % hk:
        raise _lib.BasedLAError(f"q must be ({b}, h, {d}) with h a multiple of {hk}, k ({b}, {hk}, {d}), v ({b}, {hk}, {dv})")
    dt = q.dtype
    if k.dtype != dt or v.dtype != dt:
        raise _lib.BasedLAError("q, k, v must share one dtype")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise _lib.BasedLAError("sliding_decode_step has no gradient: call it under torch.no_grad()")
    lengths = _counts(lengths, q, dev, b, "lengths")
    if lengths is None:
        raise _lib.BasedLAError(f"lengths must be int32 of shape ({b},)")
    window = 0 if window_size is None else int(window_size)
    if window_size is not None and not 1 <= window <= CACHE_BLOCK * (blocks - 1) + 1:
        raise _lib.BasedLAError(f"window_size must be >= 1 and at most {CACHE_BLOCK * (blocks - 1) + 1} for this cache "
                                f"(tokens - 63): a window of w tokens needs a cache of w + 63")
    h = qs[1]
    cdt = _compute_dtype(dt)
    kdt = dt if dt in _KERNEL_TYPES else torch.float32
    qc, kc, vc = _kernel_row(q, cdt), _kernel_row(k, cdt), _kernel_row(v, cdt)
    out = torch.empty((b, h, 1, dv) if squeeze else (b, h, dv), dtype=kdt, device=q.device)
    ws_ptr, ws_bytes = 0, _lib.lib().la_sliding_decode_workspace_bytes(b, h, hk, d, dv, blocks, window)
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        ws_ptr = ws.data_ptr()
    _lib.launch(dev, "la_sliding_decode_step", qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), _lib.dtype_code(cdt), out.data_ptr(),
                _lib.dtype_code(kdt), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
                cache.v_scale.data_ptr(), lengths.data_ptr(), b, h, hk, d, dv, blocks, window,
                1.0 / math.sqrt(d) if scale is None else float(scale), ws_ptr, ws_bytes, _lib.stream_of(q))
    return out if kdt == dt else out.to(dt)
