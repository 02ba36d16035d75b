"""Attention over a sliding window with first tokens that stay visible.

The companion of ``attention`` for layers that look at a part of the sequence:
the neighbourhood of each token, and optionally the first tokens (for a
streamed video, the first frame).  It computes in 16-bit operands with FP32
accumulation, with no quantisation, clustering or schedule."""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from .layer import (_PLANS, _TYPES, _Plan, _check_out, _check_status, _meta, _no_rows, _packed_strides, _ptr, _remember,
                    _require_b200, _written)


def _bound(value, name):
    if value is None:
        return -1
    if isinstance(value, bool) or not isinstance(value, int) or value < 0:
        raise ValueError(f"{name} must be a non-negative integer or None")
    return min(value, (1 << 40) - 1)           # positions stay below 2^39 + 2^31: no bound at all


def window_attention(q, k, v, *, window=(None, None), sinks=0, causal=False, q_offset=None, kv_lens=None, scale=None,
                     out=None, status=None):
    """softmax(scale * q @ k.T) @ v over the keys that each query sees.

    ``q`` is [B, H, Sq, D], ``k`` and ``v`` are [B, H, Sk, D]: FP16 or BF16,
    D <= 128, any strides (for example rows of a longer cache).  Query i stands
    at position p = i + ``q_offset``; by default the last query stands on the
    last key.  It sees key j when ``(j < sinks or p - left <= j <= p + right)
    and (not causal or j <= p)``, with ``window=(left, right)`` and None for no
    bound.  ``kv_lens``: an int32 CUDA tensor [B] with each batch entry's number
    of keys (values are clamped to 0..Sk; whatever the padding behind it holds,
    it does not reach the output).  A query that sees no key gives zeros.
    ``scale`` defaults to D ** -0.5.

    Returns [B, H, Sq, D], or writes ``out``, which shares no memory with an
    input.  The call only queues work on the current stream, and its result
    carries no gradient; ``status`` is as for ``linear``."""
    if not isinstance(window, (tuple, list)) or len(window) != 2:
        raise ValueError("window must be (left, right)")
    key = ("window", _meta(q), _meta(k), _meta(v), *window, *(type(w) for w in window), sinks, type(sinks), bool(causal),
           q_offset, type(q_offset), _meta(kv_lens), scale, _meta(out), _meta(status))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _remember(key, _window_plan(q, k, v, window, sinks, bool(causal), q_offset, kv_lens, scale, out, status))
    if out is not None:
        _check_out(out, q.shape, q, "out", (q, k, v, kv_lens))
    if plan.copy:
        q, k, v, kv_lens = (t.contiguous() if _no_rows(t) else t for t in (q, k, v, kv_lens))
        return window_attention(q, k, v, window=window, sinks=sinks, causal=causal, q_offset=q_offset, kv_lens=kv_lens,
                                scale=scale, out=out, status=status)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _written(out)
    plan.call(q.device, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), kv_lens=_ptr(kv_lens),
              status=_ptr(status))
    return out


def _window_plan(q, k, v, window, sinks, causal, q_offset, kv_lens, scale, out, status):
    """The checks of ``window_attention`` and its arguments without addresses."""
    if any(t.ndim != 4 for t in (q, k, v)):
        raise ValueError("Expected BNSD tensors")
    if q.shape[:2] != k.shape[:2] or k.shape != v.shape or q.shape[3] != k.shape[3]:
        raise ValueError("Incompatible Q/K/V shape; batch, heads and head dimension must match")
    if any(0 in t.shape for t in (q, k, v)):
        raise ValueError("Empty Q/K/V are not supported")
    if any(t.device != q.device or t.dtype != q.dtype for t in (k, v)):
        raise ValueError("Q/K/V must have the same device and dtype")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("window_attention takes FP16 or BF16 inputs")
    b, h, sq, d = q.shape
    if d > 128:
        raise ValueError("window_attention supports head dimensions <= 128")
    left, right = _bound(window[0], "left"), _bound(window[1], "right")
    if sinks is None:
        raise ValueError("sinks must be a non-negative integer")
    first = _bound(sinks, "sinks")
    if q_offset is not None and (isinstance(q_offset, bool) or not isinstance(q_offset, int) or
                                 abs(q_offset) >= 1 << 39):
        raise ValueError("q_offset must be an integer position")
    if kv_lens is not None and (kv_lens.dtype != torch.int32 or tuple(kv_lens.shape) != (b,) or
                                kv_lens.device != q.device):
        raise ValueError("kv_lens must be an int32 tensor [B] on the inputs' device")
    scale = d ** -0.5 if scale is None else scale
    if not isinstance(scale, (int, float)) or not 1e-30 <= scale <= 1e30:
        raise ValueError("scale must be positive and finite, in [1e-30, 1e30]")
    _check_status(status, q.device)
    if out is not None:
        _check_out(out, q.shape, q, "out", (q, k, v, kv_lens))
    _require_b200(q, "window_attention")
    triple = ctypes.c_int64 * 3
    return _Plan(_abi.WindowArgs(
        dtype=_TYPES[q.dtype], batch=b, heads=h, sq=sq, sk=k.shape[2], d=d, q_stride=triple(*q.stride()[:3]),
        k_stride=triple(*k.stride()[:3]), v_stride=triple(*v.stride()[:3]),
        out_stride=triple(*(_packed_strides(q.shape) if out is None else out.stride()[:3])), left=left, right=right,
        sinks=first, causal=int(causal), has_offset=int(q_offset is not None), q_offset=q_offset or 0,
        scale=float(scale)), "vcb_window_attention", tuple(i for i, t in enumerate((q, k, v, kv_lens)) if _no_rows(t)),
        "vcb_window_workspace", ("q", "k", "v"))
