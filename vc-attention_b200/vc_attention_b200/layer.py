"""The operators around the attention call: projections and the norm and
rotation of queries and keys.

The reference receives post-RoPE Q/K/V from the model (core.py:243-262); these
operators make them, and consume the attention's output, on the same terms as
the rest of the package: hand-written sm_100a kernels behind the C ABI, work
queued on the current stream, no CPU fallback, ValueError for arguments that
do not fit, and no gradients (the results carry no graph)."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _abi
from .b200_backend import _DTYPES, _extension, _require_b200, _stream

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4}


def _rows(x):
    """``x`` with a contiguous last axis (a copy only when it has none)."""
    return x if x.shape[-1] == 1 or x.stride(-1) == 1 else x.contiguous()


def _interval(t):
    """First and one-past-last byte address that ``t`` can touch."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlaps_itself(t):
    """Whether two indices of ``t`` may be one address (outputs must not)."""
    span = 0
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda a: a[1]):
        if s <= span:
            return True
        span += (n - 1) * s
    return False


def _shares_memory(a, b):
    """Whether ``a`` and ``b`` may have an element in common.  Exact for two
    views of one shape and strides (such as the Q and K parts of a fused
    projection); otherwise their address ranges decide."""
    a0, a1 = _interval(a)
    b0, b1 = _interval(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.stride() != b.stride() or a.shape != b.shape or a.dtype != b.dtype or (b0 - a0) % a.element_size():
        return True
    axes = sorted(((s, n) for n, s in zip(a.shape, a.stride()) if n > 1), reverse=True)
    spans = [sum((n - 1) * s for s, n in axes[i + 1:]) for i in range(len(axes))]

    def reach(delta, i):
        # is delta a sum of d_i * stride_i with |d_i| < n_i?
        if i == len(axes):
            return delta == 0
        s, n = axes[i]
        if s == 0:
            return reach(delta, i + 1)
        near = delta // s
        return any(abs(d) < n and abs(delta - d * s) <= spans[i] and reach(delta - d * s, i + 1)
                   for d in range(near - spans[i] // s - 1, near + spans[i] // s + 3))

    return reach((b0 - a0) // a.element_size(), 0)


def _same_view(a, b):
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype


def _check_out(out, shape, like, what, inputs, may_be=None):
    """An output the caller gives: shape, type, device, a contiguous last axis,
    no overlap with itself or with an input other than ``may_be`` itself."""
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{what} must be a {tuple(shape)} tensor of the inputs' dtype and device")
    if out.shape[-1] != 1 and out.stride(-1) != 1:
        raise ValueError(f"{what} must have a contiguous last axis")
    if _overlaps_itself(out):
        raise ValueError(f"{what} must not overlap itself")
    for t in inputs:
        if t is None or (may_be is not None and t is may_be and _same_view(out, t)):
            continue
        if _shares_memory(out, t):
            raise ValueError(f"{what} must not share memory with an input")


def _check_status(status, device):
    if status is not None and (status.device != device or status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be a one-element int32 tensor on the inputs' device")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _side_dtype(t, like, what):
    if t.dtype not in (like.dtype, torch.float32) or t.device != like.device:
        raise ValueError(f"{what} must have the inputs' dtype or float32, on their device")
    return _DTYPES[t.dtype]


@torch.no_grad()
def linear(x, weight, bias=None, *, activation=None, gate=None, residual=None, heads_in=False, heads_out=None,
           out=None, status=None):
    """``residual + gate * act(x @ weight.T + bias)`` in one kernel.

    ``x`` is [B, S, K] or [S, K], or with ``heads_in`` the attention's output
    [B, H, S, D] with K = H * D (no transposed copy is made).  ``weight`` is
    [N, K].  FP16 or BF16; products are summed in FP32 and the result is
    rounded once.  ``bias`` [N] and ``gate`` (broadcast against [B, S, N], for
    example [B, 1, N] for one vector per batch entry) may be FP32.
    ``activation``: None, "silu", "gelu" (erf), "gelu_tanh" or "relu".
    ``residual`` has the result's shape and dtype.

    Returns [B, S, N] (or [S, N]), or with ``heads_out=H`` the attention's
    input layout [B, H, S, N / H], without gate or residual.  ``out`` may be
    given, with any strides but a contiguous last axis; it may be ``residual``
    itself and shares memory with no other input.

    The call only queues work on the current stream.  ``status``: a
    caller-owned, zeroed one-element int32 CUDA tensor that receives the
    kernel's flags for ``b200_backend.raise_for_status`` (an expired device
    wait)."""
    if activation not in ACTIVATIONS:
        raise ValueError('activation must be None, "silu", "gelu", "gelu_tanh" or "relu"')
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("linear takes FP16 or BF16 inputs")
    if heads_in and x.ndim != 4:
        raise ValueError("heads_in expects x as [B, H, S, D]")
    if not heads_in and x.ndim not in (2, 3):
        raise ValueError("linear expects x as [S, K] or [B, S, K]")
    if 0 in x.shape or weight.ndim != 2 or 0 in weight.shape:
        raise ValueError("linear expects a nonempty x and a nonempty weight [N, K]")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError("x and weight must have the same device and dtype")
    n, k = weight.shape
    if heads_in:
        b, hi, s, kh = x.shape
    else:
        b, hi, s, kh = (x.shape[0] if x.ndim == 3 else 1), 1, x.shape[-2], x.shape[-1]
    if hi * kh != k:
        raise ValueError(f"x has {hi * kh} features, weight takes {k}")
    lead = (s,) if x.ndim == 2 else (b, s)
    if heads_out is not None:
        if isinstance(heads_out, bool) or not isinstance(heads_out, int) or heads_out < 1 or n % heads_out:
            raise ValueError("heads_out must be a positive integer that divides the output features")
        if gate is not None or residual is not None:
            raise ValueError("gate and residual need the token-major output")
        if x.ndim == 2:
            raise ValueError("heads_out expects a batch axis")
        shape = (b, heads_out, s, n // heads_out)
    else:
        shape = (*lead, n)
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be [{n}]")
        bias_dtype = _side_dtype(bias, x, "bias")
        bias = bias.contiguous()
    if gate is not None:
        gate_dtype = _side_dtype(gate, x, "gate")
        if gate.ndim < 1 or gate.ndim > len(shape) or gate.shape[-1] != n or any(
                g not in (1, full) for g, full in zip(reversed(gate.shape), reversed(shape))):
            raise ValueError(f"gate must broadcast against {shape} with its last axis of {n}")
        gate = _rows(gate).expand(b, s, n)
    if residual is not None and (tuple(residual.shape) != shape or residual.dtype != x.dtype or
                                 residual.device != x.device):
        raise ValueError("residual must have the result's shape, dtype and device")
    _check_status(status, x.device)
    if out is not None:
        _check_out(out, shape, x, "out", (x, weight, bias, gate, residual), may_be=residual)
    _require_b200(x, "linear")
    lib = _extension()
    x, weight = _rows(x), _rows(weight)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    res = None if residual is None else _rows(residual)
    if heads_in:
        xs = (x.stride(0), x.stride(1), x.stride(2))
    else:
        xs = (x.stride(0) if x.ndim == 3 else 0, 0, x.stride(-2))
    if heads_out is not None:
        n_head, ys = n // heads_out, out.stride()[:3]
    else:
        n_head, ys = n, (out.stride(0) if out.ndim == 3 else 0, 0, out.stride(-2))
    a = _abi.LinearArgs(
        x=x.data_ptr(), w=weight.data_ptr(), dtype=_DTYPES[x.dtype], batch=b, tokens=s, n=n, heads_in=hi, k_head=kh,
        x_stride_b=xs[0], x_stride_h=xs[1], x_stride_s=xs[2], w_stride=weight.stride(0) if n > 1 else k,
        activation=ACTIVATIONS[activation], y=out.data_ptr(), n_head=n_head, y_stride_b=ys[0], y_stride_h=ys[1],
        y_stride_s=ys[2], status=_ptr(status))
    if bias is not None:
        a.bias, a.bias_dtype = bias.data_ptr(), bias_dtype
    if gate is not None:
        a.gate, a.gate_dtype, a.gate_stride_b, a.gate_stride_s = gate.data_ptr(), gate_dtype, *gate.stride()[:2]
    if res is not None:
        a.residual = res.data_ptr()
        a.residual_stride_b, a.residual_stride_s = (res.stride(0) if res.ndim == 3 else 0), res.stride(-2)
    need = lib.vcb_linear_workspace(ctypes.byref(a))
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    with torch.cuda.device(x.device):
        _abi.check(lib, lib.vcb_linear(ctypes.byref(a), _stream(x.device)))
    return out


@torch.no_grad()
def qk_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None, *, eps=1e-6, interleaved=True, out=None):
    """RMS norm of each head's row of Q and K and the position rotation, in
    one pass: ``n = x / sqrt(mean(x^2) + eps) * weight`` over the head's
    channels, then ``(a, b) -> (a cos - b sin, a sin + b cos)``.

    ``q`` [B, H, S, D] and ``k`` [B, Hk, S, D] (FP32, FP16 or BF16, D <= 128)
    may be views with any strides, for example
    ``qkv.view(B, S, 3, H, D)[:, :, 0].transpose(1, 2)`` of a fused
    projection.  Weights are [D] in the inputs' dtype or FP32; None stands for
    ones.  ``eps=None`` leaves the norm out.  ``cos`` and ``sin`` are FP32
    tables [R, r / 2] or [B, R, r / 2]: the first r channels are rotated, in
    pairs (2i, 2i + 1), or (i, i + r / 2) with ``interleaved=False``; row t
    belongs to token t, and tokens from R on (text behind a video, padding)
    are not rotated.  Arithmetic is FP32 with one rounding at the end.

    Returns (q, k) as contiguous BNSD tensors, or writes ``out=(q_out,
    k_out)``, for example rows of a K buffer; an output may be its own
    input."""
    for name, t in (("q", q), ("k", k)):
        if t.ndim != 4 or 0 in t.shape:
            raise ValueError(f"{name} must be a nonempty [B, H, S, D] tensor")
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError("q and k must match in batch, tokens and head dimension")
    if q.dtype != k.dtype or q.device != k.device or q.dtype not in _DTYPES:
        raise ValueError("q and k must share a device and an FP32/FP16/BF16 dtype")
    b, h, s, d = q.shape
    if d > 128:
        raise ValueError("qk_norm_rope supports head dimensions <= 128")
    if eps is not None and not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative, or None")
    weights = [t for t in (q_weight, k_weight) if t is not None]
    for t in weights:
        if tuple(t.shape) != (d,):
            raise ValueError(f"weights must be [{d}]")
        _side_dtype(t, q, "weights")
    if len({t.dtype for t in weights}) > 1:
        raise ValueError("q_weight and k_weight must share a dtype")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    rows = rotary = 0
    if cos is not None:
        if cos.shape != sin.shape or cos.ndim not in (2, 3) or 0 in cos.shape:
            raise ValueError("cos and sin must be nonempty [R, r / 2] or [B, R, r / 2] tables of one shape")
        if any(t.dtype != torch.float32 or t.device != q.device for t in (cos, sin)):
            raise ValueError("cos and sin must be float32 on the inputs' device")
        rows, rotary = cos.shape[-2], 2 * cos.shape[-1]
        if rows > s:
            raise ValueError("the tables have more rows than there are tokens: slice the tokens' rows")
        if rotary > d:
            raise ValueError("the tables rotate more channels than a head has")
        if cos.ndim == 3 and cos.shape[0] not in (1, b):
            raise ValueError("batched tables need one entry, or one for each batch entry")
        cos, sin = _rows(cos), _rows(sin)
        if cos.stride() != sin.stride():
            cos, sin = cos.contiguous(), sin.contiguous()
    if out is not None:
        if len(out) != 2:
            raise ValueError("out must be (q_out, k_out)")
        others = (q_weight, k_weight, cos, sin)
        _check_out(out[0], q.shape, q, "q_out", (q, k, *others), may_be=q)
        _check_out(out[1], k.shape, k, "k_out", (k, q, *others), may_be=k)
        if _shares_memory(out[0], out[1]):
            raise ValueError("q_out and k_out must not share memory")
    _require_b200(q, "qk_norm_rope")
    lib = _extension()
    q, k = _rows(q), _rows(k)
    qo, ko = out if out is not None else (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    q_weight, k_weight = (None if t is None else t.contiguous() for t in (q_weight, k_weight))
    triple = ctypes.c_int64 * 3
    a = _abi.QKNormRopeArgs(
        q=q.data_ptr(), k=k.data_ptr(), q_out=qo.data_ptr(), k_out=ko.data_ptr(), dtype=_DTYPES[q.dtype], batch=b,
        q_heads=h, k_heads=k.shape[1], tokens=s, d=d, q_stride=triple(*q.stride()[:3]),
        k_stride=triple(*k.stride()[:3]), q_out_stride=triple(*qo.stride()[:3]),
        k_out_stride=triple(*ko.stride()[:3]), q_weight=_ptr(q_weight), k_weight=_ptr(k_weight),
        weight_dtype=_DTYPES[weights[0].dtype] if weights else 0, rows=rows, rotary=rotary,
        interleaved=int(bool(interleaved)), norm=int(eps is not None), eps=0.0 if eps is None else float(eps))
    if cos is not None:
        a.cos, a.sin, a.table_stride_s = cos.data_ptr(), sin.data_ptr(), cos.stride(-2)
        a.table_stride_b = cos.stride(0) if cos.ndim == 3 and cos.shape[0] > 1 else 0
    with torch.cuda.device(q.device):
        _abi.check(lib, lib.vcb_qk_norm_rope(ctypes.byref(a), _stream(q.device)))
    return qo, ko
