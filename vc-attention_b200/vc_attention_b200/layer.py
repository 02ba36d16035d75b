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
import threading

import torch

from . import _abi

_TYPES = {torch.float32: _abi.VCB_F32, torch.float16: _abi.VCB_F16, torch.bfloat16: _abi.VCB_BF16}
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4}


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


# A call's checks and argument struct depend on its tensors' shapes, strides,
# types and devices and on its options alone.  They are worked out once for each
# such combination; a call then only fills in the addresses.  (Checking anew
# took 20-30 us of host time a call, more than the small calls take on the GPU.)
_PLANS = {}


def _require_b200(t, what):
    from .b200_backend import _require_b200 as check

    check(t, what)


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _remember(key, plan):
    if len(_PLANS) >= 1024:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


# Where calls without a status word of their own leave their flags: a word of
# pinned host memory for each device, which the next such call reads without
# waiting for the device.  A wait that gave up is a fault of the library; its call
# has returned by then, but it does not go unnoticed.
_WORDS = {}
_WORDS_LOCK = threading.Lock()


def _shared_status(device):
    """The address of the device's shared status word.  Raises what an earlier
    call left there, once."""
    word = _WORDS.get(device.index)
    if word is None:
        with _WORDS_LOCK:
            if device.index not in _WORDS:
                held = torch.zeros(1, dtype=torch.int32, device="cpu", pin_memory=True)
                _WORDS[device.index] = held, ctypes.c_int32.from_address(held.data_ptr())
            word = _WORDS[device.index]
    held, flags = word
    if flags.value:
        from .b200_backend import raise_for_flags

        value, flags.value = flags.value, 0
        raise_for_flags(value, f"an earlier linear or window_attention call on {device}, whose output is incomplete")
    return held.data_ptr()


class _Plan:
    """Arguments without addresses (``args``), the scratch bytes for 16-byte
    aligned operands (``need``), the C entry points, and the operands that have
    no contiguous last axis (``copy``)."""

    def __init__(self, args, entry, copy=(), workspace=None, operands=()):
        from .b200_backend import _extension

        lib = _extension()
        self.lib, self.entry, self.copy, self.operands = lib, getattr(lib, entry), copy, operands
        self.workspace = None if workspace is None else getattr(lib, workspace)
        self.cls, self.need = type(args), 0
        if workspace is not None and not copy:
            for name in operands:
                setattr(args, name, 256)
            self.need = self.workspace(ctypes.byref(args))
        self.args = bytes(args)

    def call(self, device, **pointers):
        a = self.cls.from_buffer_copy(self.args)
        for name, value in pointers.items():
            setattr(a, name, value)
        if pointers.get("status", 0) is None:
            a.status = _shared_status(device)
        need = self.need
        if self.workspace is not None and any(pointers[name] & 15 for name in self.operands):
            need = self.workspace(ctypes.byref(a))
        if need:
            scratch = torch.empty(need, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
        stream = torch._C._cuda_getCurrentRawStream(device.index)      # current_stream() makes an object: 3 us
        if torch.cuda.current_device() == device.index:
            rc = self.entry(ctypes.byref(a), stream)
        else:
            with torch.cuda.device(device):
                rc = self.entry(ctypes.byref(a), stream)
        if rc:
            _abi.check(self.lib, rc)


def _no_rows(t):
    return t is not None and t.shape[-1] != 1 and t.stride(-1) != 1


def _strides_differ(a, b):
    """Whether two tensors of one shape step differently.  Axes of length one
    do not step: contiguous() leaves their strides as they are."""
    return any(n > 1 and i != j for n, i, j in zip(a.shape, a.stride(), b.stride()))


def _check_out(out, shape, like, what, inputs, may_be=None):
    """An output the caller gives: shape, type, device, a contiguous last axis,
    no overlap with itself, with ``inputs``, or with a part of ``may_be``: the
    argument that it may be itself.  (By argument and not by object: a tensor
    that is the residual and x too may not be overwritten while x is read.)"""
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{what} must be a {tuple(shape)} tensor of the inputs' dtype and device")
    if out.shape[-1] != 1 and out.stride(-1) != 1:
        raise ValueError(f"{what} must have a contiguous last axis")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and results carry none")
    if _overlaps_itself(out):
        raise ValueError(f"{what} must not overlap itself")
    if may_be is not None and not _same_view(out, may_be):
        inputs = (*inputs, may_be)
    for t in inputs:
        if t is not None and _shares_memory(out, t):
            raise ValueError(f"{what} must not share memory with an input")


def _written(*outs):
    """The library writes by address: autograd has to hear of it, so that a graph
    that saved the tensor does not read the new values in its backward pass."""
    for out in outs:
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)


def _check_status(status, device):
    if status is not None and (status.device != device or status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be a one-element int32 tensor on the inputs' device")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _side_dtype(t, like, what):
    if t.dtype not in (like.dtype, torch.float32) or t.device != like.device:
        raise ValueError(f"{what} must have the inputs' dtype or float32, on their device")
    return _TYPES[t.dtype]


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
    itself and shares memory with no other input.  It does not require a gradient.

    The call only queues work on the current stream, and its result carries no
    gradient.  An expired device wait, which leaves the output incomplete, is
    raised by the next call of this kind on the device (RuntimeError).
    ``status`` takes that over: a caller-owned, zeroed one-element int32 CUDA
    tensor that receives the kernel's flags for
    ``b200_backend.raise_for_status``."""
    key = ("linear", _meta(x), _meta(weight), _meta(bias), activation, _meta(gate), _meta(residual), bool(heads_in),
           heads_out, type(heads_out), _meta(out), _meta(status))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _linear_plan(x, weight, bias, activation, gate, residual, bool(heads_in), heads_out, out, status)
        _remember(key, plan)
    if out is not None:
        _check_out(out, plan.shape, x, "out", (x, weight, bias, gate), may_be=residual)
    if plan.copy:
        x, weight, bias, gate, residual = (t.contiguous() if _no_rows(t) else t
                                           for t in (x, weight, bias, gate, residual))
        return linear(x, weight, bias, activation=activation, gate=gate, residual=residual, heads_in=heads_in,
                      heads_out=heads_out, out=out, status=status)
    if out is None:
        out = x.new_empty(plan.shape)
    else:
        _written(out)
    plan.call(x.device, x=x.data_ptr(), w=weight.data_ptr(), y=out.data_ptr(), bias=_ptr(bias), gate=_ptr(gate),
              residual=_ptr(residual), status=_ptr(status))
    return out


def _linear_plan(x, weight, bias, activation, gate, residual, heads_in, heads_out, out, status):
    """The checks of ``linear`` and its arguments without addresses."""
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
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias must be [{n}]")
    bias_dtype = 0 if bias is None else _side_dtype(bias, x, "bias")
    gate_dtype = 0
    if gate is not None:
        gate_dtype = _side_dtype(gate, x, "gate")
        if gate.ndim < 1 or gate.ndim > len(shape) or gate.shape[-1] != n or any(
                g not in (1, full) for g, full in zip(reversed(gate.shape), reversed(shape))):
            raise ValueError(f"gate must broadcast against {shape} with its last axis of {n}")
    if residual is not None and (tuple(residual.shape) != shape or residual.dtype != x.dtype or
                                 residual.device != x.device):
        raise ValueError("residual must have the result's shape, dtype and device")
    _check_status(status, x.device)
    if out is not None:
        _check_out(out, shape, x, "out", (x, weight, bias, gate), may_be=residual)
    _require_b200(x, "linear")
    copy = tuple(i for i, t in enumerate((x, weight, bias, gate, residual)) if _no_rows(t))
    if heads_in:
        xs = x.stride()[:3]
    else:
        xs = (x.stride(0) if x.ndim == 3 else 0, 0, x.stride(-2))
    n_head = n if heads_out is None else n // heads_out
    if heads_out is not None:
        ys = (heads_out * s * n_head, s * n_head, n_head) if out is None else out.stride()[:3]
    elif out is None:
        ys = (s * n, 0, n)
    else:
        ys = (out.stride(0) if out.ndim == 3 else 0, 0, out.stride(-2))
    gs = gate.expand(b, s, n).stride() if gate is not None else (0, 0)
    rs = (0, 0) if residual is None else (residual.stride(0) if residual.ndim == 3 else 0, residual.stride(-2))
    plan = _Plan(_abi.LinearArgs(
        dtype=_TYPES[x.dtype], batch=b, tokens=s, n=n, heads_in=hi, k_head=kh, x_stride_b=xs[0], x_stride_h=xs[1],
        x_stride_s=xs[2], w_stride=weight.stride(0) if n > 1 else k, bias_dtype=bias_dtype,
        activation=ACTIVATIONS[activation], gate_dtype=gate_dtype, gate_stride_b=gs[0], gate_stride_s=gs[1],
        residual_stride_b=rs[0], residual_stride_s=rs[1], n_head=n_head, y_stride_b=ys[0], y_stride_h=ys[1],
        y_stride_s=ys[2]), "vcb_linear", copy, "vcb_linear_workspace", ("x", "w"))
    plan.shape = shape
    return plan


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
    k_out)``, for example rows of a K buffer; q_out may be ``q`` itself and
    k_out ``k``, and neither shares memory with another argument.  The call
    only queues work on the current stream, and its results carry no
    gradient."""
    if out is None:
        outs = None
    else:
        if len(out) != 2:
            raise ValueError("out must be (q_out, k_out)")
        outs = _meta(out[0]), _meta(out[1])
    key = ("rope", _meta(q), _meta(k), _meta(q_weight), _meta(k_weight), _meta(cos), _meta(sin), eps, bool(interleaved),
           outs)
    plan = _PLANS.get(key)
    if plan is None:
        plan = _remember(key, _rope_plan(q, k, q_weight, k_weight, cos, sin, eps, bool(interleaved), out))
    if out is not None:
        _check_rope_out(out, q, k, q_weight, k_weight, cos, sin)
    if plan.copy:
        if cos is not None and _strides_differ(cos, sin):
            cos, sin = cos.contiguous(), sin.contiguous()
        q, k, q_weight, k_weight, cos, sin = (t.contiguous() if _no_rows(t) else t
                                              for t in (q, k, q_weight, k_weight, cos, sin))
        return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps=eps, interleaved=interleaved, out=out)
    if out is None:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        qo, ko = out
        _written(qo, ko)
    plan.call(q.device, q=q.data_ptr(), k=k.data_ptr(), q_out=qo.data_ptr(), k_out=ko.data_ptr(),
              q_weight=_ptr(q_weight), k_weight=_ptr(k_weight), cos=_ptr(cos), sin=_ptr(sin))
    return qo, ko


def _check_rope_out(out, q, k, *others):
    _check_out(out[0], q.shape, q, "q_out", (k, *others), may_be=q)
    _check_out(out[1], k.shape, k, "k_out", (q, *others), may_be=k)
    if _shares_memory(out[0], out[1]):
        raise ValueError("q_out and k_out must not share memory")


def _packed_strides(shape):
    return tuple(math.prod(shape[i + 1:]) for i in range(3))


def _rope_plan(q, k, q_weight, k_weight, cos, sin, eps, interleaved, out):
    """The checks of ``qk_norm_rope`` and its arguments without addresses."""
    for name, t in (("q", q), ("k", k)):
        if t.ndim != 4 or 0 in t.shape:
            raise ValueError(f"{name} must be a nonempty [B, H, S, D] tensor")
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError("q and k must match in batch, tokens and head dimension")
    if q.dtype != k.dtype or q.device != k.device or q.dtype not in _TYPES:
        raise ValueError("q and k must share a device and an FP32/FP16/BF16 dtype")
    b, h, s, d = q.shape
    if d > 128:
        raise ValueError("qk_norm_rope supports head dimensions <= 128")
    if eps is not None and not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
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
    ts = (0, 0)
    copy = tuple(i for i, t in enumerate((q, k, q_weight, k_weight, cos, sin)) if _no_rows(t))
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
        if _strides_differ(cos, sin):
            copy = (*copy, 4, 5)
        ts = (cos.stride(0) if cos.ndim == 3 and cos.shape[0] > 1 else 0, cos.stride(-2))
    if out is not None:
        _check_rope_out(out, q, k, q_weight, k_weight, cos, sin)
    _require_b200(q, "qk_norm_rope")
    qs, ks = (_packed_strides(t.shape) if out is None else o.stride()[:3]
              for t, o in ((q, out and out[0]), (k, out and out[1])))
    triple = ctypes.c_int64 * 3
    return _Plan(_abi.QKNormRopeArgs(
        dtype=_TYPES[q.dtype], batch=b, q_heads=h, k_heads=k.shape[1], tokens=s, d=d, q_stride=triple(*q.stride()[:3]),
        k_stride=triple(*k.stride()[:3]), q_out_stride=triple(*qs), k_out_stride=triple(*ks),
        weight_dtype=_TYPES[weights[0].dtype] if weights else 0, rows=rows, rotary=rotary, table_stride_b=ts[0],
        table_stride_s=ts[1], interleaved=int(interleaved), norm=int(eps is not None),
        eps=0.0 if eps is None else float(eps)), "vcb_qk_norm_rope", copy)
