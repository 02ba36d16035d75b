"""Arguments that the layer operators refuse, before they touch a device."""
import ctypes

import pytest
import torch

from vc_attention_b200 import _abi, layer, linear, qk_norm_rope, window_attention
from vc_attention_b200.layer import _overlaps_itself, _shares_memory

BF16 = torch.bfloat16


def _t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,match", [
    ((_t(2, 3, 8), _t(4, 8)), dict(activation="tanh"), "activation"),
    ((_t(2, 3, 8, dtype=torch.float32), _t(4, 8, dtype=torch.float32)), {}, "FP16 or BF16"),
    ((_t(2, 3, 8), _t(4, 8, dtype=torch.float16)), {}, "dtype"),
    ((_t(8), _t(4, 8)), {}, r"\[S, K\]"),
    ((_t(2, 3, 8), _t(4, 8)), dict(heads_in=True), "heads_in"),
    ((_t(2, 0, 8), _t(4, 8)), {}, "nonempty"),
    ((_t(2, 3, 8), _t(0, 8)), {}, "nonempty"),
    ((_t(2, 3, 8), _t(4, 9)), {}, "features"),
    ((_t(2, 2, 3, 4), _t(4, 9)), dict(heads_in=True), "features"),
    ((_t(2, 3, 8), _t(4, 8), _t(5)), {}, "bias"),
    ((_t(2, 3, 8), _t(4, 8), _t(4, dtype=torch.float16)), {}, "bias"),
    ((_t(2, 3, 8), _t(4, 8)), dict(heads_out=3), "heads_out"),
    ((_t(2, 3, 8), _t(4, 8)), dict(heads_out=True), "heads_out"),
    ((_t(3, 8), _t(4, 8)), dict(heads_out=2), "batch axis"),
    ((_t(2, 3, 8), _t(4, 8)), dict(heads_out=2, residual=_t(2, 3, 4)), "token-major"),
    ((_t(2, 3, 8), _t(4, 8)), dict(gate=_t(2, 4)), "gate"),
    ((_t(2, 3, 8), _t(4, 8)), dict(gate=_t(2, 1, 1)), "gate"),
    ((_t(2, 3, 8), _t(4, 8)), dict(residual=_t(3, 4)), "residual"),
    ((_t(2, 3, 8), _t(4, 8)), dict(out=_t(2, 3, 5)), "out must be"),
    ((_t(2, 3, 8), _t(4, 8)), dict(out=_t(1, 3, 4).expand(2, 3, 4)), "overlap itself"),
    ((_t(2, 3, 8), _t(4, 8)), dict(out=_t(2, 4, 3).transpose(1, 2)), "contiguous last axis"),
    ((_t(2, 3, 8), _t(4, 8)), dict(status=_t(1)), "status"),
    ((_t(2, 3, 8), _t(4, 8)), {}, "no CPU fallback"),
])
def test_linear_refuses(args, kw, match):
    with pytest.raises(ValueError, match=match):
        linear(*args, **kw)


def test_linear_refuses_an_output_over_an_input():
    x, w = _t(2, 3, 8), _t(8, 8)
    with pytest.raises(ValueError, match="share memory"):
        linear(x, w, out=x)
    res = _t(2, 4, 8)
    with pytest.raises(ValueError, match="share memory"):
        linear(x, w, residual=res[:, :3], out=res[:, 1:])
    with pytest.raises(ValueError, match="no CPU fallback"):      # in place on the residual is allowed
        linear(x, w, residual=res[:, :3], out=res[:, :3])


Q = _t(2, 4, 6, 16)
TAB = _t(6, 8, dtype=torch.float32)


@pytest.mark.parametrize("args,kw,match", [
    ((_t(4, 6, 16), Q), {}, "q must be"),
    ((Q, _t(2, 4, 0, 16)), {}, "k must be"),
    ((Q, _t(2, 4, 5, 16)), {}, "match"),
    ((Q, _t(2, 4, 6, 16, dtype=torch.float16)), {}, "dtype"),
    ((_t(1, 1, 2, 130), _t(1, 1, 2, 130)), {}, "<= 128"),
    ((Q, Q), dict(eps=-1.0), "eps"),
    ((Q, Q), dict(eps=float("nan")), "eps"),
    ((Q, Q), dict(eps=torch.tensor(1e-6)), "eps"),
    ((Q, Q, _t(15)), {}, "weights"),
    ((Q, Q, _t(16, dtype=torch.float16)), {}, "weights"),
    ((Q, Q, _t(16), _t(16, dtype=torch.float32)), {}, "share a dtype"),
    ((Q, Q), dict(cos=TAB), "come together"),
    ((Q, Q, None, None, TAB, _t(6, 7, dtype=torch.float32)), {}, "one shape"),
    ((Q, Q, None, None, TAB.double(), TAB.double()), {}, "float32"),
    ((Q, Q, None, None, _t(7, 8, dtype=torch.float32), _t(7, 8, dtype=torch.float32)), {}, "more rows"),
    ((Q, Q, None, None, _t(6, 9, dtype=torch.float32), _t(6, 9, dtype=torch.float32)), {}, "more channels"),
    ((Q, Q, None, None, TAB.expand(3, 6, 8), TAB.expand(3, 6, 8)), {}, "batch"),
    ((Q, Q), dict(out=(Q,)), "out must be"),
    ((Q, Q), dict(out=(_t(2, 4, 6, 15), _t(2, 4, 6, 16))), "q_out"),
    ((Q, Q), {}, "no CPU fallback"),
])
def test_rope_refuses(args, kw, match):
    with pytest.raises(ValueError, match=match):
        qk_norm_rope(*args, **kw)


def test_rope_outputs_and_inputs_in_one_buffer():
    qkv = _t(2, 6, 3, 4, 16)
    q, k = (qkv[:, :, i].transpose(1, 2) for i in range(2))
    with pytest.raises(ValueError, match="no CPU fallback"):      # the parts of a fused projection, in place
        qk_norm_rope(q, k, out=(q, k))
    with pytest.raises(ValueError, match="share memory"):
        qk_norm_rope(q, k, out=(k, q))
    with pytest.raises(ValueError, match="share memory"):
        qk_norm_rope(q, q, out=(q, q))


def test_shares_memory_is_exact_for_equal_strides():
    base = torch.zeros(4, 6, 8)
    assert not _shares_memory(base[:, :3], base[:, 3:])
    assert _shares_memory(base[:, :3], base[:, 2:5])
    assert not _shares_memory(base[..., :4], base[..., 4:])
    assert _shares_memory(base[..., :4], base[..., 3:7])
    assert not _shares_memory(base[0::2], base[1::2])
    assert _shares_memory(base[:, :3], base.transpose(0, 1)[:4, :3])      # unequal strides: by address range
    assert _overlaps_itself(base[:1].expand(2, 6, 8)) and not _overlaps_itself(base.transpose(0, 2))


def test_c_entries_refuse_without_a_device():
    lib = _abi.load()
    assert lib.vcb_linear(None, None) == _abi.VCB_ERR_INVALID_ARGUMENT
    assert lib.vcb_linear_workspace(None) == 0
    assert lib.vcb_qk_norm_rope(None, None) == _abi.VCB_ERR_INVALID_ARGUMENT
    a = _abi.LinearArgs(x=16, w=16, y=16, dtype=2, batch=1, tokens=4, n=8, heads_in=1, k_head=9, x_stride_s=9,
                        w_stride=9, n_head=8)
    need = lib.vcb_linear_workspace(ctypes.byref(a))
    assert need >= (4 + 8) * 16 * 2                       # both operands packed to 16 channels
    assert lib.vcb_linear(ctypes.byref(a), None) == _abi.VCB_ERR_INVALID_ARGUMENT
    assert "workspace" in _abi.last_error(lib)
    a.workspace, a.workspace_bytes = 256, need - 1
    assert lib.vcb_linear(ctypes.byref(a), None) == _abi.VCB_ERR_WORKSPACE
    for field, value, match in [("dtype", 0, "dtype"), ("n_head", 3, "n_head"), ("activation", 9, "activation"),
                                ("tokens", 0, "positive"), ("w_stride", 8, "overlap"), ("tokens", 1 << 31, "int32")]:
        keep = getattr(a, field)
        setattr(a, field, value)
        assert lib.vcb_linear(ctypes.byref(a), None) == _abi.VCB_ERR_INVALID_ARGUMENT
        assert match in _abi.last_error(lib)
        setattr(a, field, keep)
    r = _abi.QKNormRopeArgs(q=16, k=16, q_out=16, k_out=16, dtype=2, batch=1, q_heads=1, k_heads=1, tokens=4, d=8,
                            rows=4, rotary=8, norm=1, eps=1e-6, cos=16, sin=16)
    for field, value, match in [("d", 129, "128"), ("rotary", 7, "rotary"), ("rows", 5, "rows"), ("eps", -1.0, "eps"),
                                ("tokens", 1 << 31, "int32"), ("sin", None, "cos")]:
        keep = getattr(r, field)
        setattr(r, field, value)
        assert lib.vcb_qk_norm_rope(ctypes.byref(r), None) == _abi.VCB_ERR_INVALID_ARGUMENT
        assert match in _abi.last_error(lib)
        setattr(r, field, keep)


W = _t(2, 3, 5, 16)


@pytest.mark.parametrize("args,kw,match", [
    ((_t(3, 5, 16), W, W), {}, "BNSD"),
    ((W, _t(2, 4, 5, 16), _t(2, 4, 5, 16)), {}, "Incompatible"),
    ((W, W, _t(2, 3, 6, 16)), {}, "Incompatible"),
    ((W, _t(2, 3, 5, 8), _t(2, 3, 5, 8)), {}, "Incompatible"),
    ((_t(2, 3, 0, 16), W, W), {}, "Empty"),
    ((W, W, W.half()), {}, "dtype"),
    ((W.float(), W.float(), W.float()), {}, "FP16 or BF16"),
    ((_t(1, 1, 2, 129), _t(1, 1, 2, 129), _t(1, 1, 2, 129)), {}, "<= 128"),
    ((W, W, W), dict(window=(1, 2, 3)), "window"),
    ((W, W, W), dict(window=(-1, 0)), "left"),
    ((W, W, W), dict(window=(1, 1.5)), "right"),
    ((W, W, W), dict(sinks=-1), "sinks"),
    ((W, W, W), dict(sinks=None), "sinks"),
    ((W, W, W), dict(q_offset=1.0), "q_offset"),
    ((W, W, W), dict(kv_lens=torch.zeros(2, dtype=torch.int64)), "kv_lens"),
    ((W, W, W), dict(kv_lens=torch.zeros(3, dtype=torch.int32)), "kv_lens"),
    ((W, W, W), dict(scale=0.0), "scale"),
    ((W, W, W), dict(scale=float("inf")), "scale"),
    ((W, W, W), dict(scale=torch.tensor(0.5)), "scale"),
    ((W, W, W), dict(window=None), "window"),
    ((W, W, W), dict(out=W), "share memory"),
    ((W, W, W), dict(status=_t(2, dtype=torch.int32)), "status"),
    ((W, W, W), {}, "no CPU fallback"),
])
def test_window_refuses(args, kw, match):
    with pytest.raises(ValueError, match=match):
        window_attention(*args, **kw)


def test_window_c_entry_refuses_without_a_device():
    lib = _abi.load()
    assert lib.vcb_window_attention(None, None) == _abi.VCB_ERR_INVALID_ARGUMENT
    a = _abi.WindowArgs(q=16, k=16, v=16, out=16, dtype=2, batch=1, heads=1, sq=4, sk=4, d=16, left=-1, right=-1,
                        scale=1.0)
    for field, value, match in [("dtype", 0, "dtype"), ("d", 200, "128"), ("left", -2, "window"), ("sinks", -1, "sinks"),
                                ("scale", -1.0, "scale"), ("sk", 1 << 31, "int32"), ("heads", 70000, "int32"),
                                ("out", None, "non-null")]:
        keep = getattr(a, field)
        setattr(a, field, value)
        assert lib.vcb_window_attention(ctypes.byref(a), None) == _abi.VCB_ERR_INVALID_ARGUMENT
        assert match in _abi.last_error(lib)
        setattr(a, field, keep)


def test_tables_of_one_row_from_two_caches_are_not_copied_forever(monkeypatch):
    """One token's rows of tables with different row strides: contiguous()
    returns them unchanged, so they must not count as different."""
    calls = []

    class Plan:
        def __init__(self, args, entry, copy=(), *rest):
            self.copy = copy

        def call(self, device, **pointers):
            calls.append(self.copy)

    monkeypatch.setattr(layer, "_require_b200", lambda t, what: None)
    monkeypatch.setattr(layer, "_Plan", Plan)
    monkeypatch.setattr(layer, "_PLANS", {})
    q = torch.randn(1, 2, 1, 16)
    cos, sin = torch.randn(5, 8)[2:3], torch.randn(5, 16)[2:3, :8]
    assert cos.stride() != sin.stride()
    layer.qk_norm_rope(q, q, cos=cos, sin=sin)
    layer.qk_norm_rope(q, q, cos=cos[None], sin=sin[None].expand(1, 1, 8))
    assert calls == [(), ()]
    q = torch.randn(1, 2, 5, 16)
    layer.qk_norm_rope(q, q, cos=torch.randn(5, 8), sin=torch.randn(5, 16)[:, :8])     # these do differ: copied once
    assert calls == [(), (), ()]


class _NoKernel:
    """Stands in for a call's plan: no library, no device."""

    def __init__(self, args, entry, copy=(), *rest):
        self.args, self.entry, self.copy = args, entry, copy

    def call(self, device, **pointers):
        pass


@pytest.fixture
def on_cpu(monkeypatch):
    """Calls run through their checks and stop before the library."""
    from vc_attention_b200 import window
    for module in (layer, window):
        monkeypatch.setattr(module, "_require_b200", lambda t, what: None)
        monkeypatch.setattr(module, "_Plan", _NoKernel)
    monkeypatch.setattr(layer, "_PLANS", plans := {})
    monkeypatch.setattr(window, "_PLANS", plans)


def test_an_output_may_be_one_argument_only(on_cpu):
    """The tensor that an output may overwrite (the residual; Q for q_out, K for
    k_out) is not exempt where it is another argument too: the products still
    read it while the output is written."""
    x, w = _t(2, 3, 8), _t(8, 8)
    for _ in range(2):                          # the second time the shapes are known
        assert linear(x, w, residual=x).shape == x.shape
        held = _t(2, 3, 8)
        assert linear(x, w, residual=held, out=held) is held
        for kw in (dict(residual=x, out=x), dict(residual=held, gate=held, out=held)):
            with pytest.raises(ValueError, match="share memory"):
                linear(x, w, **kw)
    square = _t(8, 8)
    for _ in range(2):
        with pytest.raises(ValueError, match="share memory"):
            linear(_t(8, 8), square, residual=square, out=square)
    q, k, other = _t(2, 4, 6, 16), _t(2, 4, 6, 16), _t(2, 4, 6, 16)
    for _ in range(2):
        assert qk_norm_rope(q, k, out=(q, k)) == (q, k)
        assert qk_norm_rope(q, q, out=(k, other)) == (k, other)
        for out in ((q, other), (other, q)):
            with pytest.raises(ValueError, match="share memory"):
                qk_norm_rope(q, q, out=out)
    row = _t(1, 1, 1, 16)
    with pytest.raises(ValueError, match="share memory"):
        qk_norm_rope(row, _t(1, 1, 1, 16), row[0, 0, 0], out=(row, _t(1, 1, 1, 16)))


def test_window_bounds_are_wider_than_any_position(on_cpu):
    """The widest bounds are passed on as ones that no position reaches, inside
    what the C entry takes."""
    from vc_attention_b200 import window
    q, far = _t(1, 1, 7, 16), 2 ** 39 - 1
    for offset in (far, -far):
        plan = window._window_plan(q, q, q, (2 ** 70, 2 ** 45), 2 ** 50, False, offset, None, None, None, None)
        for bound in (plan.args.left, plan.args.right, plan.args.sinks):
            assert far + 2 ** 31 < bound < 1 << 40


def test_products_too_large_to_be_cut_are_not():
    """73 row tiles of 2^25 chunks: more units of a cut than its 32-bit counters
    hold, so the tiles are walked whole and need no scratch."""
    lib = _abi.load()
    k = 2 ** 31 - 512
    a = _abi.LinearArgs(x=256, w=256, y=256, dtype=2, batch=73, tokens=17, n=32, heads_in=1, k_head=k, x_stride_b=16,
                        x_stride_h=8, x_stride_s=8, w_stride=k, n_head=32)
    assert lib.vcb_linear_workspace(ctypes.byref(a)) == 0
    a.k_head = a.w_stride = 2 ** 24
    assert lib.vcb_linear_workspace(ctypes.byref(a)) > 0      # the same tiles, cut


def test_outputs_written_in_place_are_known_to_autograd(on_cpu):
    """A tensor that a graph has saved may not change unnoticed, and one that
    requires a gradient is no output, as for torch's own out= functions."""
    x, w = _t(2, 3, 8), _t(8, 8)
    q, k = _t(2, 4, 6, 16), _t(2, 4, 6, 16)
    outs = [_t(2, 3, 8), _t(2, 4, 6, 16), _t(2, 4, 6, 16), _t(2, 4, 6, 16)]

    def write():
        linear(x, w, out=outs[0])
        qk_norm_rope(q, k, out=(outs[1], outs[2]))
        window_attention(q, k, q, out=outs[3])

    leaf = torch.ones(1, requires_grad=True)
    losses = [(leaf * o).sum() for o in outs]
    write()
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        outs = [torch.empty_like(o) for o in outs]
        write()
    write()                                     # inference tensors have no version to count
    turned = torch.zeros((3, 2, 8), dtype=BF16).transpose(0, 1)
    before = turned._version                    # x without rows: copied, and written once
    linear(_t(2, 8, 3).transpose(1, 2), w, out=turned)
    assert turned._version == before + 1
    outs = [torch.zeros_like(o).requires_grad_() for o in outs]
    for call in (lambda: linear(x, w, out=outs[0]), lambda: qk_norm_rope(q, k, out=(_t(2, 4, 6, 16), outs[2])),
                 lambda: window_attention(q, k, q, out=outs[3])):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()


def test_flags_of_an_earlier_call_are_raised_once(monkeypatch):
    held = torch.zeros(1, dtype=torch.int32)
    word = ctypes.c_int32.from_address(held.data_ptr())
    monkeypatch.setattr(layer, "_WORDS", {0: (held, word)})
    device = torch.device("cuda", 0)
    for flag, match in ((_abi.FLAG_TIMEOUT, "wait expired"), (_abi.FLAG_INTERNAL, "layout check")):
        held[0] = flag
        with pytest.raises(RuntimeError, match="an earlier linear or window_attention call on cuda:0.*" + match):
            layer._shared_status(device)
        assert held.item() == 0 and layer._shared_status(device) == held.data_ptr()
