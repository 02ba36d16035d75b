"""The projections and the Q/K norm with rotation against plain 64-bit forms.

Tolerances are bounds, not fits.  ``linear``: a sum of K products is formed in
FP32 in K / 16 steps (one MMA step adds 16 products), each off by at most
2^-22 of the sum of magnitudes S (two units in the last place, as the steps
may truncate); bias, activation, gate and residual add a few FP32 roundings,
and an activation's slope is below 1.2.  The store rounds by half a step of
the output type.  ``qk_norm_rope``: the sum of squares is a chain of at most
nine additions and five shuffles (half of its relative error reaches the
norm), then two products and a rotation with two roundings: under 16 units
of 2^-24 of |n_a| + |n_b|, and the store's half step."""
import math

import pytest
import torch

from conftest import has_b200

gpu = [pytest.mark.gpu, pytest.mark.skipif(not has_b200(), reason="needs a B200 GPU")]
pytestmark = gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _act(kind, z):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if kind == "relu":
        return torch.clamp(z, min=0)
    return z


def _linear_ref(x, w, bias=None, activation=None, gate=None, residual=None):
    """(y, bound on the error before the store) in 64 bits; x [..., K]."""
    xd, wd = x.double(), w.double()
    acc = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    err = (x.shape[-1] / 16 + 2) * 2.0 ** -22 * mag
    size = acc.abs()
    if bias is not None:
        acc = acc + bias.double()
        size = size + bias.double().abs()
    y = _act(activation, acc)
    err = 1.2 * err + 16 * 2.0 ** -24 * size
    if gate is not None:
        y = y * gate.double()
        err = err * gate.double().abs()
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, err


def _check(got, ref, err, what=""):
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    tol = err + eps / 2 * (ref.abs() + err) + tiny
    diff = (got.double() - ref).abs()
    worst = (diff / tol).max().item()
    assert worst <= 1, f"{what}: {worst:.3f} of the tolerance"


LINEAR = [
    # batch, tokens, K, N
    (1, 1, 8, 8), (1, 1, 128, 64), (1, 1, 5120, 520), (2, 1, 1000, 24), (1, 2, 64, 16), (3, 5, 72, 40),
    (1, 16, 512, 4096), (1, 17, 136, 264), (1, 100, 520, 1032), (1, 127, 256, 256), (1, 128, 64, 256),
    (1, 129, 320, 248), (2, 255, 192, 504), (1, 257, 1024, 768), (1, 600, 128, 2048), (3, 333, 640, 1304),
    (1, 2100, 264, 4104), (1, 32, 640, 96), (4, 8, 1032, 72), (1, 33, 640, 96), (5, 7, 2048, 136),
    # tiles cut along K, alone and behind whole ones
    (1, 64, 5120, 512), (2, 200, 4096, 1000), (1, 2600, 2048, 2048),
    # off the 16-byte grid
    (1, 1, 1, 1), (1, 1, 77, 33), (1, 7, 9, 5), (2, 33, 100, 65), (1, 130, 257, 255), (3, 257, 1147, 2049),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,s,k,n", LINEAR)
def test_linear_sizes(b, s, k, n, dtype):
    from vc_attention_b200 import linear
    g = _gen(b * 7 + s + k + n)
    x, w = _randn((b, s, k), dtype, g), _randn((n, k), dtype, g, k ** -0.5)
    bias = _randn((n,), dtype, g)
    got = linear(x, w, bias)
    assert got.shape == (b, s, n) and got.dtype == dtype
    _check(got, *_linear_ref(x, w, bias))
    if b == 1:
        assert torch.equal(linear(x[0], w, bias), got[0])


@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_linear_epilogue(activation, dtype):
    from vc_attention_b200 import linear
    g = _gen(3)
    for b, s, k, n in [(2, 300, 256, 392), (2, 1, 256, 392), (2, 77, 131, 203)]:
        x, w = _randn((b, s, k), dtype, g, 2.0), _randn((n, k), dtype, g, 2 * k ** -0.5)
        res = _randn((b, s, n), dtype, g)
        for bias in (None, _randn((n,), FP32, g), _randn((n,), dtype, g)):
            for gate in (None, _randn((n,), dtype, g), _randn((b, 1, n), FP32, g), _randn((b, s, n), dtype, g)):
                kw = dict(activation=activation, gate=gate, residual=res if gate is not None else None)
                _check(linear(x, w, bias, **kw), *_linear_ref(x, w, bias, **kw), (activation, n))
        # in place on the residual stream
        want = linear(x, w, activation=activation, residual=res)
        held = res.clone()
        assert linear(x, w, activation=activation, residual=held, out=held) is held
        assert torch.equal(held, want)


@pytest.mark.parametrize("heads,dim", [(3, 128), (5, 64), (2, 96), (3, 80), (1, 40), (4, 41)])
@pytest.mark.parametrize("b,s", [(1, 1), (2, 1), (1, 300), (2, 129), (3, 70)])
def test_linear_head_layouts(heads, dim, b, s):
    from vc_attention_b200 import linear
    g = _gen(heads + dim + s)
    k = heads * dim
    x, w = _randn((b, s, k), BF16, g), _randn((3 * k, k), BF16, g, k ** -0.5)
    bias = _randn((3 * k,), BF16, g)
    want, err = _linear_ref(x, w, bias)
    got = linear(x, w, bias, heads_out=3 * heads)
    assert got.shape == (b, 3 * heads, s, dim) and got.is_contiguous()
    _check(got.transpose(1, 2).reshape(b, s, 3 * k), want, err)
    # the attention's output as input, contiguous and as a view of token-major memory
    xh = x.view(b, s, heads, dim).transpose(1, 2)
    for src in (xh.contiguous(), xh):
        _check(linear(src, w, bias, heads_in=True), want, err)
        out = linear(src, w, bias, heads_in=True, heads_out=3 * heads)
        _check(out.transpose(1, 2).reshape(b, s, 3 * k), want, err)


def test_linear_strides_and_guards():
    """Views as operands, outputs inside larger buffers: nothing around an
    output is written, and the value does not depend on the layout."""
    from vc_attention_b200 import linear
    g = _gen(5)
    b, s, k, n = 2, 150, 200, 136
    x, w = _randn((b, s, k), FP16, g), _randn((n, k), FP16, g)
    res = _randn((b, s, n), FP16, g)
    want = linear(x, w, residual=res)
    big = _randn((b, s + 3, k + 24), FP16, g)
    views = [big[:, 1:s + 1, 8:k + 8], big[:, :s, 3:k + 3], _randn((s, b, k), FP16, g).transpose(0, 1),
             torch.empty(b, s, 2 * k, device="cuda", dtype=FP16)[..., ::2]]
    for v in views:
        v.copy_(x)
        assert torch.equal(linear(v, w, residual=res), want)
    wide = _randn((n, k + 5), FP16, g)
    wide[:, :k] = w
    assert torch.equal(linear(x, wide[:, :k], residual=res), want)
    one = x[:1, :1].expand(b, s, k)
    assert torch.equal(linear(one, w), linear(one.contiguous(), w))
    for lo in (0, 1, 8):
        buf = torch.full((b, s + 2, n + 16), 7.0, device="cuda", dtype=FP16)
        out = buf[:, 1:s + 1, lo:lo + n]
        linear(x, w, residual=res, out=out)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert (buf == 7.0).all()
    buf = torch.full((b, 4, s + 9, n // 4), 7.0, device="cuda", dtype=FP16)
    linear(x, w, heads_out=4, out=buf[:, :, 5:s + 5])
    assert torch.equal(buf[:, :, 5:s + 5], linear(x, w, heads_out=4))
    assert (buf[:, :, :5] == 7.0).all() and (buf[:, :, s + 5:] == 7.0).all()


@pytest.mark.parametrize("s", [1, 9, 200])
def test_linear_non_finite_values_stay_in_their_row_and_column(s):
    from vc_attention_b200 import linear
    g = _gen(6)
    k, n = 264, 96
    x, w = _randn((1, s + 2, k), BF16, g), _randn((n, k), BF16, g)
    clean = linear(x, w, activation="relu")
    x2, w2 = x.clone(), w.clone()
    x2[0, s, 7] = float("nan")
    x2[0, s - 1, 3] = float("inf")
    w2[5, 0] = float("nan")
    got = linear(x2, w2, activation="relu")
    assert got[0, s].isnan().all() and got[..., 5].isnan().all()
    keep = [c for c in range(n) if c != 5]
    assert torch.equal(got[0, :s - 1][:, keep], clean[0, :s - 1][:, keep])
    assert torch.equal(got[0, s + 1][keep], clean[0, s + 1][keep])
    row = got[0, s - 1][keep]
    assert ((row == float("inf")) | (row == 0)).all()        # relu of +-inf


def test_linear_graph_stream_and_repeat():
    """A captured call replays on new contents, calls on two streams do not
    disturb one another, and a repeat gives the same bits."""
    from vc_attention_b200 import linear
    g = _gen(8)
    x, w = _randn((1, 90, 333), BF16, g), _randn((520, 333), BF16, g)
    x1, w1 = _randn((1, 1, 2048), BF16, g), _randn((512, 2048), BF16, g)
    want, want1 = linear(x, w), linear(x1, w1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, out1 = linear(x, w), linear(x1, w1)
    fresh, fresh1 = _randn(x.shape, BF16, g), _randn(x1.shape, BF16, g)
    expect, expect1 = linear(fresh, w), linear(fresh1, w1)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(out1, want1)
    x.copy_(fresh)
    x1.copy_(fresh1)
    graph.replay()
    assert torch.equal(out, expect) and torch.equal(out1, expect1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(linear(x, w) if i % 3 else linear(x1, w1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expect if i % 3 else expect1) for i, o in enumerate(got))


def _rope_ref(x, weight, cos, sin, interleaved, eps):
    n = x.double()
    if eps is not None:
        n = n / (n.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        n = n * weight.double()
    err = 16 * 2.0 ** -24 * n.abs()
    if cos is None:
        return n, err
    r, h = cos.shape[-2:]
    c, s = (t.double() if t.ndim == 2 else t.double()[:, None] for t in (cos, sin))
    idx = torch.arange(2 * h, device=x.device)
    a, b = (idx[0::2], idx[1::2]) if interleaved else (idx[:h], idx[h:])
    y = n.clone()
    na, nb = n[:, :, :r][..., a], n[:, :, :r][..., b]
    y[:, :, :r, a], y[:, :, :r, b] = na * c - nb * s, na * s + nb * c
    pair = 16 * 2.0 ** -24 * (na.abs() + nb.abs())
    err[:, :, :r, a] = pair
    err[:, :, :r, b] = pair
    return y, err


def _tables(rows, half, g, batch=None):
    shape = (rows, half) if batch is None else (batch, rows, half)
    angle = torch.rand(shape, device="cuda", generator=g) * 6.28
    return angle.cos(), angle.sin()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,h,hk,s,d,rotary,rows", [
    (1, 1, 1, 1, 128, 128, 1), (4, 40, 40, 1, 128, 128, 1), (2, 3, 1, 17, 128, 96, 17), (1, 5, 5, 40, 64, 64, 33),
    (1, 9, 2, 9, 96, 64, 9), (2, 2, 3, 8, 80, 80, 5), (1, 17, 4, 30, 32, 16, 30), (1, 3, 3, 10, 41, 22, 7),
    (2, 2, 2, 11, 2, 2, 11), (1, 2, 2, 5, 1, 0, 0), (1, 3, 3, 21, 126, 126, 21), (1, 2, 2, 6, 16, 10, 6),
])
def test_rope_sizes(b, h, hk, s, d, rotary, rows, interleaved, dtype):
    from vc_attention_b200 import qk_norm_rope
    g = _gen(h + s + d)
    q, k = _randn((b, h, s, d), dtype, g, 3.0), _randn((b, hk, s, d), dtype, g, 0.5)
    for weights in (True, False):
        qw, kw = (_randn((d,), dtype, g), _randn((d,), dtype, g)) if weights else (None, None)
        for batch in (None, b):
            cos, sin = _tables(rows, rotary // 2, g, batch) if rotary else (None, None)
            qo, ko = qk_norm_rope(q, k, qw, kw, cos, sin, interleaved=interleaved)
            assert qo.is_contiguous() and ko.is_contiguous()
            _check(qo, *_rope_ref(q, qw, cos, sin, interleaved, 1e-6))
            _check(ko, *_rope_ref(k, kw, cos, sin, interleaved, 1e-6))
    qo, ko = qk_norm_rope(q, k, None, None, cos, sin, interleaved=interleaved, eps=None)
    _check(qo, *_rope_ref(q, None, cos, sin, interleaved, None))
    qo, ko = qk_norm_rope(q, k, q_weight=_randn((d,), FP32, g), eps=0.5)
    _check(ko, *_rope_ref(k, None, None, None, interleaved, 0.5))


@pytest.mark.parametrize("d", [128, 64, 41])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_views_in_place_and_guards(d, interleaved):
    from vc_attention_b200 import qk_norm_rope
    g = _gen(d)
    b, h, s, half = 2, 5, 19, d // 4
    qkv = _randn((b, s, 3, h, d), BF16, g)
    q, k = (qkv[:, :, i].transpose(1, 2) for i in range(2))
    w = _randn((d,), FP32, g)
    wide = torch.rand((s, 3 * half + 1), device="cuda", generator=g)
    cos, sin = wide[:, :half].cos(), wide[:, 1:half + 1]
    kw = dict(interleaved=interleaved)
    want = qk_norm_rope(q.contiguous(), k.contiguous(), w, w, cos.contiguous(), sin.contiguous(), **kw)
    got = qk_norm_rope(q, k, w, w, cos, sin, **kw)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # rows of a longer K buffer, off the 16-byte grid too
    for shift in (0, 3):
        buf = torch.full((b, h, s + 6, d + 8), 7.0, device="cuda", dtype=BF16)
        ko = buf[:, :, 4:s + 4, shift:shift + d]
        qo = torch.empty_like(want[0])
        qk_norm_rope(q, k, w, w, cos, sin, out=(qo, ko), **kw)
        assert torch.equal(ko, want[1]) and torch.equal(qo, want[0])
        ko.fill_(7.0)
        assert (buf == 7.0).all()
    v = qkv[:, :, 2].clone()
    qk_norm_rope(q, k, w, w, cos, sin, out=(q, k), **kw)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, :, 2], v)


def test_rope_non_finite_rows_and_zero_rows():
    from vc_attention_b200 import qk_norm_rope
    g = _gen(12)
    for d in (128, 41):
        q = _randn((1, 4, 9, d), BF16, g)
        cos, sin = _tables(9, d // 2, g)
        want, _ = qk_norm_rope(q, q, None, None, cos, sin)
        bad = q.clone()
        bad[0, 1, 3, 5] = float("nan")
        bad[0, 2] = 0
        got, _ = qk_norm_rope(bad, q, None, None, cos, sin)
        assert got[0, 1, 3].isnan().all() and (got[0, 2] == 0).all()
        got[0, 1, 3], got[0, 2] = want[0, 1, 3], want[0, 2]
        assert torch.equal(got, want)
        # without the norm, an infinity reaches its own pair only, and only where the token turns
        bad = q.clone()
        bad[0, 0, 8, 0] = float("inf")
        got, _ = qk_norm_rope(bad, q, None, None, cos[:8], sin[:8], eps=None)
        assert got[0, 0, 8, 0] == float("inf") and got[0, 0, 8, 1:].isfinite().all()


def test_offsets_past_32_bits():
    """Outputs, inputs and caches of more than 2^31 elements: the last rows are
    what the same rows give alone."""
    from vc_attention_b200 import linear, qk_norm_rope, window_attention
    g = _gen(21)
    s, k, n = 135000, 64, 16000                      # 2.16e9 outputs
    x, w = _randn((1, s, k), BF16, g), _randn((n, k), BF16, g)
    y = linear(x, w)
    for lo in (0, s // 2, s - 300):
        assert torch.equal(y[:, lo:lo + 300], linear(x[:, lo:lo + 300].contiguous(), w))
    heads = linear(x, w, heads_out=125)
    assert torch.equal(heads[:, 124, -300:], y[:, -300:, -128:])
    del heads
    back = linear(y[:, -40:], w.t().contiguous())    # rows behind 2^31 elements as input
    assert torch.equal(back, linear(y[:, -40:].clone(), w.t().contiguous()))
    del y, back
    b, h, s, d = 1, 40, 425000, 128                  # 2.18e9 elements
    big = torch.empty((b, h, s, d), device="cuda", dtype=BF16).normal_(generator=g)
    cos, sin = _tables(s, d // 2, g)
    q, ko = qk_norm_rope(big, big, None, None, cos, sin)
    assert torch.equal(q, ko)
    tail, _ = qk_norm_rope(big[:, :, -100:], big[:, :, -100:], None, None, cos[-100:], sin[-100:])
    assert torch.equal(q[:, :, -100:], tail)
    del ko
    got = window_attention(q[:, :, -3:], q, big, window=(500, 0), causal=True)
    near = slice(s - 640, s)
    want = window_attention(q[:, :, -3:], q[:, :, near].contiguous(), big[:, :, near].contiguous(), window=(500, 0),
                            causal=True)
    assert (got.double() - want.double()).abs().max() <= 2.0 ** -7 * big[:, :, near].abs().max().double()


def test_calls_of_one_shape_from_two_threads():
    """The checked arguments of a shape are shared; addresses are not."""
    import threading

    from vc_attention_b200 import linear
    g = _gen(22)
    x = [_randn((1, 40, 256), BF16, g) for _ in range(8)]
    w = _randn((96, 256), BF16, g)
    want = [linear(t, w) for t in x]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(linear(x[i], w), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_rope_one_token_with_tables_from_two_caches():
    from vc_attention_b200 import qk_norm_rope
    g = _gen(77)
    q, k = _randn((2, 3, 1, 64), BF16, g), _randn((2, 1, 1, 64), BF16, g)
    cos_cache = _tables(9, 32, g)[0]
    for start in (0, 4, 5):                     # the second table on and off the 16-byte grid
        sin_cache = _tables(9, 48, g)[1][:, start:start + 32]
        cos, sin = cos_cache[5:6], sin_cache[5:6]
        for c, s in ((cos, sin), (sin, cos), (cos[None], sin[None])):
            qo, ko = qk_norm_rope(q, k, None, None, c, s)
            _check(qo, *_rope_ref(q, None, c, s, True, 1e-6))
            _check(ko, *_rope_ref(k, None, c, s, True, 1e-6))


def test_linear_few_rows_with_the_longest_sum():
    """K at the bound that the entry point takes: the walk over K ends there."""
    from vc_attention_b200 import linear
    k = 2 ** 31 - 264
    x = torch.zeros((1, k), device="cuda", dtype=BF16)
    w = torch.ones((1, k), device="cuda", dtype=BF16)
    for at, value in ((0, 1.0), (1023, 2.0), (1024, 4.0), (k // 2, 8.0), (k - 1025, 16.0), (k - 1, 32.0)):
        x[0, at] = value
    assert linear(x, w).item() == 63.0
    w[0, k - 1] = 0.5
    assert linear(x, w).item() == 47.0


def test_an_expired_wait_is_raised_by_the_next_call():
    """The self-test of the bounded waits (no fault, no hang: it gives up after
    2 s) sets the flag that a projection's or attention's own expired wait sets."""
    from vc_attention_b200 import layer, linear, window_attention
    g = _gen(41)
    x, w = _randn((1, 40, 64), BF16, g), _randn((32, 64), BF16, g)
    q = _randn((1, 1, 40, 64), BF16, g)
    own = torch.zeros(1, dtype=torch.int32, device="cuda")
    for call in (lambda **kw: linear(x, w, **kw), lambda **kw: window_attention(q, q, q, **kw)):
        want = call()
        src = torch.zeros(256, dtype=torch.int32, device="cuda")
        report = torch.empty(4, dtype=torch.int32, device="cuda")
        lib = layer._abi.load()
        word = layer._shared_status(x.device)
        layer._abi.check(lib, lib.vcb_wait_selftest(0, src.data_ptr(), word, report.data_ptr(), None))
        torch.cuda.synchronize()
        assert torch.equal(call(status=own), want) and own.item() == 0      # that caller looks after itself
        with pytest.raises(RuntimeError, match="an earlier .* wait expired"):
            call()
        assert torch.equal(call(), want)


def test_the_first_call_of_a_process_may_be_captured():
    import pathlib
    import subprocess
    import sys
    code = """
import torch
from vc_attention_b200 import linear, window_attention
x = torch.ones((1, 40, 64), device="cuda", dtype=torch.bfloat16)
w = torch.ones((32, 64), device="cuda", dtype=torch.bfloat16)
q = torch.ones((1, 1, 40, 64), device="cuda", dtype=torch.bfloat16)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, o = linear(x, w), window_attention(q, q, q)
graph.replay()
torch.cuda.synchronize()
assert (y == 64).all() and (o == 1).all()
print("captured")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).resolve().parents[1] / "vc-attention_b200",
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,s,heads,k,n", [
    (1, 40, 1, 20000, 96), (3, 100, 1, 24000, 72), (1, 17, 1, 17832, 8), (2, 70, 192, 24576, 200),       # cut tiles alone
    (1, 40, 1, 20001, 95),                                                                               # off the grid
    (1, 6273, 1, 12040, 272), (1, 9586, 1, 9504, 240),                                                   # behind whole ones
])
def test_linear_tiles_cut_along_k(b, s, heads, k, n, dtype):
    """These shapes are cut (their scratch says so), and every epilogue and
    layout runs behind the join."""
    from vc_attention_b200 import layer, linear
    g = _gen(k + n)
    x, w = _randn((b, s, k), dtype, g), _randn((n, k), dtype, g, k ** -0.5)
    plan = layer._linear_plan(x, w, None, None, None, None, False, None, None, None)
    copies = 0 if k % 8 == 0 else 2 * (b * s + n) * (k + 7) + 512
    assert plan.need > copies
    res, bias, gate = _randn((b, s, n), dtype, g), _randn((n,), FP32, g), _randn((b, 1, n), FP32, g)
    kw = dict(activation="gelu", gate=gate, residual=res)
    want, err = _linear_ref(x, w, bias, **kw)
    got = linear(x, w, bias, **kw)
    _check(got, want, err)
    assert torch.equal(linear(x, w, bias, **kw), got)
    # in place on the residual, and inside a larger buffer on and off the 16-byte grid
    held = res.clone()
    assert torch.equal(linear(x, w, bias, activation="gelu", gate=gate, residual=held, out=held), got)
    for lo in (3, 8):
        buf = torch.full((b, s + 2, n + 16), 7.0, device="cuda", dtype=dtype)
        out = buf[:, 1:s + 1, lo:lo + n]
        linear(x, w, bias, out=out, **kw)
        assert torch.equal(out, got)
        out.fill_(7.0)
        assert (buf == 7.0).all()
    if heads > 1:
        xh = x.view(b, s, heads, k // heads).transpose(1, 2).contiguous()
        _check(linear(xh, w, bias, heads_in=True, **kw), want, err)
    if n % 8 == 0:
        split = linear(x, w, bias, heads_out=4)
        _check(split.transpose(1, 2).reshape(b, s, n), *_linear_ref(x, w, bias))


def test_calls_under_a_default_device(monkeypatch):
    from vc_attention_b200 import layer, linear, window_attention
    g = _gen(43)
    x, w = _randn((1, 40, 64), BF16, g), _randn((32, 64), BF16, g)
    q = _randn((1, 1, 40, 64), BF16, g)
    want = linear(x, w), window_attention(q, q, q)
    torch.cuda.synchronize()
    held = layer._WORDS
    monkeypatch.setattr(layer, "_WORDS", {})
    with torch.device("cuda"):
        got = linear(x, w), window_attention(q, q, q)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and layer._WORDS.keys() == held.keys()
