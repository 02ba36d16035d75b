"""window_attention against the definition in 64 bits.

Tolerance, a bound for one row with seen keys j, softmax weights w_j and
A = sum_j w_j |v_j| (per channel):
- the weights are rounded to the operand type before the product with V, half
  a step each, and the sum of the rounded weights divides: 2 (eps / 2) A;
- a logit is a sum of D products in FP32 steps of 16, off by at most
  d = (D / 16 + 2) 2^-22 scale sum |q||k|; weights and their sum move by 2 d A;
- the exponential's argument and result round in FP32: 2^-20 (1 + max |logit|) A;
- the product with V adds (n / 16 + 8) FP32 steps of 2^-22 A;
- FP16 weights below 2^-14 of the reference round by 2^-25: n 2^-25 max |v|;
and the store rounds by half a step."""
import pytest
import torch

from conftest import has_b200

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_b200(), reason="needs a B200 GPU")]

BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _seen(b, sq, sk, window, sinks, causal, q_offset, lens):
    """[B, Sq, Sk] truth table of the definition."""
    left, right = window
    j = torch.arange(sk, device="cuda")
    rows = []
    for e in range(b):
        n = sk if lens is None else min(max(lens[e], 0), sk)
        p = torch.arange(sq, device="cuda")[:, None] + (n - sq if q_offset is None else q_offset)
        near = torch.ones((sq, sk), dtype=torch.bool, device="cuda")
        if left is not None:
            near &= j >= p - left
        if right is not None:
            near &= j <= p + right
        seen = (near | (j < sinks)) & (j < n)
        if causal:
            seen &= j <= p
        rows.append(seen)
    return torch.stack(rows)


def _reference(q, k, v, seen, scale):
    qd, kd, vd = q.double(), k.double(), v.double()
    s = qd @ kd.transpose(-1, -2) * scale
    mag = qd.abs() @ kd.abs().transpose(-1, -2) * scale
    hidden = ~seen[:, None]
    s = s.masked_fill(hidden, float("-inf"))
    empty = hidden.all(-1, keepdim=True)
    w = torch.softmax(s.masked_fill(empty, 0.0), -1).masked_fill(hidden, 0.0)
    out = w @ vd
    big = w @ vd.abs()
    dot = (q.shape[-1] / 16 + 2) * 2.0 ** -22 * mag.masked_fill(hidden, 0).amax(-1, keepdim=True)
    top = s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True)
    n = seen.sum(-1)[:, None, :, None].double()
    eps = torch.finfo(q.dtype).eps
    err = (eps + 2 * dot + 2.0 ** -20 * (1 + top) + (n / 16 + 8) * 2.0 ** -22) * big
    if q.dtype == FP16:
        err = err + n * 2.0 ** -25 * vd.abs().amax(2, keepdim=True)
    return out, err


def _check(got, ref, err):
    if not got.numel():
        return
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    worst = ((got.double() - ref).abs() / (err + eps / 2 * (ref.abs() + err) + tiny)).max().item()
    assert worst <= 1, f"{worst:.3f} of the tolerance"


def _run(q, k, v, *, window=(None, None), sinks=0, causal=False, q_offset=None, lens=None, scale=None, **kw):
    from vc_attention_b200 import window_attention
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = window_attention(q, k, v, window=window, sinks=sinks, causal=causal, q_offset=q_offset, kv_lens=kv_lens,
                           scale=scale, **kw)
    seen = _seen(q.shape[0], q.shape[2], k.shape[2], window, sinks, causal, q_offset, lens)
    return got, _reference(q, k, v, seen, scale or q.shape[-1] ** -0.5), seen


SHAPES = [
    # B, H, Sq, Sk, D
    (1, 1, 1, 1, 128), (1, 2, 1, 2, 128), (2, 3, 1, 700, 128), (1, 2, 3, 129, 128), (1, 1, 16, 128, 64),
    (2, 2, 65, 65, 128), (1, 2, 128, 128, 128), (1, 2, 129, 400, 128), (1, 3, 255, 257, 128), (1, 1, 256, 1024, 128),
    (1, 2, 300, 300, 80), (1, 1, 700, 1300, 128), (2, 1, 515, 515, 41), (1, 2, 40, 90, 1), (1, 2, 130, 260, 96),
    (1, 1, 400, 150, 128),
]
MASKS = [
    dict(), dict(causal=True), dict(window=(0, 0)), dict(window=(70, 0), causal=True),
    dict(window=(100, 37), sinks=5), dict(window=(20, None), sinks=130), dict(window=(None, 10)),
    dict(window=(128, 128), sinks=128, causal=True), dict(window=(3, 1000), sinks=1), dict(sinks=64, window=(0, 0)),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("shape", SHAPES)
def test_window_sizes_and_masks(shape, mask, dtype):
    b, h, sq, sk, d = shape
    g = _gen(sq + sk + d + mask)
    q, k, v = _randn((b, h, sq, d), dtype, g), _randn((b, h, sk, d), dtype, g), _randn((b, h, sk, d), dtype, g)
    got, (ref, err), seen = _run(q, k, v, **MASKS[mask])
    assert got.shape == q.shape and got.is_contiguous()
    _check(got, ref, err)
    assert (got.transpose(1, 2)[~seen.any(-1)] == 0).all()


@pytest.mark.parametrize("offset", [-500, -3, 0, 17, 250, 5000])
@pytest.mark.parametrize("mask", [1, 3, 4, 7])
def test_window_offsets_and_empty_rows(offset, mask):
    g = _gen(offset + 999)
    q, k, v = _randn((1, 2, 200, 128), BF16, g), _randn((1, 2, 333, 128), BF16, g), _randn((1, 2, 333, 128), BF16, g)
    got, (ref, err), seen = _run(q, k, v, q_offset=offset, **MASKS[mask])
    _check(got, ref, err)
    assert (got.transpose(1, 2)[~seen.any(-1)] == 0).all()


@pytest.mark.parametrize("sq", [1, 130, 300])
@pytest.mark.parametrize("mask", [0, 1, 3, 4, 7])
def test_window_padded_batch(sq, mask):
    """Entries of different lengths, zero and out-of-range ones among them; the
    padding holds NaN and infinities and must not reach the output."""
    g = _gen(sq)
    lens = [700, 0, 1, 129, 300, 900, -4]
    b = len(lens)
    q, k, v = _randn((b, 2, sq, 128), FP16, g), _randn((b, 2, 700, 128), FP16, g), _randn((b, 2, 700, 128), FP16, g)
    ref_out, (ref, err), seen = _run(q, k, v, lens=lens, **MASKS[mask])
    _check(ref_out, ref, err)
    for e, n in enumerate(lens):
        k[e, :, max(n, 0):] = float("nan")
        v[e, :, max(n, 0):] = float("inf")
    got, _, _ = _run(q, k, v, lens=lens, **MASKS[mask])
    assert torch.equal(got, ref_out)


@pytest.mark.parametrize("sq,sk", [(1, 600), (200, 600), (600, 600)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_window_non_finite_keys_reach_the_rows_that_see_them_only(sq, sk, bad):
    g = _gen(sq)
    q, k, v = _randn((1, 2, sq, 128), BF16, g), _randn((1, 2, sk, 128), BF16, g), _randn((1, 2, sk, 128), BF16, g)
    kw = dict(window=(60, 0), sinks=2, causal=True)
    clean, (ref, err), seen = _run(q, k, v, **kw)
    _check(clean, ref, err)
    for key in (sk - 30, sk - 300, 1):
        for which in (k, v):
            held = which[0, 1, key].clone()
            which[0, 1, key] = bad
            got, _, _ = _run(q, k, v, **kw)
            which[0, 1, key] = held
            sees = seen[0, :, key]
            assert torch.equal(got[0, 0], clean[0, 0])
            # a row that does not see the key keeps its value within the bound
            _check(got[:, 1:, ~sees], ref[:, 1:, ~sees], err[:, 1:, ~sees])
            if which is v and sees.any():
                assert not got[0, 1][sees].isfinite().any()


def test_window_views_guards_and_scale():
    from vc_attention_b200 import window_attention
    g = _gen(4)
    b, h, sq, sk, d = 2, 3, 140, 500, 128
    q, k, v = _randn((b, h, sq, d), BF16, g), _randn((b, h, sk, d), BF16, g), _randn((b, h, sk, d), BF16, g)
    kw = dict(window=(90, 10), sinks=4, scale=0.3)
    got, (ref, err), _ = _run(q, k, v, **kw)
    _check(got, ref, err)
    qkv = torch.empty((b, sk, 3, h, d), device="cuda", dtype=BF16)
    kt, vt = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    kt.copy_(k)
    vt.copy_(v)
    assert torch.equal(window_attention(q, kt, vt, **kw), got)
    odd = torch.empty((b, h, sk + 3, d + 3), device="cuda", dtype=BF16)[:, :, 1:sk + 1, 1:d + 1]
    odd.copy_(k)
    assert torch.equal(window_attention(q, odd, vt, **kw), got)
    for shift in (0, 1, 8):
        buf = torch.full((b, h, sq + 4, d + 16), 7.0, device="cuda", dtype=BF16)
        out = buf[:, :, 2:sq + 2, shift:shift + d]
        window_attention(q, k, v, out=out, **kw)
        assert torch.equal(out, got)
        out.fill_(7.0)
        assert (buf == 7.0).all()
    one = q[:, :1, :1].expand(b, h, sq, d)
    assert torch.equal(window_attention(one, k, v, **kw), window_attention(one.contiguous(), k, v, **kw))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_window_peaked_and_rising_logits(dtype):
    """Logits that rise along the keys move the running maximum at every tile;
    one dominant key must come back with its value almost exactly."""
    g = _gen(9)
    sq, sk, d = 150, 1500, 128
    q, v = _randn((1, 1, sq, d), dtype, g), _randn((1, 1, sk, d), dtype, g)
    k = _randn((1, 1, sk, d), dtype, g, 0.05)
    up = torch.linspace(-40, 40, sk, device="cuda")
    q[..., 0] = 8.0
    k[..., 0] = (up * d ** 0.5 / 8.0).to(dtype)
    for kw in (dict(), dict(window=(700, 0), causal=True, sinks=3)):
        got, (ref, err), _ = _run(q, k, v, **kw)
        _check(got, ref, err)
    k[..., 0] = (-up * d ** 0.5 / 8.0).to(dtype)
    got, (ref, err), _ = _run(q, k, v)
    _check(got, ref, err)
    k[0, 0, 777] = 30.0 * q[0, 0, 0] / q[0, 0, 0].float().norm()
    got, (ref, err), _ = _run(q, k, v, scale=1.0)
    _check(got, ref, err)


def test_window_long_chunk_and_one_query():
    g = _gen(10)
    q, k, v = _randn((1, 3, 520, 128), BF16, g), _randn((1, 3, 9000, 128), BF16, g), _randn((1, 3, 9000, 128), BF16, g)
    for kw in (dict(window=(5000, 519), sinks=300), dict(window=(100, 50), sinks=4000), dict()):
        got, (ref, err), _ = _run(q, k, v, **kw)
        _check(got, ref, err)
        got, (ref, err), _ = _run(q[:, :, -1:], k, v, **kw)
        _check(got, ref, err)


def test_window_graph_streams_and_repeat():
    from vc_attention_b200 import window_attention
    g = _gen(11)
    q, k, v = _randn((1, 2, 64, 128), BF16, g), _randn((1, 2, 4000, 128), BF16, g), _randn((1, 2, 4000, 128), BF16, g)
    lens = torch.tensor([3500], dtype=torch.int32, device="cuda")
    kw = dict(window=(2000, 0), sinks=16, causal=True, kv_lens=lens)
    want = window_attention(q, k, v, **kw)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention(q, k, v, **kw)
    with torch.cuda.graph(other):
        out2 = window_attention(q[:, :, :1], k, v, **kw)
    graph.replay()
    assert torch.equal(out, want)
    # the cache grows on the device between replays
    lens.fill_(4000)
    k.normal_(generator=g)
    other.replay()
    graph.replay()
    assert torch.equal(out, window_attention(q, k, v, **kw))
    assert torch.equal(out2, window_attention(q[:, :, :1], k, v, **kw))
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [window_attention(q, k, v, **kw), window_attention(q[:, :, :1], k, v, **kw)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(window_attention(q if i % 3 else q[:, :, :1], k, v, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0 if i % 3 else 1]) for i, o in enumerate(got))


def test_layer_chain_runs_as_one_block():
    """Projection, norm with rotation, windowed and full attention, projection
    back onto the residual: the chain equals its parts in 64 bits within the
    16-bit roundings in between, captured and replayed."""
    from vc_attention_b200 import Config, attention, linear, qk_norm_rope, window_attention
    g = _gen(13)
    b, s, h, d = 1, 640, 2, 128
    c = h * d
    x = _randn((b, s, c), BF16, g)
    w_in, w_out = _randn((3 * c, c), BF16, g, c ** -0.5), _randn((c, c), BF16, g, c ** -0.5)
    qw, kw = _randn((d,), BF16, g, 0.1) + 1, _randn((d,), BF16, g, 0.1) + 1
    angle = torch.arange(s, device="cuda")[:, None] * 0.9 ** torch.arange(d // 2, device="cuda")
    cos, sin = angle.cos(), angle.sin()
    gate = torch.full((b, 1, c), 0.5, device="cuda")

    def block():
        q, k, v = linear(x, w_in, heads_out=3 * h).split(h, dim=1)
        q, k = qk_norm_rope(q, k, qw, kw, cos, sin)
        near = window_attention(q, k, v, window=(128, 128), sinks=64)
        return q, k, v, near, linear(near, w_out, heads_in=True, gate=gate, residual=x)

    q, k, v, near, y = block()
    qkv = (x.double() @ w_in.double().t()).view(b, s, 3, h, d)
    # two roundings to BF16 lie between qkv and q; one before v
    assert (v.double() - qkv[:, :, 2].transpose(1, 2)).abs().max() <= 2.0 ** -8 * qkv.abs().max() + 1e-3
    seen = _seen(b, s, s, (128, 128), 64, False, None, None)
    ref, err = _reference(q, k, v, seen, d ** -0.5)
    _check(near, ref, err)
    flat = near.transpose(1, 2).reshape(b, s, c).double()
    want = x.double() + 0.5 * (flat @ w_out.double().t())
    mag = flat.abs() @ w_out.double().abs().t()
    # the store's half step: BF16 keeps 8 bits, so values in [1, 2) are 2^-7 apart and a
    # rounding moves one by up to 2^-8 of itself
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.01 + (c / 16 + 2) * 2.0 ** -22 * mag + 1e-6).all()
    full, stats = attention(q, k, v, Config())
    assert stats["native_fused_attention"] and full.shape == near.shape
    linear(full, w_out, heads_in=True, residual=x, out=x.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()[-1]
    x.normal_(generator=g)
    graph.replay()
    assert torch.equal(out, block()[-1])


def test_preflight_covers_the_layer_operators():
    from vc_attention_b200 import b200_backend
    b200_backend._preflight_layer("cuda:0")
    assert b200_backend.preflight("cuda:0")["preflight"] == "passed"


@pytest.mark.parametrize("d", [128, 41])
@pytest.mark.parametrize("sq,sk", [(1, 40), (1, 3000), (70, 600), (200, 600)])
def test_window_rows_whose_logits_are_all_minus_infinity(sq, sk, d):
    """Softmax has no value there (0 / 0) and the output is NaN; zeros are for
    rows that see no key.  One finite key among them takes the whole weight."""
    g = _gen(sq + d)
    q = _randn((2, 2, sq, d), BF16, g).abs() + 0.5
    k, v = _randn((2, 2, sk, d), BF16, g), _randn((2, 2, sk, d), BF16, g)
    k[0, 1, :, 0] = -float("inf")
    lens = [sk, 0]
    for kw in (dict(), dict(window=(3, 0), causal=True)):
        got, (ref, err), seen = _run(q, k, v, lens=lens, **kw)
        _check(got[:1, :1], ref[:1, :1], err[:1, :1])
        assert got[0, 1].isnan().all()
        assert (got[1] == 0).all()
        held = k[0, 1, sk - 2].clone()
        k[0, 1, sk - 2, 0] = 1.0
        got, _, _ = _run(q, k, v, lens=lens, **kw)
        k[0, 1, sk - 2] = held
        sees = seen[0, :, sk - 2]
        assert sees.any() and torch.equal(got[0, 1][sees], v[0, 1, sk - 2].expand(int(sees.sum()), d))
        assert got[0, 1][~sees].isnan().all()


@pytest.mark.parametrize("sq,sk,d", [(1, 60000, 128), (200, 60000, 128), (300, 60000, 64), (40, 700, 80)])
def test_window_small_fp16_weights_keep_their_share(sq, sk, d):
    """One key of value 0 above very many of value 1 with weights near 2^-26
    each: their sum is the output.  A weight is held as 2^7 w or more, so a step
    of FP16's smallest numbers is 2^-24 / 2^7, a rounding at most half of it."""
    q = torch.zeros((1, 2, sq, d), device="cuda", dtype=FP16)
    k, v = (torch.zeros((1, 2, sk, d), device="cuda", dtype=FP16) for _ in range(2))
    q[..., 0] = 1.0
    for first in (0, sk // 2, sk - 1):
        k[..., 0], v[:] = -18.203125, 1.0
        k[:, :, first], v[:, :, first] = 0.0, 0.0
        got, _, _ = _run(q, k, v, q_offset=0, scale=1.0)
        rest = (sk - 1) * torch.tensor(-18.203125, dtype=torch.float64).exp().item()
        want = rest / (1 + rest)
        # the weights' roundings, the exponential's (2^-20 (1 + 18.2) of each), the sums' steps, the store
        tol = (sk - 1) * 2.0 ** -32 + (2.0 ** -15 + (sk / 16 + 8) * 2.0 ** -22) * want + 2.0 ** -11 * want + 2.0 ** -25
        assert (got.double() - want).abs().max() <= tol


def _tight(q, k, v, seen, scale):
    """(output, bound) with one rounding of the weights: they are summed before
    it, so only the product with V takes their half steps, (eps / 2) A, and in
    FP16 half a step of its smallest numbers, 2^-25 of 2^7 or more: n 2^-32 max |v|.
    The other terms are those of _reference."""
    qd, kd, vd = q.double(), k.double(), v.double()
    hidden = ~seen[:, None]
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(hidden, float("-inf"))
    mag = (qd.abs() @ kd.abs().transpose(-1, -2) * scale).masked_fill(hidden, 0)
    w = torch.softmax(s.masked_fill(hidden.all(-1, keepdim=True), 0.0), -1).masked_fill(hidden, 0.0)
    big = w @ vd.abs()
    dot = (q.shape[-1] / 16 + 2) * 2.0 ** -22 * mag.amax(-1, keepdim=True)
    top = s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True)
    n = seen.sum(-1)[:, None, :, None].double()
    eps = torch.finfo(q.dtype).eps
    err = (eps / 2 + 2 * dot + 2.0 ** -20 * (1 + top) + (n / 16 + 8) * 2.0 ** -22) * big
    if q.dtype == FP16:
        err = err + n * 2.0 ** -32 * vd.abs().amax(2, keepdim=True)
    return w @ vd, err


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("shape", [(1, 2, 1, 700, 128), (1, 2, 130, 260, 96), (2, 1, 515, 515, 41), (1, 1, 300, 5000, 64)])
def test_window_weights_are_rounded_once(shape, mask, dtype):
    b, h, sq, sk, d = shape
    g = _gen(sq + sk + d + mask)
    q, k, v = (_randn((b, h, n, d), dtype, g, a) for n, a in ((sq, 3.0), (sk, 1.0), (sk, 1.0)))
    got, _, seen = _run(q, k, v, **MASKS[mask])
    _check(got, *_tight(q, k, v, seen, d ** -0.5))


@pytest.mark.parametrize("sq,sk,d", [(1, 40, 128), (1, 3000, 128), (70, 600, 80), (200, 600, 41), (300, 300, 64)])
def test_window_sums_of_the_largest_values_stay_finite(sq, sk, d):
    """Finite BF16 values whose unnormalised sum passes FP32's range: the mean
    is in range and must come out."""
    g = _gen(sq + sk)
    q, k = _randn((1, 2, sq, d), BF16, g), _randn((1, 2, sk, d), BF16, g)
    most = torch.finfo(BF16).max
    v = (torch.rand((1, 2, sk, d), device="cuda", generator=g) * 2 - 1).mul(most).to(BF16)
    v[:, 1] = most                             # equal values: their mean is the value itself
    for kw in (dict(), dict(window=(90, 0), causal=True, sinks=7)):
        got, _, seen = _run(q, k, v, **kw)
        ref, err = _reference(q.double(), k.double(), v.double(), seen, d ** -0.5)
        eps = torch.finfo(BF16).eps
        err = err + (eps + torch.finfo(torch.float32).eps) * most      # (_reference took eps from 64-bit copies)
        assert got.isfinite().all()
        assert ((got.double() - ref).abs() <= err + eps / 2 * (ref.abs() + err)).all()
        assert (got[:, 1][seen.any(-1)] == most).all()


@pytest.mark.parametrize("sq", [3, 200])
def test_window_bounds_past_the_farthest_position(sq):
    """A bound wider than any position sees every key on its side."""
    from vc_attention_b200 import window_attention
    g = _gen(31)
    q, k, v = _randn((1, 1, sq, 64), BF16, g), _randn((1, 1, 50, 64), BF16, g), _randn((1, 1, 50, 64), BF16, g)
    want = window_attention(q, k, v)
    far = 2 ** 39 - 1
    assert torch.equal(window_attention(q, k, v, window=(2 ** 41, 0), q_offset=far), want)
    assert torch.equal(window_attention(q, k, v, window=(0, 2 ** 41), q_offset=-far), want)
    assert torch.equal(window_attention(q, k, v, window=(0, 0), sinks=2 ** 41, q_offset=far), want)


@pytest.mark.parametrize("sq,sk", [(1, 600), (200, 600), (300, 3000)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_window_non_finite_keys_give_what_the_definition_gives(sq, sk, bad):
    """A key with one bad channel: a NaN or +inf logit makes its rows NaN, a
    -inf logit takes the key out of them; rows that do not see it keep their value."""
    g = _gen(sq + 5)
    q, k, v = _randn((1, 2, sq, 128), BF16, g), _randn((1, 2, sk, 128), BF16, g), _randn((1, 2, sk, 128), BF16, g)
    kw = dict(window=(60, 0), sinks=2, causal=True)
    _, (clean, clean_err), seen = _run(q, k, v, **kw)
    for key in (sk - 30, sk - 100, 1, sk - 1):
        held = k[0, 1, key].clone()
        k[0, 1, key, 3] = bad
        got, _, _ = _run(q, k, v, **kw)
        k[0, 1, key] = held
        sees = seen[0, :, key]
        _check(got[:, :, ~sees], clean[:, :, ~sees], clean_err[:, :, ~sees])
        _check(got[:, :1], clean[:, :1], clean_err[:, :1])
        sign = q[0, 1, :, 3].sign() * bad                     # the logit's infinity, or NaN
        gone = sees & (sign < 0)
        assert got[0, 1][sees & ~gone].isnan().all()
        without = seen.clone()
        without[:, :, key] = False
        ref, err = _reference(q, k, v, without, 128 ** -0.5)
        _check(got[:, 1:, gone], ref[:, 1:, gone], err[:, 1:, gone])


@pytest.mark.parametrize("b,h,sq,sk,d", [
    (2, 41, 300, 1500, 128), (2, 41, 300, 1500, 80), (2, 41, 300, 1500, 41), (2, 41, 300, 1500, 64),     # two query tiles
    (2, 151, 3, 3000, 128), (2, 151, 3, 3000, 72),                                                       # one
])
@pytest.mark.parametrize("mask", [0, 3, 4])
def test_window_whole_items_and_items_cut_along_their_keys(b, h, sq, sk, d, mask):
    """More items than CTAs at once: those behind the full rounds are cut along
    their keys.  Entries of different lengths, padding and a key that hold NaN."""
    from vc_attention_b200 import window
    g = _gen(sq + d + mask)
    q, k, v = _randn((b, h, sq, d), BF16, g), _randn((b, h, sk, d), BF16, g), _randn((b, h, sk, d), BF16, g)
    kw = dict(dict(causal=mask == 3, window=(None, None), sinks=0), **MASKS[mask])
    if mask:
        kw["window"] = tuple(None if x is None else 16 * x for x in kw["window"])
    slots = torch.cuda.get_device_properties(0).multi_processor_count * (2 if sq <= 128 else 1)
    assert b * h * -(-sq // (128 if sq <= 128 else 256)) > slots
    if d % 8 == 0:                          # nothing is copied, so scratch means items cut along their keys
        plan = window._window_plan(q, k, v, kw["window"], kw["sinks"], kw["causal"], None, None, None, None, None)
        assert plan.need > 0
    lens = [sk, sk - 389]
    clean, (ref, err), seen = _run(q, k, v, lens=lens, **kw)
    _check(clean, ref, err)
    for e, n in enumerate(lens):
        k[e, :, n:], v[e, :, n:] = float("nan"), float("inf")
    assert torch.equal(_run(q, k, v, lens=lens, **kw)[0], clean)
    for e, head in ((0, 0), (b - 1, h - 1)):                  # the first item and the last
        key = lens[e] - 300
        held = v[e, head, key].clone()
        v[e, head, key] = float("nan")
        got, _, _ = _run(q, k, v, lens=lens, **kw)
        v[e, head, key] = held
        sees = seen[e, :, key]
        assert got[e, head][sees].isnan().all()
        _check(got[e, head][~sees], ref[e, head][~sees], err[e, head][~sees])
        got[e, head] = clean[e, head]
        assert torch.equal(got, clean)
