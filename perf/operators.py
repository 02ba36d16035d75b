"""Performance cases of the operators around the attention call: the
projections (``linear``), the per-head norm and rotation of queries and keys
(``qk_norm_rope``) and the 16-bit attention over a sliding window with first
tokens that stay visible (``window_attention``).

``listed()`` and ``draw(rng)`` give cases, ``prepare`` makes a case's inputs,
``run`` makes one pass (the plain form, or the package's kernels where ``own``
is true), ``work`` counts the bytes and operations that a pass cannot do
without, and ``exact`` evaluates the definitions in 64 bits.
"""
import math
import pathlib
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ROOT = pathlib.Path(__file__).resolve().parents[1]


def _package():
    path = str(_ROOT / "vc-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vc_attention_b200

    return vc_attention_b200


# ------------------------------------------------------------------ the cases
#
# linear: y = residual + gate * act(x W^T + bias).
#   batch, tokens, in_features, out_features: x is [batch, tokens, in_features];
#   heads_in > 0: x comes as the attention's output [batch, heads_in, tokens, D];
#   heads_out > 0: y goes out as [batch, heads_out, tokens, D].
# qk_norm_rope: batch, heads, tokens, dim; rotary: rotated channels of a head;
#   rows: tokens that have a row in the tables (the rest keep their angle);
#   per_batch: one table for each batch entry.
# window_attention: batch, heads, queries, keys, dim; left / right: keys before
#   and after a query's position (-1: no bound); sinks: first keys that stay
#   visible; len_step: batch entry b holds keys - b * len_step keys (0: all).

def listed():
    return [
        # The conditioning embedding of one denoising step: one token, a
        # 40 x 128 wide layer, SiLU behind it.  The weights' bytes count.
        dict(name="linear_one_token", op="linear", dtype="bf16", batch=1, tokens=1, in_features=5120,
             out_features=5120, heads_in=0, heads_out=0, activation="silu", bias=True, gate=False, residual=False),
        # Q, K and V of a 32k-token video in one product, written head by head
        # as the attention reads them.
        dict(name="linear_qkv", op="linear", dtype="bf16", batch=1, tokens=32768, in_features=5120,
             out_features=15360, heads_in=0, heads_out=120, activation="none", bias=True, gate=False,
             residual=False),
        # The projection behind the attention: head-major input, gated residual.
        dict(name="linear_out", op="linear", dtype="fp16", batch=2, tokens=4095, in_features=5120,
             out_features=5120, heads_in=40, heads_out=0, activation="none", bias=True, gate=True, residual=True),
        # Widths that no 16-byte rule holds for, a short text, GELU.
        dict(name="linear_odd", op="linear", dtype="bf16", batch=3, tokens=257, in_features=1147,
             out_features=2049, heads_in=0, heads_out=0, activation="gelu", bias=True, gate=False, residual=True),
        # One new token for each of four sequences.
        dict(name="qk_one_token", op="qk_norm_rope", dtype="bf16", batch=4, heads=40, tokens=1, dim=128,
             rotary=128, rows=1, per_batch=True, interleaved=True, weights=True),
        # A 32k-token video, all channels rotated in adjacent pairs.
        dict(name="qk_video", op="qk_norm_rope", dtype="bf16", batch=1, heads=40, tokens=32768, dim=128,
             rotary=128, rows=32768, per_batch=False, interleaved=True, weights=True),
        # Video and text tokens in one sequence: the text's rows have no angle;
        # halves of the head are paired, and some channels are not rotated.
        dict(name="qk_joint", op="qk_norm_rope", dtype="fp16", batch=2, heads=24, tokens=4399, dim=96,
             rotary=64, rows=4173, per_batch=False, interleaved=False, weights=True),
        # 32-bit activations, odd length, no weights.
        dict(name="qk_fp32", op="qk_norm_rope", dtype="fp32", batch=2, heads=3, tokens=2001, dim=64,
             rotary=64, rows=2001, per_batch=False, interleaved=True, weights=False),
        # One query for each sequence against a long cache.
        dict(name="window_one_query", op="window_attention", dtype="bf16", batch=2, heads=40, queries=1,
             keys=32771, dim=128, left=8191, right=0, sinks=130, causal=True, len_step=1001),
        # A 32k-token video, each token with 4096 neighbours on both sides and
        # the first 1024 tokens.
        dict(name="window_video", op="window_attention", dtype="bf16", batch=1, heads=40, queries=32768,
             keys=32768, dim=128, left=4096, right=4096, sinks=1024, causal=False, len_step=0),
        # The next chunk of a video against the cache of the chunks before it.
        dict(name="window_chunk", op="window_attention", dtype="fp16", batch=1, heads=24, queries=1560,
             keys=24960, dim=128, left=16384, right=1559, sinks=1560, causal=False, len_step=0),
        # A padded batch of short causal sequences with an odd head width.
        dict(name="window_ragged", op="window_attention", dtype="bf16", batch=3, heads=5, queries=333,
             keys=1733, dim=80, left=200, right=0, sinks=3, causal=True, len_step=707),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_linear(rng):
    case = dict(op="linear", dtype=rng.choice(["bf16", "fp16"]), batch=rng.choice([1, 1, 2, 3]),
                tokens=_log_int(rng, 1, 8192), heads_in=0, heads_out=0,
                activation=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]), bias=rng.random() < 0.7,
                gate=False, residual=False)
    aligned = rng.random() < 0.7
    unit = 8 if aligned else 1
    if rng.random() < 0.3:
        heads = rng.randint(1, 40)
        dim = rng.choice([64, 80, 96, 128])
        case["heads_in"], case["in_features"] = heads, heads * dim
    else:
        case["in_features"] = unit * _log_int(rng, 1, 8192 // unit)
    if rng.random() < 0.3:
        heads = rng.randint(1, 72)
        dim = rng.choice([64, 80, 96, 128])
        case["heads_out"], case["out_features"] = heads, heads * dim
    else:
        case["out_features"] = unit * _log_int(rng, 1, 15360 // unit)
        case["gate"] = rng.random() < 0.5
        case["residual"] = case["gate"] or rng.random() < 0.5
    return case


def _draw_qk(rng):
    dim = 2 * rng.randint(8, 64) if rng.random() < 0.5 else rng.choice([64, 128])
    tokens = _log_int(rng, 1, 16384)
    return dict(op="qk_norm_rope", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), batch=rng.choice([1, 1, 2, 3]),
                heads=rng.randint(1, 40), tokens=tokens, dim=dim, rotary=2 * rng.randint(dim // 4, dim // 2),
                rows=tokens if rng.random() < 0.6 else rng.randint(1, tokens), per_batch=rng.random() < 0.3,
                interleaved=rng.random() < 0.5, weights=rng.random() < 0.8)


def _draw_window(rng):
    while True:
        keys = _log_int(rng, 1, 32768)
        kind = rng.choice(["one", "chunk", "all"])
        queries = {"one": 1, "chunk": _log_int(rng, 1, keys), "all": keys}[kind]
        causal = rng.random() < 0.5
        case = dict(op="window_attention", dtype=rng.choice(["bf16", "fp16"]), batch=rng.choice([1, 1, 2, 3]),
                    heads=rng.randint(1, 40), queries=queries, keys=keys,
                    dim=rng.choice([128, 128, 128, 64, 72, 80, 96, 41]),
                    left=rng.choice([-1, 0, _log_int(rng, 1, keys), _log_int(rng, 1, keys)]),
                    right=0 if causal else rng.choice([-1, 0, _log_int(rng, 1, keys), _log_int(rng, 1, keys)]),
                    sinks=rng.choice([0, 1, 4, _log_int(rng, 1, keys)]), causal=causal, len_step=0)
        if case["batch"] > 1 and rng.random() < 0.5:
            case["len_step"] = rng.randint(1, keys)
        if work(case)["flops"] <= 3e12:
            return case


def draw(rng):
    return rng.choice([_draw_linear, _draw_qk, _draw_window])(rng)


# ------------------------------------------------------------------ the inputs

def _lengths(case):
    return [max(0, case["keys"] - b * case["len_step"]) for b in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, mean=0.0, dt=dtype):
        out = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, scale, generator=g)
        return out.to(dt)

    state = dict(case=dict(case))
    b = case["batch"]
    if case["op"] == "linear":
        s, kf, nf = case["tokens"], case["in_features"], case["out_features"]
        # activations behind a norm, weights of variance 1 / in_features
        state["x"] = randn(b, case["heads_in"], s, kf // case["heads_in"]) if case["heads_in"] else randn(b, s, kf)
        state["weight"] = randn(nf, kf, scale=kf ** -0.5)
        state["bias"] = randn(nf, scale=0.1) if case["bias"] else None
        # one gate vector for each batch entry, kept in 32 bits as the
        # modulation of a denoising step is
        state["gate"] = randn(b, 1, nf, scale=0.5, dt=torch.float32) if case["gate"] else None
        state["residual"] = randn(b, s, nf) if case["residual"] else None
    elif case["op"] == "qk_norm_rope":
        h, s, d = case["heads"], case["tokens"], case["dim"]
        # Q and K as parts of one fused projection, seen as [B, H, S, D]
        qkv = randn(b, s, 3, h, d)
        state["q"], state["k"] = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
        state["q_weight"] = randn(d, scale=0.1, mean=1.0) if case["weights"] else None
        state["k_weight"] = randn(d, scale=0.1, mean=1.0) if case["weights"] else None
        half, rows = case["rotary"] // 2, case["rows"]
        tables = b if case["per_batch"] else 1
        # angles in 64 bits: position times frequency, positions starting
        # somewhere in a long video
        start = torch.randint(0, 100000, (tables, 1, 1), device="cuda", generator=g)
        pos = start.double() + torch.arange(rows, device="cuda", dtype=torch.float64).view(1, rows, 1)
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
        angle = pos * freq
        cos, sin = angle.cos().float(), angle.sin().float()
        state["cos"], state["sin"] = (cos, sin) if case["per_batch"] else (cos[0], sin[0])
    else:
        h, d = case["heads"], case["dim"]
        state["q"] = randn(b, h, case["queries"], d)
        # keys carry a channel offset, as they do behind the rotation
        offset = randn(b, h, 1, d, scale=0.5, dt=torch.float32)
        state["k"] = (randn(b, h, case["keys"], d, dt=torch.float32) + offset).to(dtype)
        state["v"] = randn(b, h, case["keys"], d)
        state["lengths"] = _lengths(case)
        state["kv_lens"] = (torch.tensor(state["lengths"], dtype=torch.int32, device="cuda") if case["len_step"]
                            else None)
    return state


# -------------------------------------------------------------- one pass

def _bound(value):
    return None if value < 0 else value


def _run_own(state):
    case = state["case"]
    vc = _package()
    if case["op"] == "linear":
        return vc.linear(state["x"], state["weight"], state["bias"],
                         activation=None if case["activation"] == "none" else case["activation"],
                         gate=state["gate"], residual=state["residual"], heads_in=case["heads_in"] > 0,
                         heads_out=case["heads_out"] or None)
    if case["op"] == "qk_norm_rope":
        return vc.qk_norm_rope(state["q"], state["k"], state["q_weight"], state["k_weight"], state["cos"],
                               state["sin"], eps=1e-6, interleaved=case["interleaved"])
    return vc.window_attention(state["q"], state["k"], state["v"], window=(_bound(case["left"]), _bound(case["right"])),
                               sinks=case["sinks"], causal=case["causal"], kv_lens=state["kv_lens"])


def _plain_linear(state):
    case, x = state["case"], state["x"]
    if case["heads_in"]:
        b, h, s, d = x.shape
        x = x.transpose(1, 2).reshape(b, s, h * d)
    y = x.float() @ state["weight"].float().t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    act = case["activation"]
    if act == "silu":
        y = y * (1 / (1 + torch.exp(-y)))
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.7071067811865476))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    elif act == "relu":
        y = torch.clamp(y, min=0)
    if state["gate"] is not None:
        y = y * state["gate"].float()
    if state["residual"] is not None:
        y = state["residual"].float() + y
    y = y.to(x.dtype)
    if case["heads_out"]:
        b, s, n = y.shape
        y = y.view(b, s, case["heads_out"], n // case["heads_out"]).transpose(1, 2).contiguous()
    return y


def _plain_norm_rope(x, weight, cos, sin, interleaved, eps):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    rows, half = cos.shape[-2], cos.shape[-1]
    if cos.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    head = y[..., :rows, :2 * half]
    if interleaved:
        a, c = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - c * sin, a * sin + c * cos), dim=-1).flatten(-2)
    else:
        a, c = head[..., :half], head[..., half:]
        turned = torch.cat((a * cos - c * sin, a * sin + c * cos), dim=-1)
    out = y.contiguous()
    out[..., :rows, :2 * half] = turned
    return out.to(x.dtype)


def _plain_window(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    scale = q.shape[-1] ** -0.5
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    block = 1024
    for b, length in enumerate(state["lengths"]):
        offset = length - case["queries"]
        for i in range(0, case["queries"], block):
            j = min(i + block, case["queries"])
            first, last = i + offset, j - 1 + offset
            lo = 0 if case["left"] < 0 else min(max(first - case["left"], 0), length)
            hi = length if case["right"] < 0 else min(last + case["right"] + 1, length)
            sink_hi = min(case["sinks"], length)
            if case["causal"]:
                hi, sink_hi = min(hi, last + 1), min(sink_hi, last + 1)
            hi, sink_hi = max(hi, lo), max(sink_hi, 0)
            if lo <= sink_hi:
                index = torch.arange(0, max(hi, sink_hi), device=q.device)
                kk, vv = k[b, :, :index.numel()].float(), v[b, :, :index.numel()].float()
            else:
                index = torch.cat((torch.arange(0, sink_hi, device=q.device),
                                   torch.arange(lo, hi, device=q.device)))
                kk = torch.cat((k[b, :, :sink_hi], k[b, :, lo:hi]), dim=1).float()
                vv = torch.cat((v[b, :, :sink_hi], v[b, :, lo:hi]), dim=1).float()
            if index.numel() == 0:
                out[b, :, i:j] = 0
                continue
            pos = torch.arange(first, last + 1, device=q.device)[:, None]
            seen = torch.ones(1, 1, dtype=torch.bool, device=q.device)
            if case["left"] >= 0:
                seen = seen & (index >= pos - case["left"])
            if case["right"] >= 0:
                seen = seen & (index <= pos + case["right"])
            seen = seen | (index < case["sinks"])
            if case["causal"]:
                seen = seen & (index <= pos)
            score = (q[b, :, i:j].float() @ kk.transpose(-1, -2)) * scale
            score = torch.where(seen, score, float("-inf"))
            top = score.amax(-1, keepdim=True)
            top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
            weight = torch.exp(score - top)
            total = weight.sum(-1, keepdim=True)
            total = torch.where(total == 0, torch.ones_like(total), total)
            out[b, :, i:j] = ((weight @ vv) / total).to(q.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "linear":
        return _plain_linear(state)
    if case["op"] == "qk_norm_rope":
        return (_plain_norm_rope(state["q"], state["q_weight"], state["cos"], state["sin"], case["interleaved"], 1e-6),
                _plain_norm_rope(state["k"], state["k_weight"], state["cos"], state["sin"], case["interleaved"], 1e-6))
    return _plain_window(state)


# -------------------------------------------------------------- the work

def _visible(case):
    """(pairs of a query and a key that it sees, keys that some query sees)
    of one head, summed over the batch."""
    pairs = keys = 0
    for length in _lengths(case):
        if length == 0:
            continue
        pos = torch.arange(case["queries"], dtype=torch.int64) + (length - case["queries"])
        lo = torch.zeros_like(pos) if case["left"] < 0 else (pos - case["left"]).clamp(0, length)
        hi = torch.full_like(pos, length) if case["right"] < 0 else (pos + case["right"] + 1).clamp(0, length)
        sink = torch.full_like(pos, min(case["sinks"], length))
        if case["causal"]:
            hi, sink = torch.minimum(hi, (pos + 1).clamp(min=0)), torch.minimum(sink, (pos + 1).clamp(min=0))
        hi = torch.maximum(hi, lo)
        # first the sinks, then the window's keys behind them
        pairs += int((sink + (hi - torch.maximum(lo, sink)).clamp(min=0)).sum())
        steps = torch.zeros(length + 1, dtype=torch.int64)
        some = hi > lo
        steps.index_add_(0, lo[some], torch.ones_like(lo[some]))
        steps.index_add_(0, hi[some], -torch.ones_like(hi[some]))
        seen = steps.cumsum(0)[:length] > 0
        seen[:int(sink.max())] = True
        keys += int(seen.sum())
    return pairs, keys


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    b = case["batch"]
    if case["op"] == "linear":
        m, n, k = b * case["tokens"], case["out_features"], case["in_features"]
        data = size * (m * k + n * k + m * n + n * case["bias"] + m * n * case["residual"])
        return {"bytes": data + 4 * b * n * case["gate"], "flops": 2 * m * n * k}
    if case["op"] == "qk_norm_rope":
        elements = 2 * b * case["heads"] * case["tokens"] * case["dim"]
        tables = (b if case["per_batch"] else 1) * case["rows"] * (case["rotary"] // 2) * 2
        return {"bytes": 2 * size * elements + 4 * tables + 2 * size * case["dim"] * case["weights"],
                "flops": 7 * elements}
    pairs, keys = _visible(case)
    rows = b * case["queries"]
    return {"bytes": size * case["heads"] * case["dim"] * (2 * rows + 2 * keys) + 4 * b * (case["len_step"] > 0),
            "flops": 4 * case["heads"] * case["dim"] * pairs}


# ------------------------------------------------------- the definitions, in 64 bits

def _exact_linear(state, case):
    x, w = state["x"].double(), state["weight"].double()
    if case["heads_in"]:
        h, d = x.shape[1], x.shape[3]
        # the sum over heads of each head's own product
        z = torch.einsum("bhsd,nhd->bsn", x, w.view(w.shape[0], h, d))
    else:
        z = torch.einsum("bsk,nk->bsn", x, w)
    del x, w
    if state["bias"] is not None:
        z += state["bias"].double()
    kind = case["activation"]
    if kind == "silu":
        z = z * torch.sigmoid(z)
    elif kind == "gelu":
        z = z * torch.special.ndtr(z)
    elif kind == "gelu_tanh":
        # 0.5 (1 + tanh u) is the logistic function at 2 u
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    elif kind == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    if state["gate"] is not None:
        z *= state["gate"].double()
    if state["residual"] is not None:
        z += state["residual"].double()
    if case["heads_out"]:
        z = torch.stack(z.chunk(case["heads_out"], dim=-1), dim=1)
    return z


def _exact_norm_rope(x, weight, cos, sin, interleaved):
    z = x.double()
    z = z / (z.pow(2).sum(-1, keepdim=True) / z.shape[-1] + 1e-6).sqrt()
    if weight is not None:
        z = z * weight.double()
    rows, half = cos.shape[-2], cos.shape[-1]
    turn = torch.complex(cos.double(), sin.double())
    if turn.dim() == 3:
        turn = turn.unsqueeze(1)
    part = z[:, :, :rows]
    if interleaved:
        pair = torch.complex(part[..., 0:2 * half:2], part[..., 1:2 * half:2]) * turn
        z[:, :, :rows, 0:2 * half:2], z[:, :, :rows, 1:2 * half:2] = pair.real, pair.imag
    else:
        pair = torch.complex(part[..., :half], part[..., half:2 * half]) * turn
        z[:, :, :rows, :half], z[:, :, :rows, half:2 * half] = pair.real, pair.imag
    return z


def _exact_window(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    b, h, sq, d = q.shape
    result = torch.zeros((b, h, sq, d), dtype=torch.float64, device=q.device)
    j = torch.arange(case["keys"], device=q.device)
    for entry in range(b):
        length = case["keys"] - entry * case["len_step"]
        if length <= 0:
            continue
        for begin in range(0, sq, 512):
            p = torch.arange(begin, min(begin + 512, sq), device=q.device).view(-1, 1) + (length - sq)
            after = torch.ones_like(p * j, dtype=torch.bool) if case["left"] < 0 else j >= p - case["left"]
            before = torch.ones_like(after) if case["right"] < 0 else j <= p + case["right"]
            allowed = ((j < case["sinks"]) | (after & before)) & (j < length)
            if case["causal"]:
                allowed &= j <= p
            columns = allowed.any(0).nonzero().flatten()
            if columns.numel() == 0:
                continue
            allowed = allowed[:, columns]
            some = allowed.any(1)
            rows = p.flatten()[some] - (length - sq)
            hidden = ~allowed[some]
            for head in range(h):
                logits = (q[entry, head, rows].double() @ k[entry, head, columns].double().t()) / math.sqrt(d)
                logits.masked_fill_(hidden, float("-inf"))
                result[entry, head, rows] = torch.softmax(logits, dim=-1) @ v[entry, head, columns].double()
    return result


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(state, case)
    if case["op"] == "qk_norm_rope":
        return tuple(_exact_norm_rope(state[x], state[x + "_weight"], state["cos"], state["sin"], case["interleaved"])
                     for x in "qk")
    return _exact_window(state, case)
