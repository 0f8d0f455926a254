"""Workloads of the token operators: per-head norm with position rotation of queries and keys,
counter-based dropout with a residual, and token log probabilities with entropy and top
alternatives, forward and (in training) backward, on series of a given degree (degree 0: ordinary
tensors).  Every case runs either in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through the framework's public calls on the same inputs.
"""

import functools
import math
import pathlib
import sys

import numpy as np
import torch

own = False
device = "cuda"

_DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
_MAX_POSITION = 8192
_EPS = 1e-6
_IGNORE = -100


# ---------------------------------------------------------------------------------------------
# cases

def _qk(name, batch, length, heads, kv_heads, dim, degree, dtype, train, rotary=None, interleaved=False,
        weight="series", packed=False, decode=False):
    return {"name": name, "op": "qk_norm_rope", "batch": batch, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": dim if rotary is None else rotary,
            "interleaved": interleaved, "degree": degree, "dtype": dtype, "weight": weight, "packed": packed,
            "decode": decode, "train": train}


def _drop(name, rows, cols, degree, dtype, train, residual=True, p=0.1):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "degree": degree, "dtype": dtype,
            "residual": residual, "p": p, "train": train}


def _logp(name, rows, vocab, degree, dtype, train, top=0, masked=False, temperature=1.0):
    return {"name": name, "op": "token_log_probs", "rows": rows, "vocab": vocab, "degree": degree, "dtype": dtype,
            "top": top, "masked": masked, "temperature": temperature, "train": train}


def listed():
    return [
        # training micro-batch of the 12-layer, 768-wide decoder: 8 x 1024 tokens, 12 heads of 64, float32 degree 3
        _qk("qk_train_f32", 8, 1024, 12, 12, 64, 3, "f32", True),
        # the 32-head, 128-wide attention shape with keys shared by groups of four heads, bf16 storage, read in
        # place out of one packed projection
        _qk("qk_train_bf16_groups", 4, 4096, 32, 8, 128, 3, "bf16", True, packed=True),
        # one decoding step of 32 sequences at their own positions: latency
        _qk("qk_decode_bf16", 32, 1, 32, 8, 128, 0, "bf16", False, weight="plain", packed=True, decode=True),
        # evaluation of one document of odd length, half of each head rotated, adjacent pairs, first derivative
        _qk("qk_partial_f16_odd", 1, 777, 13, 1, 96, 1, "f16", False, rotary=48, interleaved=True, weight="plain"),
        # residual branch of the same micro-batch
        _drop("dropout_train_f32", 8 * 1024, 768, 3, "f32", True),
        # residual branch of the wide activations, ordinary tensors in bf16
        _drop("dropout_train_bf16", 16384, 4096, 0, "bf16", True, p=0.05),
        # a fine-tuning batch of one short, ragged sequence: latency, and a tail that fills no vector
        _drop("dropout_f16_odd", 33, 777, 2, "f16", True, residual=False, p=0.25),
        # policy-gradient loss on the answers' tokens: 2 x 1024 rows of the 32000-word vocabulary
        _logp("logp_train_f32", 2 * 1024, 32000, 3, "f32", True),
        # the same with an odd vocabulary, words masked off and padded rows, in bf16
        _logp("logp_train_bf16_odd", 1511, 50021, 1, "bf16", True, top=4, masked=True, temperature=0.7),
        # serving: four sequences' next-token statistics with the best five alternatives
        _logp("logp_decode_bf16", 4, 32000, 0, "bf16", False, top=5),
        # serving one sequence of a large vocabulary, with its first derivative
        _logp("logp_decode_f32_wide", 1, 128256, 1, "f32", False, top=20, temperature=0.8),
        # evaluation in double precision
        _logp("logp_eval_f64", 300, 8191, 2, "f64", True, top=1),
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "f16", "f64"])
    degree = rng.choice([0, 1, 2, 3, 3, 4])
    size = _BYTES[dtype] * (degree + 1)
    train = rng.random() < 0.6
    op = rng.choice(["qk", "dropout", "logp"])
    if op == "qk":
        kv = rng.choice([1, 2, 3, 4, 8, 12])
        heads = kv * rng.choice([1, 1, 2, 4])
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
        tokens = _spread(rng, 1, max(2, min(20000, int(4.0e8 / (size * dim * (heads + kv))))))
        batch = min(tokens, rng.choice([1, 1, 2, 3, 8, 32]))
        length = max(1, tokens // batch)
        rotary = rng.choice([dim, dim, dim // 2])
        return _drawn(_qk("", batch, min(length, _MAX_POSITION), heads, kv, dim, degree, dtype, train,
                          rotary=rotary - rotary % 2, interleaved=rng.random() < 0.3,
                          weight=rng.choice(["series", "plain"]), packed=rng.random() < 0.5,
                          decode=rng.random() < 0.3))
    if op == "dropout":
        cols = _spread(rng, 5, 8192)
        rows = _spread(rng, 1, max(2, int(2.0e8 / (size * cols))))
        return _drawn(_drop("", rows, cols, degree, dtype, train, residual=rng.random() < 0.6,
                            p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5])))
    vocab = _spread(rng, 1000, 130000)
    rows = _spread(rng, 1, max(2, int(7.0e8 / (size * vocab))))
    return _drawn(_logp("", rows, vocab, degree, dtype, train, top=rng.choice([0, 0, 1, 5, 20]),
                        masked=rng.random() < 0.3, temperature=rng.choice([1.0, 1.0, 0.7])))


def _drawn(case):
    return {k: v for k, v in case.items() if k != "name"}


def work(case):
    planes, e = case["degree"] + 1, _BYTES[case["dtype"]]
    train = case["train"]
    products = planes * (planes + 1) // 2
    if case["op"] == "qk_norm_rope":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        # forward: x in, y out; backward: x and g in, dx out
        return {"bytes": n * planes * e * (5 if train else 2), "flops": n * products * (16 if train else 6)}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        moved = 2 + case["residual"] + (2 if train else 0)
        return {"bytes": n * planes * e * moved, "flops": n * planes * (3 if train else 2)}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * planes * e * (3 if train else 1), "flops": n * products * (8 if train else 4)}


# ---------------------------------------------------------------------------------------------
# inputs

def _series(shape, case, g, std=1.0, mean=0.0):
    """Planes N(mean, std) and N(0, std / k!) of the case's type."""
    dt = _DTYPES[case["dtype"]]
    make = dt if dt == torch.float64 else torch.float32
    return [((torch.randn(shape, generator=g, device=device, dtype=make) * (std / math.factorial(k)))
             + (mean if k == 0 else 0.0)).to(dt) for k in range(case["degree"] + 1)]


def prepare(case, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    state = {"case": dict(case)}
    if case["op"] == "qk_norm_rope":
        B, T, H, K, D = (case[k] for k in ("batch", "length", "heads", "kv_heads", "dim"))
        if case["packed"]:
            packed = _series((B, T, (H + 2 * K) * D), case, g, 1.3)
            state["q"] = [p[..., :H * D].unflatten(-1, (H, D)) for p in packed]
            state["k"] = [p[..., H * D:(H + K) * D].unflatten(-1, (K, D)) for p in packed]
        else:
            state["q"], state["k"] = _series((B, T, H, D), case, g, 1.3), _series((B, T, K, D), case, g, 1.3)
        planes = case["degree"] + 1 if case["weight"] == "series" else 1
        state["qw"] = _series((D,), case, g, 0.02, 1.0)[:planes]
        state["kw"] = _series((D,), case, g, 0.02, 1.0)[:planes]
        # the rotation's angles: base 10000, one row for each position
        wide = torch.float64
        inv = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device=device, dtype=wide) / case["rotary"])
        angle = torch.arange(_MAX_POSITION, device=device, dtype=wide)[:, None] * inv
        table = torch.float64 if case["dtype"] == "f64" else torch.float32
        state["cos"], state["sin"] = angle.cos().to(table), angle.sin().to(table)
        if case["decode"]:
            first = torch.randint(0, _MAX_POSITION - T + 1, (B, 1), generator=g, device=device)
            state["positions"] = first + torch.arange(T, device=device)
        else:
            state["positions"] = None
        if case["train"]:
            state["gq"], state["gk"] = _series((B, H, T, D), case, g), _series((B, K, T, D), case, g)
    elif case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        state["x"] = _series(shape, case, g)
        state["residual"] = _series(shape, case, g, 2.0) if case["residual"] else None
        state["seed"], state["offset"] = 0x9E37_79B9_0000 + 7919 * seed, 3 + seed % 5
        if case["train"]:
            state["g"] = _series(shape, case, g)
    else:
        R, V = case["rows"], case["vocab"]
        state["logits"] = _series((R, V), case, g, 2.5)
        state["tokens"] = torch.randint(0, V, (R,), generator=g, device=device)
        if case["masked"]:
            # a tenth of the words is not allowed here, one row in 16 is padding
            off = torch.rand(V, generator=g, device=device) < 0.1
            state["logits"][0].masked_fill_(off, -math.inf)
            allowed = (~off).nonzero().flatten()
            state["tokens"] = allowed[state["tokens"] % allowed.numel()]
            state["tokens"].masked_fill_(torch.rand(R, generator=g, device=device) < 1 / 16, _IGNORE)
        if case["train"]:
            state["ga"], state["gb"] = (
                [p.to(torch.promote_types(p.dtype, torch.float32)) for p in _series((R,), case, g)] for _ in range(2))
    return state


# ---------------------------------------------------------------------------------------------
# the plain forms: planes as lists, 32 bits, rounded once at the end

def _wide(planes):
    """The planes in the type that they are computed in."""
    return [p if p.dtype == torch.float64 else p.float() for p in planes]


def _round(planes, like):
    return [p.to(like) for p in planes]


def _mul(a, b):
    """The truncated product of two series; a short one has zeros in its missing planes."""
    n = max(len(a), len(b))
    return [sum(a[i] * b[k - i] for i in range(k + 1) if i < len(a) and k - i < len(b)) for k in range(n)]


def _recur(first, step, n):
    """Planes 0 .. n-1, each from the earlier ones."""
    return functools.reduce(lambda y, k: y + [step(y, k)], range(1, n), [first])


def _exp(x):
    return _recur(torch.exp(x[0]), lambda y, k: sum((i / k) * x[i] * y[k - i] for i in range(1, k + 1)), len(x))


def _log(x):
    """The logarithm's planes: k x_0 y_k = k x_k - sum_i i y_i x_{k-i}."""
    return _recur(torch.log(x[0]), lambda y, k: (x[k] - sum((i / k) * y[i] * x[k - i] for i in range(1, k))) / x[0],
                  len(x))


def _div(a, b):
    """The quotient's planes: b_0 y_k = a_k - sum_i b_i y_{k-i}."""
    return _recur(a[0] / b[0], lambda y, k: (a[k] - sum(b[i] * y[k - i] for i in range(1, k + 1))) / b[0], len(a))


def _rsqrt(s):
    return _recur(s[0].rsqrt(),
                  lambda y, k: -sum((2 * k - i) / (2 * k) * s[i] * y[k - i] for i in range(1, k + 1)) / s[0], len(s))


def _halves(x, case):
    """The two members of each rotated pair, and the features that are not rotated."""
    rot = case["rotary"]
    if case["interleaved"]:
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]


def _rotate(x, cos, sin, case):
    a, b, rest = _halves(x, case)
    lo, hi = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((lo, hi), -1).flatten(-2) if case["interleaved"] else torch.cat((lo, hi), -1)
    return torch.cat((turned, rest), -1)


def _angles(state):
    T = state["case"]["length"]
    rows = slice(0, T) if state["positions"] is None else state["positions"]
    cos, sin = (t[rows] for t in (state["cos"], state["sin"]))
    return (cos[:, None], sin[:, None]) if cos.dim() == 2 else (cos[:, :, None], sin[:, :, None])


def _plain_norm_rope(x, w, cos, sin, case):
    x, w, like = _wide(x), _wide(w), x[0].dtype
    s = [t.mean(-1, keepdim=True) for t in _mul(x, x)]
    r = _rsqrt([s[0] + _EPS] + s[1:])
    y = [_rotate(t, cos, sin, case).transpose(1, 2) for t in _mul(_mul(x, r), w)]
    return [t.contiguous().to(like) for t in y]


def _plain_norm_rope_grad(x, w, g, cos, sin, case):
    like, weights = x[0].dtype, len(w)
    x, w = _wide(x), _wide(w)
    s = [t.mean(-1, keepdim=True) for t in _mul(x, x)]
    r = _rsqrt([s[0] + _EPS] + s[1:])
    g = [_rotate(t.transpose(1, 2), cos, -sin, case) for t in _wide(g)]
    gy = _mul(g, w)
    c = [t.mean(-1, keepdim=True) for t in _mul(x, gy)]
    scale = _mul(_mul(_mul(r, r), r), c)
    dx = [p - q for p, q in zip(_mul(gy, r), _mul(x, scale))]
    dw = [t.sum((0, 1, 2)) for t in _mul(g, _mul(x, r))]
    return _round(dx, like), _round(dw[:weights], like)


def _plain_qk(state):
    case = state["case"]
    cos, sin = _angles(state)
    out = {"q": _plain_norm_rope(state["q"], state["qw"], cos, sin, case),
           "k": _plain_norm_rope(state["k"], state["kw"], cos, sin, case)}
    if case["train"]:
        out["dq"], out["dqw"] = _plain_norm_rope_grad(state["q"], state["qw"], state["gq"], cos, sin, case)
        out["dk"], out["dkw"] = _plain_norm_rope_grad(state["k"], state["kw"], state["gk"], cos, sin, case)
    return out


_M32 = 0xFFFFFFFF


def _philox_words(seed, offset, count):
    """The first ``count`` 32-bit words of the stream (seed, offset) of Philox4x32-10 (Salmon et al.,
    "Parallel random numbers: as easy as 1, 2, 3", SC 2011): word i is word i % 4 of counter i / 4."""
    i = torch.arange((count + 3) // 4, device=device, dtype=torch.int64)
    start = (i & _M32, i >> 32, torch.full_like(i, offset & _M32), torch.full_like(i, (offset >> 32) & _M32))

    def turn(c, n):
        k0, k1 = (seed + n * 0x9E3779B9) & _M32, ((seed >> 32) + n * 0xBB67AE85) & _M32
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        return (((q >> 32) & _M32) ^ c[1] ^ k0, q & _M32, ((p >> 32) & _M32) ^ c[3] ^ k1, p & _M32)

    return torch.stack(functools.reduce(turn, range(10), start), -1).flatten()[:count]


def _plain_dropout(state):
    case = state["case"]
    x = state["x"]
    keep = _philox_words(state["seed"], state["offset"], x[0].numel()).view_as(x[0]) >= int(case["p"] * 2**32)
    scale = 1.0 / (1.0 - case["p"])
    kept = lambda planes: [torch.where(keep, t * scale, 0.0) for t in _wide(planes)]  # noqa: E731
    y = kept(x)
    if state["residual"] is not None:
        y = [a + b for a, b in zip(y, _wide(state["residual"]))]
    out = {"y": _round(y, x[0].dtype)}
    if case["train"]:
        out["dx"] = _round(kept(state["g"]), x[0].dtype)
    return out


def _plain_log_probs(state):
    case, tokens = state["case"], state["tokens"]
    like = state["logits"][0].dtype
    z = [t * (1.0 / case["temperature"]) for t in _wide(state["logits"])]
    open_ = z[0] > -math.inf
    read = tokens != _IGNORE
    at = tokens.clamp(min=0)[:, None]
    top = torch.argsort(state["logits"][0].to(z[0].dtype), dim=-1, descending=True, stable=True)[:, :case["top"]]
    m = z[0].amax(-1, keepdim=True)
    shifted = [torch.where(open_, t, 0.0) for t in [z[0] - m] + z[1:]]
    weight = [torch.where(open_, t, 0.0) for t in _exp(shifted)]
    total = [t.sum(-1, keepdim=True) for t in weight]
    log_total = _log(total)
    mean = _div([t.sum(-1, keepdim=True) for t in _mul(weight, shifted)], total)
    entropy = [a - b for a, b in zip(log_total, mean)]
    # log probabilities, -inf (and no direction) at masked words
    logp = [torch.where(open_, a - b, -math.inf if k == 0 else 0.0)
            for k, (a, b) in enumerate(zip(shifted, log_total))]
    row = lambda t: torch.where(read, t, 0.0)  # noqa: E731
    out = {"log_probs": [row(t.gather(1, at)[:, 0]) for t in logp], "entropy": [row(t[:, 0]) for t in entropy]}
    if case["top"]:
        out["top"] = [torch.where(read[:, None], t.gather(1, top), 0.0) for t in logp]
        out["top_tokens"] = torch.where(read[:, None], top, -1)
    if case["train"]:
        a, b = ([row(t)[:, None] for t in _wide(state[name])] for name in ("ga", "gb"))
        p = _div(weight, total)
        finite = [torch.where(open_, t, 0.0) for t in logp]
        inner = [s + t for s, t in zip(a, _mul(b, [s + t for s, t in zip(finite, entropy)]))]
        hit = torch.zeros_like(open_).scatter_(1, at, True)
        dz = [torch.where(open_, torch.where(hit, s, 0.0) - t, 0.0) for s, t in zip(a, _mul(p, inner))]
        out["dlogits"] = _round([t * (1.0 / case["temperature"]) for t in dz], like)
    return out


# ---------------------------------------------------------------------------------------------
# the framework's calls

def _polytensor():
    path = str(pathlib.Path(__file__).resolve().parents[1] / "poly-tensors_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from polytensors_b200 import PolyTensor
    return PolyTensor


def _in(P, planes, grad=False):
    """Planes as the user's variable: a PolyTensor, or an ordinary tensor where there is one plane."""
    if len(planes) > 1:
        return P(tuple(planes), requires_grad=grad)
    return planes[0].detach().requires_grad_() if grad else planes[0]


def _out(x):
    """A variable's planes."""
    return list(x.coeffs) if hasattr(x, "coeffs") else [x.detach()]


def _own_qk(P, state):
    case, train = state["case"], state["case"]["train"]
    q, k, qw, kw = (_in(P, state[n], train) for n in ("q", "k", "qw", "kw"))
    y = P.qk_norm_rope(q, k, qw, kw, state["cos"], state["sin"], positions=state["positions"], eps=_EPS,
                       interleaved=case["interleaved"], check_indices=False)
    out = {"q": _out(y[0]), "k": _out(y[1])}
    if train:
        d = torch.autograd.grad(y, (q, k, qw, kw), (_in(P, state["gq"]), _in(P, state["gk"])))
        out |= {n: _out(t) for n, t in zip(("dq", "dk", "dqw", "dkw"), d)}
    return out


def _own_dropout(P, state):
    case = state["case"]
    x = _in(P, state["x"], case["train"])
    residual = _in(P, state["residual"]) if state["residual"] is not None else None
    y = P.dropout(x, case["p"], seed=state["seed"], offset=state["offset"], residual=residual)
    out = {"y": _out(y)}
    if case["train"]:
        out["dx"] = _out(torch.autograd.grad(y, x, _in(P, state["g"]))[0])
    return out


def _own_log_probs(P, state):
    case = state["case"]
    z = _in(P, state["logits"], case["train"])
    got = P.token_log_probs(z, state["tokens"], top=case["top"], temperature=case["temperature"],
                            ignore_index=_IGNORE, check_indices=False)
    out = {"log_probs": _out(got.log_probs), "entropy": _out(got.entropy)}
    if case["top"]:
        out["top"], out["top_tokens"] = _out(got.top_log_probs), got.top_tokens
    if case["train"]:
        seeds = (_in(P, state["ga"]), _in(P, state["gb"]))
        out["dlogits"] = _out(torch.autograd.grad((got.log_probs, got.entropy), z, seeds)[0])
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"qk_norm_rope": _plain_qk, "dropout": _plain_dropout, "token_log_probs": _plain_log_probs}[op](state)
    P = _polytensor()
    with P.plain_range(), P.retain_wrappers():
        return {"qk_norm_rope": _own_qk, "dropout": _own_dropout, "token_log_probs": _own_log_probs}[op](P, state)


# ---------------------------------------------------------------------------------------------
# 64 bits, from the definitions: series functions by Newton's iteration and power sums, gradients by
# differentiating the coefficient map (the gradient series' plane j is the derivative of
# sum_k <G_k, y_(n-k)> by input plane n - j), the generator in numpy

def _times(a, b):
    n = len(a)
    return [torch.stack([a[i] * b[k - i] for i in range(k + 1)]).sum(0) for k in range(n)]


def _powers(u, coefficients):
    """sum_j coefficients[j] u^j for a series u without constant term."""
    one = [torch.ones_like(u[0])] + [torch.zeros_like(t) for t in u[1:]]
    total = [torch.zeros_like(t) for t in u]
    for c in coefficients[:len(u)]:
        total = [t + c * o for t, o in zip(total, one)]
        one = _times(one, u)
    return total


def _newton_rsqrt(s):
    y = [s[0] ** -0.5] + [torch.zeros_like(t) for t in s[1:]]
    for _ in range(4):   # 1, 3, 7, 15 planes right
        e = _times(s, _times(y, y))
        y = _times(y, [(3.0 if k == 0 else 0.0) * 0.5 - 0.5 * t for k, t in enumerate(e)])
    return y


def _vjp(outputs, seeds, inputs):
    """The gradient series of ``inputs`` (lists of leaf planes) for the output series' seeds."""
    total = sum((g.double() * y).sum() for ys, gs in zip(outputs, seeds) for g, y in zip(gs, reversed(ys)))
    flat = torch.autograd.grad(total, [t for x in inputs for t in x], allow_unused=True)
    n = len(inputs[0])
    planes = [torch.zeros_like(t) if d is None else d for d, t in zip(flat, [t for x in inputs for t in x])]
    return [list(reversed(planes[i * n:(i + 1) * n])) for i in range(len(inputs))]


def _leaves(planes, n, grad):
    full = [p.double() for p in planes] + [torch.zeros_like(planes[0], dtype=torch.float64)] * (n - len(planes))
    return [p.clone().requires_grad_(grad) for p in full]


def _exact_heads(x, w, g, cos, sin, case):
    """One batch entry: x (T, H, D), angles (T, 1, rot / 2), g (H, T, D) or None."""
    n = case["degree"] + 1
    x, w = _leaves(x, n, g is not None), _leaves(w, n, g is not None)
    s = [t.mean(-1, keepdim=True) for t in _times(x, x)]
    r = _newton_rsqrt([s[0] + _EPS] + s[1:])
    v = _times(_times(x, r), [t.expand_as(x[0]) for t in w])
    rot = case["rotary"]
    first = torch.arange(0, rot, 2, device=device) if case["interleaved"] else torch.arange(rot // 2, device=device)
    second = first + (1 if case["interleaved"] else rot // 2)
    turn = torch.complex(cos, sin)
    y = []
    for t in v:
        pair = torch.complex(t[..., first], t[..., second]) * turn
        y.append(t.index_copy(-1, first, pair.real).index_copy(-1, second, pair.imag).transpose(0, 1))
    if g is None:
        return y, None, None
    dx, dw = _vjp([y], [g], [x, w])
    return [t.detach() for t in y], dx, dw


def _exact_qk(state):
    case, out = state["case"], {}
    if case["degree"] > 5:
        return None
    T = case["length"]
    rows = state["positions"] if state["positions"] is not None else torch.arange(T, device=device).expand(case["batch"], T)
    # the angles are inputs: the tables' own values
    for name, weight in (("q", "qw"), ("k", "kw")):
        ys, dxs, dws = [], [], None
        for b in range(case["batch"]):
            cos, sin = (t[rows[b]].double()[:, None] for t in (state["cos"], state["sin"]))
            g = [t[b] for t in state["g" + name]] if case["train"] else None
            y, dx, dw = _exact_heads([t[b] for t in state[name]], state[weight], g, cos, sin, case)
            ys.append(y)
            if g is not None:
                dxs.append(dx)
                dws = dw if dws is None else [s + t for s, t in zip(dws, dw)]
        stack = lambda parts: [torch.stack([p[k] for p in parts]) for k in range(case["degree"] + 1)]  # noqa: E731
        out[name] = stack(ys)
        if case["train"]:
            out["d" + name], out["d" + weight] = stack(dxs), dws[:len(state[weight])]
    return out


def _exact_dropout(state):
    case = state["case"]
    n = state["x"][0].numel()
    if n > 1 << 27:
        return None
    low, high, shift, mask = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(32), np.uint64(_M32)
    words = np.empty(((n + 3) // 4, 4), dtype=np.uint32)
    for first in range(0, len(words), 1 << 17):   # a counter block that stays in the cache
        block = words[first:first + (1 << 17)]
        i = np.arange(first, first + len(block), dtype=np.uint64)
        c = [i & mask, i >> shift, np.uint64(state["offset"] & _M32), np.uint64(state["offset"] >> 32)]
        key = [state["seed"] & _M32, (state["seed"] >> 32) & _M32]
        for _ in range(10):
            p, q = c[0] * low, c[2] * high
            c = [(q >> shift) ^ c[1] ^ np.uint64(key[0]), q & mask, (p >> shift) ^ c[3] ^ np.uint64(key[1]), p & mask]
            key = [(key[0] + 0x9E3779B9) & _M32, (key[1] + 0xBB67AE85) & _M32]
        for j in range(4):
            block[:, j] = c[j]
    words = words.reshape(-1)[:n]
    keep = torch.from_numpy(words >= np.uint32(int(case["p"] * 2**32))).to(device).view_as(state["x"][0])
    drop = lambda planes: [t.double() * keep / (1.0 - case["p"]) for t in planes]  # noqa: E731
    y = drop(state["x"])
    if state["residual"] is not None:
        y = [s + t.double() for s, t in zip(y, state["residual"])]
    out = {"y": y}
    if case["train"]:
        out["dx"] = drop(state["g"])
    return out


def _exact_rows(z, token, top, ga, gb, case):
    """Rows of logits planes (R, V) whose tokens are all read."""
    n, train = len(z), case["train"]
    leaf = _leaves(z, n, train)
    closed = torch.isneginf(z[0])
    with torch.enable_grad():
        x = [t.masked_fill(closed, 0.0) / case["temperature"] for t in leaf]
        top_value = x[0].detach().masked_fill(closed, -math.inf).amax(-1, keepdim=True)
        base = (x[0] - top_value).exp().masked_fill(closed, 0.0)
        u = [torch.zeros_like(x[0])] + x[1:]
        e = [base * t for t in _powers(u, [1.0 / math.factorial(j) for j in range(n)])]
        total = [t.sum(-1, keepdim=True) for t in e]
        v = [torch.zeros_like(total[0])] + [t / total[0] for t in total[1:]]
        log_total = _powers(v, [0.0] + [(-1.0) ** (j + 1) / j for j in range(1, n)])
        log_total[0] = log_total[0] + total[0].log()
        logp = [x[0] - top_value - log_total[0]] + [s - t for s, t in zip(x[1:], log_total[1:])]
        inverse = [t / total[0] for t in _powers(v, [(-1.0) ** j for j in range(n)])]
        p = _times(e, [t.expand_as(e[0]) for t in inverse])
        entropy = [-t.sum(-1) for t in _times(p, [t.masked_fill(closed, 0.0) for t in logp])]
        chosen = [t.gather(1, token[:, None])[:, 0] for t in logp]
        d = _vjp([chosen, entropy], [ga, gb], [leaf])[0] if train else None
    best = [t.detach().masked_fill(closed, -math.inf if k == 0 else 0.0).gather(1, top) for k, t in enumerate(logp)]
    return [t.detach() for t in chosen], [t.detach() for t in entropy], best, d


def _exact_log_probs(state):
    case = state["case"]
    R, V, n = case["rows"], case["vocab"], case["degree"] + 1
    if R * V * n * n > 6e9 or n > 6:
        return None
    zeros = lambda *shape: [torch.zeros(shape, dtype=torch.float64, device=device) for _ in range(n)]  # noqa: E731
    out = {"log_probs": zeros(R), "entropy": zeros(R)}
    if case["top"]:
        out["top"] = zeros(R, case["top"])
        out["top_tokens"] = torch.full((R, case["top"]), -1, dtype=torch.int64, device=device)
    if case["train"]:
        out["dlogits"] = zeros(R, V)
    read = (state["tokens"] != _IGNORE).nonzero().flatten()
    for rows in read.split(max(1, int(2.5e8 // (V * n * n)))):
        z = [t[rows] for t in state["logits"]]
        # the k largest, ties to the lowest index
        top = torch.sort(z[0].double(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        seeds = [[t[rows] for t in state[name]] if case["train"] else None for name in ("ga", "gb")]
        a, h, best, d = _exact_rows(z, state["tokens"][rows], top, *seeds, case)
        for k in range(n):
            out["log_probs"][k][rows], out["entropy"][k][rows] = a[k], h[k]
            if case["top"]:
                out["top"][k][rows] = best[k]
            if d is not None:
                out["dlogits"][k][rows] = d[k]
        if case["top"]:
            out["top_tokens"][rows] = top
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"qk_norm_rope": _exact_qk, "dropout": _exact_dropout, "token_log_probs": _exact_log_probs}[case["op"]](state)
