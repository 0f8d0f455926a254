"""Operators around a language model's tokens, on PolyTensors and ordinary tensors (no counterpart in
the reference): per-head norm with position rotation, counter-based dropout, and token log
probabilities with entropy and top alternatives.

Each is one libpolykern kernel per direction of the pass (any degree up to 15), wrapped in an
``autograd.Function`` whose backward is the series backward rule.  An ordinary tensor is a series of
degree 0; next to PolyTensors it is a constant (zero higher planes).  Unsupported inputs raise
``NotImplementedError``, wrong shapes and values ``ValueError``, indices out of range ``IndexError``.
"""

import operator
from typing import NamedTuple

import torch

from . import _kernels as K
from . import _lib
from . import _state


class TokenLogProbs(NamedTuple):
    """What ``PolyTensor.token_log_probs`` returns (the last two are None without alternatives)."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_tokens: torch.Tensor


def _degree(what, *operands):
    """The common degree of the PolyTensors among the operands (None when all are ordinary tensors)."""
    P = _state.poly_cls()
    if _state.coefficient_autograd.get():
        raise NotImplementedError(f"{what}: not available in PolyTensor.coefficient_autograd()")
    degrees = {x.degree for x in operands if isinstance(x, P)}
    if len(degrees) > 1:
        raise ValueError("PolyTensor operands must have the same degree")
    degree = degrees.pop() if degrees else None
    if degree is not None and degree >= _lib.PK_MAX_PLANES:
        raise NotImplementedError(f"{what}: degree {degree} exceeds {_lib.PK_MAX_PLANES - 1}")
    return degree


def _coeffs(x):
    """A series' planes; an ordinary tensor is its own one plane."""
    return list(x.coeffs) if isinstance(x, _state.poly_cls()) else [x]


def _full(planes, degree):
    """The planes with the zero ones of a constant filled in."""
    return planes + [torch.zeros_like(planes[0]) for _ in range((degree or 0) + 1 - len(planes))]


def _wrap(planes, degree, cls):
    return planes[0] if degree is None else cls(tuple(planes))


def _grad_planes(g, degree, cls):
    """Planes of an incoming gradient, or None for none."""
    if g is None:
        return None
    return _full(list(g.coeffs) if isinstance(g, cls) else [g], degree)


def _check_planes(what, planes, dtype=None, device=None):
    """Every plane a real floating CUDA tensor of one type (``dtype``) on one device."""
    dtype, device = dtype or planes[0].dtype, device or planes[0].device
    for p in planes:
        if not isinstance(p, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {type(p).__name__}")
        K.dtype_code(p.dtype)
        if p.dtype != dtype:
            raise NotImplementedError(f"{what}: operands of differing types ({dtype} and {p.dtype})")
        if p.device != device:
            raise ValueError(f"{what}: operands on differing devices ({device} and {p.device})")
    K._require_cuda(planes, what)


def _check_index_tensor(what, idx, device):
    if isinstance(idx, _state.poly_cls()) or not isinstance(idx, torch.Tensor):
        raise TypeError(f"{what} must be an ordinary integer tensor")
    if idx.is_floating_point() or idx.is_complex() or idx.dtype == torch.bool:
        raise TypeError(f"{what} must be integers, got {idx.dtype}")
    if idx.device != device:
        raise ValueError(f"{what} must be on {device}, got {idx.device}")


def _wants_grad(*operands):
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in operands)


def _u64(value, what):
    if isinstance(value, bool):
        raise TypeError(f"{what} must be an int, not a bool")
    value = operator.index(value)
    if not 0 <= value < 1 << 64:
        raise ValueError(f"{what} must lie in [0, 2**64), got {value}")
    return value


# ======================================================================================
# Norm of queries and keys per head with the position rotation

class _QKNormRope(torch.autograd.Function):
    """(q', k') from (q, k): one launch forward, one and the weight sums backward."""

    @staticmethod
    def forward(ctx, query, key, q_weight, k_weight, degree, plan):
        cls = _state.poly_cls()
        Q, Kp = _full(_coeffs(query), degree), _full(_coeffs(key), degree)
        QW = _coeffs(q_weight) if q_weight is not None else []
        KW = _coeffs(k_weight) if k_weight is not None else []
        q_out, k_out = K.qk_norm_rope_fwd(Q, Kp, QW, KW, plan)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*Q, *Kp, *QW, *KW)
        ctx.counts = (len(Q), len(Kp), len(QW), len(KW))
        ctx.plan, ctx.degree, ctx.cls = plan, degree, cls
        ctx.poly = [isinstance(x, cls) for x in (query, key, q_weight, k_weight)]
        return _wrap(q_out, degree, cls), _wrap(k_out, degree, cls)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        saved, groups = list(ctx.saved_tensors), []
        for n in ctx.counts:
            groups.append(saved[:n])
            del saved[:n]
        Q, Kp, QW, KW = groups
        GQ, GK = (_grad_planes(g, ctx.degree, ctx.cls) for g in (gq, gk))
        if GQ is None and GK is None:
            return (None,) * 6
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = K.qk_norm_rope_bwd(Q, Kp, QW, KW, GQ, GK, ctx.plan, need[2], need[3])
        grads = []
        for planes, poly, wanted in zip((dq, dk, dqw, dkw), ctx.poly, need):
            grads.append(None if planes is None or not wanted else ctx.cls(tuple(planes)) if poly else planes[0])
        return (*grads, None, None)


def qk_norm_rope(query, key, query_weight, key_weight, cos, sin, positions=None, eps=1e-6, interleaved=False,
                 check_indices=True):
    """Normalise queries and keys per head and rotate them by position, in one pass.

    ``query`` (B, T, H, D) and ``key`` (B, T, K, D) are the projections viewed as heads (any strides
    whose last is 1, such as slices of one packed projection).  Every head is divided by its root mean
    square, ``x * rsqrt(mean(x * x) + eps)``, and multiplied by ``query_weight`` / ``key_weight`` (D,)
    where given.  Then feature pair j of the first ``2 * cos.shape[1]`` features turns by the angle of
    its token's position: pairs (j, j + R/2), or adjacent ones with ``interleaved``; the rest pass.
    ``cos`` and ``sin`` (positions, R/2) are ordinary tables; ``positions`` (T,) or (B, T) says which
    row a token takes (default: 0 .. T-1).

    Returns the queries (B, H, T, D) and the keys (B, K, T, D), contiguous: what
    ``scaled_dot_product_attention`` reads.  Positions outside the tables raise IndexError;
    ``check_indices=False`` leaves out that check (and its wait for the GPU): such tokens then
    become NaN.
    """
    what = "qk_norm_rope"
    degree = _degree(what, query, key, query_weight, key_weight)
    for name, x in (("query", query), ("key", key)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError(f"{what}: {name} must be (batch, tokens, heads, features)")
    B, T, _, D = query.shape
    if key.shape[:2] != (B, T) or key.shape[3] != D:
        raise ValueError(f"{what}: query {tuple(query.shape)} and key {tuple(key.shape)} differ beyond their heads")
    if not 1 <= D <= 1024:
        raise NotImplementedError(f"{what}: head dimension {D} (1 to 1024)")
    planes = _coeffs(query) + _coeffs(key)
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or tuple(w.shape) != (D,):
            raise ValueError(f"{what}: {name} must have shape ({D},)")
        planes += _coeffs(w)
    _check_planes(what, planes)
    dtype, device = planes[0].dtype, planes[0].device
    for name, t in (("cos", cos), ("sin", sin)):
        if isinstance(t, _state.poly_cls()) or not isinstance(t, torch.Tensor) or not t.is_floating_point():
            raise TypeError(f"{what}: {name} must be an ordinary floating-point tensor")
        if t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] > D:
            raise ValueError(f"{what}: cos and sin must be (positions, at most {D // 2})")
        if t.device != device:
            raise ValueError(f"{what}: {name} must be on {device}, got {t.device}")
        if t.requires_grad:
            raise NotImplementedError(f"{what}: the angle tables take no gradient")
    if positions is None:
        if T > cos.shape[0]:
            raise IndexError(f"{what}: {T} tokens need {T} table rows, got {cos.shape[0]}")
    else:
        _check_index_tensor(f"{what}: positions", positions, device)
        if tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"{what}: positions must be ({T},) or ({B}, {T}), got {tuple(positions.shape)}")
        if check_indices:
            K._check_indices(positions, cos.shape[0], f"{what} position")
        positions = positions.to(torch.int64).contiguous()
    table = K.compute_dtype(dtype)
    plan = (cos.to(table).contiguous(), sin.to(table).contiguous(), positions, float(eps), bool(interleaved))
    if _wants_grad(query, key, query_weight, key_weight):
        return _QKNormRope.apply(query, key, query_weight, key_weight, degree, plan)
    with torch.no_grad():
        q_out, k_out = K.qk_norm_rope_fwd(_full(_coeffs(query), degree), _full(_coeffs(key), degree),
                                          _coeffs(query_weight) if query_weight is not None else [],
                                          _coeffs(key_weight) if key_weight is not None else [], plan)
    cls = _state.poly_cls()
    return _wrap(q_out, degree, cls), _wrap(k_out, degree, cls)


# ======================================================================================
# Dropout

class _Dropout(torch.autograd.Function):
    """y = residual + dropout(x); the gradient of x is the same dropout of y's."""

    @staticmethod
    def forward(ctx, x, residual, degree, p, seed, offset):
        cls = _state.poly_cls()
        X = _coeffs(x)
        R = _coeffs(residual) if residual is not None else []
        y = K.dropout(X, R, (degree or 0) + 1, p, seed, offset)
        ctx.set_materialize_grads(False)
        ctx.args, ctx.cls = (degree, p, seed, offset), cls
        ctx.poly = (isinstance(x, cls), isinstance(residual, cls))
        return _wrap(y, degree, cls)

    @staticmethod
    def backward(ctx, g):
        if g is None:
            return (None,) * 6
        degree, p, seed, offset = ctx.args
        is_poly = isinstance(g, ctx.cls)

        def as_input(series, poly):
            return series if poly == isinstance(series, ctx.cls) else series.value if not poly \
                else ctx.cls.constant(series, degree)

        dx = dr = None
        if ctx.needs_input_grad[0]:
            gx = as_input(g, ctx.poly[0])
            dx = _Dropout.apply(gx, None, degree if ctx.poly[0] else None, p, seed, offset)
        if ctx.needs_input_grad[1]:
            dr = as_input(g, ctx.poly[1])
        return dx, dr, None, None, None, None


def dropout(input, p, seed, offset=0, residual=None):
    """Dropout with a mask from a counter-based generator, optionally added to ``residual``:
    ``residual + keep * input / (1 - p)``, every plane under the same mask, in one pass.

    The mask is a function of ``seed`` and ``offset`` (ints in [0, 2**64)) and the element's row-major
    index alone (Philox4x32-10 with key ``seed`` and counter (index // 4, offset)); it is not stored,
    backward forms it again.  Give every dropout of a step its own ``offset`` (or ``seed``).
    ``p`` = 0 keeps everything, 1 drops everything.  ``residual`` has the input's shape and type.
    """
    what = "dropout"
    degree = _degree(what, input, residual)
    if isinstance(p, torch.Tensor) or not 0.0 <= float(p) <= 1.0:
        raise ValueError(f"{what}: p must be a number in [0, 1], got {p}")
    p, seed, offset = float(p), _u64(seed, f"{what}: seed"), _u64(offset, f"{what}: offset")
    if not isinstance(input, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(input).__name__}")
    planes = _coeffs(input)
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != input.shape:
            raise ValueError(f"{what}: the residual must have the input's shape {tuple(input.shape)}")
        planes = planes + _coeffs(residual)
    _check_planes(what, planes)
    if _wants_grad(input, residual):
        return _Dropout.apply(input, residual, degree, p, seed, offset)
    with torch.no_grad():
        y = K.dropout(_coeffs(input), _coeffs(residual) if residual is not None else [], (degree or 0) + 1, p, seed,
                      offset)
    return _wrap(y, degree, _state.poly_cls())


# ======================================================================================
# Token log probabilities

class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, degree, ignore_index, scale, top):
        cls = _state.poly_cls()
        Z = [z.reshape(-1, z.shape[-1]) for z in _coeffs(logits)]
        out = K.token_log_probs_fwd(Z, tokens.reshape(-1), ignore_index, scale, top)
        logp, entropy, top_logp, top_tokens, stats = out
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*Z, *entropy, tokens.reshape(-1), stats, *([top_tokens] if top else []))
        ctx.args, ctx.degree, ctx.cls, ctx.shape = (ignore_index, scale, top), degree, cls, logits.shape
        lead = tuple(tokens.shape)
        shaped = [_wrap([t.view(lead) for t in planes], degree, cls) for planes in (logp, entropy)]
        if not top:
            return (*shaped, None, None)
        top_tokens = top_tokens.view(*lead, top)
        ctx.mark_non_differentiable(top_tokens)
        return (*shaped, _wrap([t.view(*lead, top) for t in top_logp], degree, cls), top_tokens)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        if g_logp is None and g_entropy is None and g_top is None:
            return (None,) * 6
        n = (ctx.degree or 0) + 1
        saved = ctx.saved_tensors
        Z, entropy, tokens, stats = saved[:n], saved[n:2 * n], saved[2 * n], saved[2 * n + 1]
        ignore_index, scale, top = ctx.args
        grads = [_grad_planes(g, ctx.degree, ctx.cls) for g in (g_logp, g_entropy, g_top)]
        dz = K.token_log_probs_bwd(list(Z), tokens, ignore_index, scale, top, stats, list(entropy),
                                   saved[-1] if top else None, grads)
        return (_wrap([t.view(ctx.shape) for t in dz], ctx.degree, ctx.cls),) + (None,) * 5


def token_log_probs(logits, tokens, top=0, temperature=1.0, ignore_index=-100, check_indices=True):
    """Log probabilities of given tokens, with the distribution's entropy and its best alternatives.

    ``logits`` (..., V) is a series or an ordinary tensor, ``tokens`` (...) ordinary integers; the
    distribution is the softmax of ``logits / temperature``.  Returns ``TokenLogProbs``:
    ``log_probs`` (...), ``entropy`` (...), and with ``top`` > 0 (at most 32) ``top_log_probs`` and
    ``top_tokens`` (..., top), the largest logits in falling order (ties to the lowest index).
    Results are at least float32; the first three pass gradients to the logits.

    A logit of -inf is masked: no part in the distribution, log probability -inf.  A row with no open
    logit has entropy 0.  Rows whose token is ``ignore_index`` are not read: zeros, ``top_tokens`` -1,
    no gradient.  Other tokens outside [0, V) raise IndexError; ``check_indices=False`` leaves out that
    check (and its wait for the GPU): such rows' log probabilities then become NaN.
    """
    what = "token_log_probs"
    degree = _degree(what, logits)
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., V) with V >= 1")
    planes = _coeffs(logits)
    _check_planes(what, planes)
    _check_index_tensor(f"{what}: tokens", tokens, planes[0].device)
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: tokens {tuple(tokens.shape)} must match the logits' rows "
                         f"{tuple(logits.shape[:-1])}")
    V = logits.shape[-1]
    top = operator.index(top)
    if not 0 <= top <= min(32, V):
        raise ValueError(f"{what}: top must lie in [0, {min(32, V)}], got {top}")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"{what}: temperature must be positive and finite, got {temperature}")
    ignore_index = operator.index(ignore_index)
    if check_indices:
        K._check_indices(tokens, V, f"{what} token", ignore=ignore_index)
    tokens = tokens.to(torch.int64)
    scale = 1.0 / temperature
    if _wants_grad(logits):
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, degree, ignore_index, scale, top))
    with torch.no_grad():
        logp, entropy, top_logp, top_tokens, _ = K.token_log_probs_fwd(
            [z.reshape(-1, V) for z in planes], tokens.reshape(-1), ignore_index, scale, top)
    cls, lead = _state.poly_cls(), tuple(tokens.shape)
    shaped = [_wrap([t.view(lead) for t in x], degree, cls) for x in (logp, entropy)]
    if not top:
        return TokenLogProbs(*shaped, None, None)
    return TokenLogProbs(*shaped, _wrap([t.view(*lead, top) for t in top_logp], degree, cls),
                         top_tokens.view(*lead, top))
