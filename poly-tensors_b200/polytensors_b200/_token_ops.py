"""Operators around a language model's tokens, on PolyTensors and ordinary tensors (no counterpart in
the reference): per-head norm with position rotation, counter-based dropout, and token log
probabilities with entropy and top alternatives.

Each is one libpolykern kernel per direction of the pass (any degree up to 15), wrapped in an
``autograd.Function`` whose backward is the series backward rule.  An ordinary tensor is a series of
degree 0; next to PolyTensors it is a constant (zero higher planes).  Unsupported inputs raise
``NotImplementedError``, wrong shapes and values ``ValueError``, indices out of range ``IndexError``.
"""

import functools
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


def _public(fn):
    """A public call: runs on its tensors' GPU and with PolyTensor's interception off, so that reading an
    operand's attributes costs no Python call (the operators handle the planes themselves)."""
    on_gpu = K.on_own_device(fn)

    @functools.wraps(fn)
    def call(*args, **kwargs):
        with torch._C.DisableTorchFunctionSubclass():
            return on_gpu(*args, **kwargs)

    return call


def _operands(what, *operands):
    """The planes of each operand ([] for None; an ordinary tensor is its own one plane), the common degree
    of the PolyTensors among them (None without any), and the PolyTensor class.  All planes are real
    floating-point tensors of one type on one device."""
    cls = _state.poly_cls()
    if _state.coefficient_autograd.get():
        raise NotImplementedError(f"{what}: not available in PolyTensor.coefficient_autograd()")
    planes, degree, dtype, device = [], None, None, None
    for x in operands:
        if x is None:
            planes.append([])
            continue
        if isinstance(x, cls):
            if degree is not None and x.degree != degree:
                raise ValueError("PolyTensor operands must have the same degree")
            degree, own = x.degree, list(x.coeffs)
        elif isinstance(x, torch.Tensor):
            own = [x]
        else:
            raise TypeError(f"{what}: expected tensors, got {type(x).__name__}")
        for p in own:
            if dtype is None:
                dtype, device = p.dtype, p.device
                K.dtype_code(dtype)
            elif p.dtype != dtype:
                raise NotImplementedError(f"{what}: operands of differing types ({dtype} and {p.dtype})")
            elif p.device != device:
                raise ValueError(f"{what}: operands on differing devices ({device} and {p.device})")
        planes.append(own)
    if degree is not None and degree >= _lib.PK_MAX_PLANES:
        raise NotImplementedError(f"{what}: degree {degree} exceeds {_lib.PK_MAX_PLANES - 1}")
    return planes, degree, cls


def _require_cuda(what, tensor):
    if not tensor.is_cuda:
        K._require_cuda([tensor], what)


def _full(planes, degree):
    """The planes with the zero ones of a constant filled in."""
    missing = (degree or 0) + 1 - len(planes)
    return planes + [torch.zeros_like(planes[0]) for _ in range(missing)] if missing else planes


def _wrap(planes, degree, cls):
    """A kernel's output planes as the caller's kind of variable."""
    if degree is None:
        return planes[0]
    return cls._of(tuple(planes))


def _grad_planes(g, degree, cls):
    """Planes of an incoming gradient, or None for none."""
    if g is None:
        return None
    return _full(list(g.coeffs) if isinstance(g, cls) else [g], degree)


def _check_index_tensor(what, idx, device, cls):
    if isinstance(idx, cls) or not isinstance(idx, torch.Tensor):
        raise TypeError(f"{what} must be an ordinary integer tensor")
    if idx.is_floating_point() or idx.is_complex() or idx.dtype == torch.bool:
        raise TypeError(f"{what} must be integers, got {idx.dtype}")
    if idx.device != device:
        raise ValueError(f"{what} must be on {device}, got {idx.device}")


def _wants_grad(*operands):
    if torch.is_grad_enabled():
        for x in operands:
            if x is not None and x.requires_grad:
                return True
    return False


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
    def forward(ctx, query, key, q_weight, k_weight, planes, degree, cls, plan):
        q_out, k_out = K.qk_norm_rope_fwd(*planes, plan)
        ctx.set_materialize_grads(False)
        # the angles' tensors may be the caller's own: saved, so that a change before backward is noticed
        angles, ctx.options = [t for t in plan[:3] if t is not None], plan[3:]
        ctx.save_for_backward(*planes[0], *planes[1], *planes[2], *planes[3], *angles)
        ctx.counts = [len(p) for p in planes]
        ctx.degree, ctx.cls = degree, cls
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
        cos, sin, *positions = saved
        plan = (cos, sin, positions[0] if positions else None, *ctx.options)
        GQ, GK = (_grad_planes(g, ctx.degree, ctx.cls) for g in (gq, gk))
        if GQ is None and GK is None:
            return (None,) * 8
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = K.qk_norm_rope_bwd(Q, Kp, QW, KW, GQ, GK, plan, need[2], need[3])
        grads = []
        for planes, poly, wanted in zip((dq, dk, dqw, dkw), ctx.poly, need):
            grads.append(None if planes is None or not wanted else _wrap(planes, ctx.degree if poly else None, ctx.cls))
        return (*grads, None, None, None, None)


@_public
def qk_norm_rope(query, key, query_weight, key_weight, cos, sin, positions=None, eps=1e-6, interleaved=False,
                 check_indices=True):
    """Normalise queries and keys per head and rotate them by position, in one pass.

    ``query`` (B, T, H, D) and ``key`` (B, T, K, D) are the projections viewed as heads (any strides
    whose last is 1, such as slices of one packed projection).  Every head is divided by its root mean
    square, ``x * rsqrt(mean(x * x) + eps)``, and multiplied by ``query_weight`` / ``key_weight`` (D,)
    where given.  Then feature pair j of the first ``2 * cos.shape[1]`` features turns by the angle of
    its token's position: pairs (j, j + R/2), or adjacent ones with ``interleaved``; the rest pass.
    ``cos`` and ``sin`` (positions, R/2) are ordinary tables; ``positions`` (T,) or (B, T) says which
    row a token takes (default: 0 .. T-1).  Tables and positions that are used as they are (no conversion) and
    change in place before backward are an error there.

    Returns the queries (B, H, T, D) and the keys (B, K, T, D), contiguous: what
    ``scaled_dot_product_attention`` reads.  Positions outside the tables raise IndexError;
    ``check_indices=False`` leaves out that check (and its wait for the GPU): such tokens then
    become NaN.
    """
    what = "qk_norm_rope"
    for name, x in (("query", query), ("key", key)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError(f"{what}: {name} must be (batch, tokens, heads, features)")
    planes, degree, cls = _operands(what, query, key, query_weight, key_weight)
    first = planes[0][0]
    device, (B, T, _, D) = first.device, first.shape
    KB, KT, _, KD = planes[1][0].shape
    if KB != B or KT != T or KD != D:
        raise ValueError(f"{what}: query {tuple(query.shape)} and key {tuple(key.shape)} differ beyond their heads")
    if not 1 <= D <= 1024:
        raise NotImplementedError(f"{what}: head dimension {D} (1 to 1024)")
    for name, w in (("query_weight", planes[2]), ("key_weight", planes[3])):
        if w and w[0].shape != (D,):
            raise ValueError(f"{what}: {name} must have shape ({D},)")
    _require_cuda(what, first)
    table = K.compute_dtype(first.dtype)
    tables = []
    for name, t in (("cos", cos), ("sin", sin)):
        if isinstance(t, cls) or not isinstance(t, torch.Tensor) or not t.is_floating_point():
            raise TypeError(f"{what}: {name} must be an ordinary floating-point tensor")
        if t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] > D:
            raise ValueError(f"{what}: cos and sin must be (positions, at most {D // 2})")
        if t.device != device:
            raise ValueError(f"{what}: {name} must be on {device}, got {t.device}")
        if t.requires_grad:
            raise NotImplementedError(f"{what}: the angle tables take no gradient")
        tables.append(t if t.dtype == table and t.is_contiguous() else t.to(table).contiguous())
    if positions is None:
        if T > cos.shape[0]:
            raise IndexError(f"{what}: {T} tokens need {T} table rows, got {cos.shape[0]}")
    else:
        _check_index_tensor(f"{what}: positions", positions, device, cls)
        if positions.shape != (T,) and positions.shape != (B, T):
            raise ValueError(f"{what}: positions must be ({T},) or ({B}, {T}), got {tuple(positions.shape)}")
        if check_indices:
            K._check_indices(positions, cos.shape[0], f"{what} position")
        if positions.dtype != torch.int64 or not positions.is_contiguous():
            positions = positions.to(torch.int64).contiguous()
    plan = (*tables, positions, float(eps), bool(interleaved))
    planes = [_full(planes[0], degree), _full(planes[1], degree), planes[2], planes[3]]
    if _wants_grad(query, key, query_weight, key_weight):
        # tensors made in inference mode cannot be saved: a copy can
        plan = (*[t.clone() if t is not None and t.is_inference() else t for t in plan[:3]], *plan[3:])
        return _QKNormRope.apply(query, key, query_weight, key_weight, planes, degree, cls, plan)
    q_out, k_out = K.qk_norm_rope_fwd(*planes, plan)
    return _wrap(q_out, degree, cls), _wrap(k_out, degree, cls)


# ======================================================================================
# Dropout

class _Dropout(torch.autograd.Function):
    """y = residual + dropout(x); the gradient of x is the same dropout of y's."""

    @staticmethod
    def forward(ctx, x, residual, planes, degree, cls, p, seed, offset):
        y = K.dropout(*planes, (degree or 0) + 1, p, seed, offset)
        ctx.set_materialize_grads(False)
        ctx.args = (degree, cls, p, seed, offset)
        ctx.poly = (isinstance(x, cls), isinstance(residual, cls))
        return _wrap(y, degree, cls)

    @staticmethod
    def backward(ctx, g):
        if g is None:
            return (None,) * 8
        degree, cls, p, seed, offset = ctx.args

        def as_input(poly):
            """The gradient for an input that is a series, or an ordinary tensor (its constant plane)."""
            if poly == isinstance(g, cls):
                return g
            return cls.constant(g, degree) if poly else g.coeffs[0]

        dx = None
        if ctx.needs_input_grad[0]:
            gx, own = as_input(ctx.poly[0]), degree if ctx.poly[0] else None
            planes = [list(gx.coeffs) if ctx.poly[0] else [gx], []]
            if torch.is_grad_enabled():
                dx = _Dropout.apply(gx, None, planes, own, cls, p, seed, offset)
            else:
                dx = _wrap(K.dropout(*planes, (own or 0) + 1, p, seed, offset), own, cls)
        dr = as_input(ctx.poly[1]) if ctx.needs_input_grad[1] else None
        return dx, dr, None, None, None, None, None, None


@_public
def dropout(input, p, seed, offset=0, residual=None):
    """Dropout with a mask from a counter-based generator, optionally added to ``residual``:
    ``residual + keep * input / (1 - p)``, every plane under the same mask, in one pass.

    The mask is a function of ``seed`` and ``offset`` (ints in [0, 2**64)) and the element's row-major
    index alone (Philox4x32-10 with key ``seed`` and counter (index // 4, offset)); it is not stored,
    backward forms it again.  Give every dropout of a step its own ``offset`` (or ``seed``).  Both are part of
    the launch: replays of a captured graph repeat the mask.  ``F.dropout`` is another generator (torch's).
    ``p`` = 0 keeps everything, 1 drops everything.  ``residual`` has the input's shape and type.
    """
    what = "dropout"
    if isinstance(p, torch.Tensor) or not 0.0 <= float(p) <= 1.0:
        raise ValueError(f"{what}: p must be a number in [0, 1], got {p}")
    p, seed, offset = float(p), _u64(seed, f"{what}: seed"), _u64(offset, f"{what}: offset")
    if residual is not None and (not isinstance(residual, torch.Tensor) or not isinstance(input, torch.Tensor)
                                 or residual.shape != input.shape):
        raise ValueError(f"{what}: the residual must have the input's shape")
    planes, degree, cls = _operands(what, input, residual)
    if not planes[0]:
        raise TypeError(f"{what}: expected a tensor, got None")
    _require_cuda(what, planes[0][0])
    if _wants_grad(input, residual):
        return _Dropout.apply(input, residual, planes, degree, cls, p, seed, offset)
    y = K.dropout(*planes, (degree or 0) + 1, p, seed, offset)
    return _wrap(y, degree, cls)


# ======================================================================================
# Token log probabilities

def _shaped(out, lead, top, degree, cls):
    """The kernel's flat results as the caller sees them."""
    logp, entropy, top_logp, top_tokens = out[:4]
    if len(lead) != 1:
        logp, entropy = ([t.view(lead) for t in planes] for planes in (logp, entropy))
        if top:
            top_logp, top_tokens = [t.view(*lead, top) for t in top_logp], top_tokens.view(*lead, top)
    return (_wrap(logp, degree, cls), _wrap(entropy, degree, cls),
            _wrap(top_logp, degree, cls) if top else None, top_tokens)


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, planes, tokens, lead, degree, cls, ignore_index, scale, top):
        out = K.token_log_probs_fwd(planes, tokens, ignore_index, scale, top)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*planes, *out[1], tokens, out[4], *([out[3]] if top else []))
        ctx.args, ctx.degree, ctx.cls, ctx.lead = (ignore_index, scale, top), degree, cls, lead
        results = _shaped(out, lead, top, degree, cls)
        if top:
            ctx.mark_non_differentiable(results[3])
        return results

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        if g_logp is None and g_entropy is None and g_top is None:
            return (None,) * 9
        n = (ctx.degree or 0) + 1
        saved = ctx.saved_tensors
        Z, entropy, tokens, stats = saved[:n], saved[n:2 * n], saved[2 * n], saved[2 * n + 1]
        ignore_index, scale, top = ctx.args
        grads = [_grad_planes(g, ctx.degree, ctx.cls) for g in (g_logp, g_entropy, g_top)]
        dz = K.token_log_probs_bwd(list(Z), tokens, ignore_index, scale, top, stats, list(entropy),
                                   saved[-1] if top else None, grads)
        if len(ctx.lead) != 1:
            dz = [t.view(*ctx.lead, t.shape[-1]) for t in dz]
        return (_wrap(dz, ctx.degree, ctx.cls),) + (None,) * 8


@_public
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
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., V) with V >= 1")
    (planes,), degree, cls = _operands(what, logits)
    first = planes[0]
    _require_cuda(what, first)
    _check_index_tensor(f"{what}: tokens", tokens, first.device, cls)
    shape, lead = first.shape, tuple(tokens.shape)
    if lead != tuple(shape[:-1]):
        raise ValueError(f"{what}: tokens {lead} must match the logits' rows {tuple(shape[:-1])}")
    V = shape[-1]
    top = operator.index(top)
    if not 0 <= top <= min(32, V):
        raise ValueError(f"{what}: top must lie in [0, {min(32, V)}], got {top}")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"{what}: temperature must be positive and finite, got {temperature}")
    ignore_index = operator.index(ignore_index)
    if check_indices:
        K._check_indices(tokens, V, f"{what} token", ignore=ignore_index)
    if tokens.dtype != torch.int64:
        tokens = tokens.to(torch.int64)
    if len(lead) != 1:
        planes, tokens = [z.reshape(-1, V) for z in planes], tokens.reshape(-1)
    scale = 1.0 / temperature
    if _wants_grad(logits):
        return TokenLogProbs(*_TokenLogProbs.apply(logits, planes, tokens, lead, degree, cls, ignore_index, scale, top))
    out = K.token_log_probs_fwd(planes, tokens, ignore_index, scale, top)
    return TokenLogProbs(*_shaped(out, lead, top, degree, cls))
