"""64-bit reference of the token operators for their tests, on CPU, with running error bounds.

Every function takes ``sign``: -1 evaluates the definition; +1 evaluates its majorant, the same formula
with absolute values and every subtraction turned into an addition.  A computation in a type of unit
roundoff u whose longest chain has C roundings differs from the exact value by at most C u times
the majorant (first order), element by element; ``bound`` adds the final rounding to the output type.
"""

import math

import torch

from oracle import polyref as ref

UNIT = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -24, torch.float16: 2.0 ** -24}
OUT = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def bound(reference, majorant, chain, compute, out):
    """Largest admissible |got - reference|: chain roundings of the compute type along the majorant, one
    rounding to the output type, and the output type's smallest step."""
    tiny = 2.0 ** -24 if out == torch.float16 else 1e-37 if out != torch.float64 else 1e-300
    return chain * UNIT[compute] * majorant + 1.01 * OUT[out] * reference.abs() + tiny


def check(got, reference, majorant, chain, compute, out, what=""):
    """Compare planes with the bound; infinities and NaN have to stand in the same places."""
    assert len(got) == len(reference), what
    for k, (g, r, m) in enumerate(zip(got, reference, majorant)):
        assert g.dtype == out, (what, k, g.dtype)
        g = g.detach().double().cpu()
        assert g.shape == r.shape, (what, k, g.shape, r.shape)
        finite = torch.isfinite(r)
        assert torch.equal(torch.isnan(g), torch.isnan(r)), (what, k)
        assert torch.equal(g[~finite & ~torch.isnan(r)], r[~finite & ~torch.isnan(r)]), (what, k)
        over = (g - r).abs()[finite] - bound(r, m, chain, compute, out)[finite]
        assert not over.numel() or over.max() <= 0, (what, "plane", k, over.max().item())


def mul(a, b):
    return ref.cauchy(a, b)


def absolute(planes):
    return [p.abs() for p in planes]


def rsqrt(s, sign):
    y = [s[0] ** -0.5]
    for k in range(1, len(s)):
        y.append(sign * sum((2 * k - i) / (2 * k) * s[i] / s[0] * y[k - i] for i in range(1, k + 1)))
    return y


def log(s, sign):
    y = [s[0].log()]
    for k in range(1, len(s)):
        y.append(s[k] / s[0] + sign * sum((i / k) * y[i] * s[k - i] / s[0] for i in range(1, k)))
    return y


def quotient(a, b, sign):
    y = [a[0] / b[0]]
    for k in range(1, len(a)):
        y.append((a[k] + sign * sum(b[i] * y[k - i] for i in range(1, k + 1))) / b[0])
    return y


# ---------------------------------------------------------------------------------------------
# norm of heads with rotation

def rotate(x, cos, sin, interleaved, sign, back=False):
    """x (B, T, H, D), tables (B, T, 1, R/2); ``back`` turns the other way."""
    half = cos.shape[-1]
    if sign > 0:
        cos, sin = cos.abs(), sin.abs()
    elif back:
        sin = -sin
    index = torch.arange(half)
    lo, hi = (2 * index, 2 * index + 1) if interleaved else (index, index + half)
    y = x.clone()
    y[..., lo] = x[..., lo] * cos + sign * x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def _norm(X, eps, sign):
    s = [t.mean(-1, keepdim=True) for t in mul(X, X)]
    return rsqrt([s[0] + eps] + s[1:], sign)


def norm_rope(X, W, cos, sin, interleaved, eps, sign=-1):
    """y (B, H, T, D); W None or a series over (D,)."""
    if sign > 0:
        X, W = absolute(X), absolute(W) if W is not None else None
    v = mul(X, _norm(X, eps, sign))
    v = mul(v, W) if W is not None else v
    return [rotate(t, cos, sin, interleaved, sign).transpose(1, 2) for t in v]


def norm_rope_grad(X, W, G, cos, sin, interleaved, eps, sign=-1):
    """(dX, dW) of norm_rope by the formula; G (B, H, T, D)."""
    if sign > 0:
        X, W, G = absolute(X), absolute(W) if W is not None else None, absolute(G)
    g = [rotate(t.transpose(1, 2), cos, sin, interleaved, sign, back=True) for t in G]
    gy = mul(g, W) if W is not None else g
    r = _norm(X, eps, sign)
    c = [t.mean(-1, keepdim=True) for t in mul(X, gy)]
    q = mul(mul(mul(r, r), r), c)
    dx = [a + sign * b for a, b in zip(mul(gy, r), mul(X, q))]
    return dx, [t.sum((0, 1, 2)) for t in mul(g, mul(X, r))]


# ---------------------------------------------------------------------------------------------
# the generator, in Python integers

def philox4x32_10(counter, key):
    """One block of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011): four words."""
    c, k, mask = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def keep_mask(shape, p, seed, offset):
    n, mask = math.prod(shape), 0xFFFFFFFF
    words = []
    for i in range((n + 3) // 4):
        words += philox4x32_10((i & mask, i >> 32, offset & mask, offset >> 32), (seed & mask, seed >> 32))
    return torch.tensor([w >= int(p * 2.0 ** 32) for w in words[:n]], dtype=torch.bool).view(shape)


# ---------------------------------------------------------------------------------------------
# token log probabilities

def _exp_directions(x, sign):
    """exp of a series without its constant plane (its planes 1.. only)."""
    y = [torch.ones_like(x[0])]
    for k in range(1, len(x)):
        y.append(sum((i / k) * x[i] * y[k - i] for i in range(1, k + 1)))
    return y


class LogProbs:
    """All of a batch of rows: ``logp`` (R, V) planes, ``entropy`` (R,) planes, ``p`` (R, V) planes."""

    def __init__(self, Z, temperature, sign=-1):
        self.sign, self.temperature = sign, temperature
        z = [t / temperature for t in Z]
        self.open = z[0] != -math.inf
        m = z[0].amax(-1, keepdim=True)
        self.empty = (m == -math.inf)
        m = torch.where(self.empty, torch.zeros_like(m), m)
        d = [torch.where(self.open, t, torch.zeros_like(t)) for t in [z[0] - m] + z[1:]]
        w0 = torch.where(self.open, d[0].exp(), torch.zeros_like(d[0]))
        if sign > 0:
            d = absolute(d)
        w = [w0 * t for t in _exp_directions(d, sign)]
        # an underflowed weight contributes nothing
        inside = [torch.where(w0 == 0, torch.zeros_like(t), t) for t in d]
        S = [t.sum(-1, keepdim=True) for t in w]
        S[0] = torch.where(self.empty, torch.ones_like(S[0]), S[0])
        T = [t.sum(-1, keepdim=True) for t in mul(w, inside)]
        L = log(S, sign)
        if sign > 0:
            L[0] = L[0] + 1.0     # a relative error of S is an absolute one of log S
        E = quotient(T, S, sign)
        self.entropy = [(a + sign * b)[:, 0] for a, b in zip(L, E)]
        closed = -math.inf if sign < 0 else 0.0
        # z - m is one rounding of the difference; a temperature rounds z and m themselves
        first = z[0] - m if sign < 0 else (z[0] - m).abs() + (z[0].abs() + m.abs() if temperature != 1.0 else 0.0)
        self.logp = [torch.where(self.open, a + sign * b, torch.full_like(a, closed if k == 0 else 0.0))
                     for k, (a, b) in enumerate(zip([first] + d[1:], L))]
        exact0 = torch.where(self.open, (z[0] - m) - (log(S, -1)[0]), torch.full_like(m, -math.inf)).exp()
        self.p = [exact0 * t for t in _exp_directions([torch.where(self.open, t, torch.zeros_like(t))
                                                       for t in self.logp], sign)]

    def gradient(self, tokens, ga, gb, top=None, gc=None):
        """dlogits planes; ga, gb (R,) planes, gc (R, k) planes, all optional."""
        R, V = self.p[0].shape
        n = len(self.p)
        zero = [torch.zeros(R, V, dtype=torch.float64) for _ in range(n)]
        fix = absolute if self.sign > 0 else list
        special = zero
        for at, g in ((tokens[:, None], [t[:, None] for t in fix(ga)] if ga else None), (top, fix(gc) if gc else None)):
            if g is None:
                continue
            keep = self.open.gather(1, at)
            special = [s.scatter_add(1, at, torch.where(keep, t, torch.zeros_like(t))) for s, t in zip(special, g)]
        A = [s.sum(-1, keepdim=True) for s in special]
        inner = A
        if gb:
            log_plus = [torch.where(self.p[0] > 0, a + h[:, None], torch.zeros_like(a))
                        for a, h in zip(self.logp, self.entropy)]
            inner = [a + b for a, b in zip(A, mul([t[:, None] for t in fix(gb)], log_plus))]
        return [(s + self.sign * t) / self.temperature for s, t in zip(special, mul(self.p, inner))]
