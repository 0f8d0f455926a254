"""Token operators on the GPU at the edges of their inputs."""

import pytest
import torch

from gpu_util import cuda, series
from polytensors_b200 import PolyTensor, _state

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
U = 2.0 ** -24          # unit roundoff of the sums
OUT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _series_mode():
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        yield


# ======================================================================================
# inputs that change between forward and backward

@pytest.mark.parametrize("n", [0, 1])
@pytest.mark.parametrize("changed", ["positions", "cos", "sin"])
def test_qk_changed_angles_are_noticed(changed, n):
    """Positions or tables changed in place between forward and backward are an error, not other angles."""
    q, k = cuda(series((2, 4, 2, 64), n, 1, F32)), cuda(series((2, 4, 1, 64), n, 2, F32))
    angle = torch.arange(20.0)[:, None] * 10000.0 ** (-torch.arange(32.0) / 32)
    plan = {"cos": angle.cos().cuda(), "sin": angle.sin().cuda(), "positions": torch.arange(4).cuda()}
    leaf = PolyTensor(tuple(q), requires_grad=True) if n else q[0].requires_grad_()
    y = PolyTensor.qk_norm_rope(leaf, PolyTensor(tuple(k)) if n else k[0], None, None, **plan)[0]
    g = series((2, 2, 4, 64), n, 3, F32)
    seed = PolyTensor(tuple(cuda(g))) if n else g[0].cuda()
    torch.autograd.grad(y, leaf, seed, retain_graph=True)
    plan[changed].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, seed)


def test_qk_angles_of_inference_mode():
    """Tables and positions made in inference mode serve training as others do."""
    q, k = (series((2, 4, h, 64), 0, h, F32)[0].cuda() for h in (2, 1))
    g = series((2, 2, 4, 64), 0, 3, F32)[0].cuda()
    angle = torch.arange(20.0)[:, None] * 10000.0 ** (-torch.arange(32.0) / 32)

    def gradient():
        leaf = q.clone().requires_grad_()
        y = PolyTensor.qk_norm_rope(leaf, k, None, None, cos, sin, positions=positions)[0]
        return torch.autograd.grad(y, leaf, g)[0]

    with torch.inference_mode():
        cos, sin, positions = angle.cos().cuda(), angle.sin().cuda(), torch.arange(4).cuda() + 3
    got = gradient()
    cos, sin, positions = (t.clone() for t in (cos, sin, positions))
    assert torch.equal(got, gradient())


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 5, 8, 12])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
def test_qk_tables_anywhere_in_their_allocation(dtype, offset):
    """Tables that start `offset` elements into an allocation (4, 8 or 16 bytes past a wider boundary) give what
    tables of their own do, forward and backward."""
    kind = F64 if dtype == F64 else F32
    angle = torch.arange(9, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=F64) / 32)
    own = [t.to(kind).cuda() for t in (angle.cos(), angle.sin())]
    moved = []
    for t in own:
        room = torch.empty(offset + t.numel(), dtype=kind, device="cuda")
        room[offset:].copy_(t.flatten())
        moved.append(room[offset:].view(t.shape))
    q, k = (cuda(series((2, 9, h, 64), 1, h, dtype)) for h in (3, 2))
    w = cuda(series((64,), 1, 5, dtype))
    gq, gk = (PolyTensor(tuple(cuda(series((2, h, 9, 64), 1, 7 + h, dtype)))) for h in (3, 2))

    def both(cos, sin):
        leaves = [PolyTensor(tuple(t), requires_grad=True) for t in (q, k, w)]
        y = PolyTensor.qk_norm_rope(leaves[0], leaves[1], leaves[2], leaves[2], cos, sin)
        d = torch.autograd.grad(y, leaves, (gq, gk))
        return [c.detach().double() for t in (*y, *d) for c in t.coeffs]

    # another vector width sums a row in another order: a few roundings of the compute type and the last one
    unit = {F32: 2.0 ** -23, F64: 2.0 ** -52, BF16: 2.0 ** -7, F16: 2.0 ** -10}[dtype]
    for a, b in zip(both(*moved), both(*own)):
        torch.testing.assert_close(a, b, rtol=64 * unit, atol=64 * unit * b.abs().max().item())


# ======================================================================================
# one word holds nearly all of a row

GAPS = (4.0, 4.7, 5.3, 6.0, 6.6, 7.1, 7.6, 7.9)


def peaked(dtype, V, base, far, scale=1.0):
    """Rows of two open words 512 groups of 16 bytes apart, the later one GAPS above the earlier; the rest at ``far``."""
    apart = 8192 // dtype.itemsize
    z = torch.full((len(GAPS), V), far, dtype=F64)
    z[:, 5] = base
    z[:, 5 + apart] = base + torch.tensor(GAPS, dtype=F64) * scale
    return z.to(dtype), 5 + apart


def check_peaked(z, top, temperature, n):
    """With m the row's largest logit and s the other word's weight, S = 1 + s is rounded at most twice (2 u), the
    weight s carries at most 20 u of its own size (difference, exponential, rescaling), and a temperature
    leaves up to 2 u more on S (the largest logit's own difference from its rounded value):
      log p:  5 u + 25 u s,        entropy: the same, 30 u |E| of E = sum p (z - m) and its last rounding,
      d entropy / dz at the word: p |log p + H| = p |E - (z - m)|, where L cancels: 2 u H + 45 u |E|,
      d log p / dz: 1 - p, p = exp(log p) with log p's bound, 4 u of the exponential, one rounding."""
    dtype, rows = z.dtype, z.shape[0]
    zeros = [torch.zeros_like(z) for _ in range(n)]
    x = torch.nn.Parameter(z.cuda()) if n == 0 else PolyTensor((z.cuda(), *[t.cuda() for t in zeros]), requires_grad=True)
    got = PolyTensor.token_log_probs(x, torch.full((rows,), top).cuda(), temperature=temperature)
    first = lambda t: (t.coeffs[0] if n else t).detach().cpu().double()  # noqa: E731
    w = z.double() / temperature
    d = w - w[:, top:top + 1]
    weight = d.exp()
    rest = weight.clone()
    rest[:, top] = 0
    s = rest.sum(1)
    logp = -torch.log1p(s)
    E = torch.where(rest > 0, rest * d, torch.zeros_like(d)).sum(1) / (1 + s)
    H = -logp - E
    room = 5 * U + 25 * U * s
    assert ((first(got.log_probs) - logp).abs() <= room).all()
    assert ((first(got.entropy) - H).abs() <= room + 30 * U * E.abs() + U * H).all()
    one = torch.ones(rows, device="cuda")
    one = PolyTensor((one,), degree=n) if n else one
    (dh,) = torch.autograd.grad(got.entropy, x, one, retain_graph=True)
    want = logp.exp() * -(logp + H) / temperature
    room = (2 * U * H + 45 * U * E.abs()) / temperature + OUT[dtype] * want.abs()
    assert ((first(dh)[:, top] - want).abs() <= room).all()
    (da,) = torch.autograd.grad(got.log_probs, x, one)
    want = -torch.expm1(logp) / temperature
    assert ((first(da)[:, top] - want).abs() <= 12 * U / temperature + OUT[dtype] * want.abs()).all()


@pytest.mark.parametrize("far", [-float("inf"), -60.0])
@pytest.mark.parametrize("dtype,V", [(F32, 32000), (F32, 5003), (BF16, 32000), (F16, 9000), (F32, 20011), (BF16, 60000),
                                     (F16, 61003)])
@pytest.mark.parametrize("n", [0, 2])
def test_log_probs_of_confident_rows(dtype, V, far, n):
    """A later word of the same thread stands 4 to 8 above the first: what is left of its log probability and
    of the entropy is of the size of the other word's weight, not of the gap."""
    check_peaked(*peaked(dtype, V, 0.375, far), 1.0, n)


@pytest.mark.parametrize("n", [0, 2])
@pytest.mark.parametrize("base", [40.3, -61.7])
def test_log_probs_of_confident_rows_at_a_temperature(base, n):
    """logit / temperature is not a float32 number; its rounding must not stand in a log probability near 0."""
    check_peaked(*peaked(F32, 5003, base, -float("inf"), scale=0.7), 0.7, n)


# ======================================================================================
# without plain_range()

def test_default_mode_takes_the_public_coefficients():
    """Outside plain_range() the operators' results and gradients are those inside it, bit for bit."""
    angle = torch.arange(9.0)[:, None] * 10000.0 ** (-torch.arange(32.0) / 32)
    cos, sin, tokens = angle.cos().cuda(), angle.sin().cuda(), torch.arange(18).cuda()
    inputs = [cuda(series(shape, 2, 20 + i, F32)) for i, shape in enumerate(((2, 9, 4, 64), (2, 9, 2, 64), (64,), (18, 300)))]
    seeds = [PolyTensor(tuple(cuda(series(shape, 2, 30 + i, F32)))) for i, shape in
             enumerate(((2, 4, 9, 64), (2, 2, 9, 64), (2, 4, 9, 64), (18,), (18,), (18, 3)))]

    def everything():
        q, k, w, z = (PolyTensor(tuple(t), requires_grad=True) for t in inputs)
        a, b = PolyTensor.qk_norm_rope(q, k, w, w, cos, sin)
        d = PolyTensor.dropout(a, 0.25, seed=3, residual=a)
        got = PolyTensor.token_log_probs(z, tokens, top=3, temperature=0.9)
        outs = (a, b, d, *got[:3])
        grads = torch.autograd.grad(outs, (q, k, w, z), seeds)
        return [c.detach() for t in (*outs, *grads) for c in t.coeffs]

    inside = everything()                  # the fixture's plain_range()
    token = _state.plain_range.set(False)
    _state.exit_plain()
    try:
        outside = everything()
    finally:
        _state.enter_plain()
        _state.plain_range.reset(token)
    assert all(torch.equal(x, y) for x, y in zip(inside, outside))
