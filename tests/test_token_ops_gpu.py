"""Token operators on the GPU against 64-bit references (tests/token_ref.py): per-head norm with
rotation, counter-based dropout, token log probabilities.  Each comparison is element by element with
a bound of (longest chain of roundings) x (unit roundoff) x (majorant), so no tolerance is fitted."""

import math

import pytest
import torch

import token_ref as R
from gpu_util import cuda, series
from oracle import polyref

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
COMPUTE = {F32: F32, F64: F64, BF16: F32, F16: F32}


def wide(planes):
    return [p.detach().cpu().double() for p in planes]


def variable(planes, grad=False):
    """A PolyTensor of several planes, an ordinary tensor of one."""
    from polytensors_b200 import PolyTensor

    if len(planes) > 1:
        return PolyTensor(tuple(planes), requires_grad=grad)
    return planes[0].detach().requires_grad_(grad)


def planes_of(x):
    return list(x.coeffs) if hasattr(x, "coeffs") else [x.detach()]


def api():
    from polytensors_b200 import PolyTensor

    return PolyTensor


@pytest.fixture(autouse=True)
def _series_mode():
    with api().plain_range(), api().retain_wrappers():
        yield


# ======================================================================================
# norm of heads with rotation

def tables(rows, half, dtype):
    angle = torch.arange(rows, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=F64) / max(half, 1))
    return angle.cos().to(COMPUTE[dtype]), angle.sin().to(COMPUTE[dtype])


def heads(B, T, H, K, D, n, dtype, seed=0, layout="dense"):
    """q and k planes on the GPU in one of several layouts, same values on the host."""
    if layout == "packed":          # slices of one projection
        x = cuda(series((B, T, (H + 2 * K) * D), n, seed, dtype))
        return ([p[..., :H * D].unflatten(-1, (H, D)) for p in x],
                [p[..., H * D:(H + K) * D].unflatten(-1, (K, D)) for p in x])
    if layout == "odd":             # bases one element past an aligned one
        x = cuda(series((B * T * (H + K) * D + 1,), n, seed, dtype))
        return ([p[1:1 + B * T * H * D].view(B, T, H, D) for p in x],
                [p[1 + B * T * H * D:].view(B, T, K, D) for p in x])
    if layout == "head_major":      # (B, H, T, D) memory
        q, k = cuda(series((B, H, T, D), n, seed, dtype)), cuda(series((B, K, T, D), n, seed + 1, dtype))
        return [p.transpose(1, 2) for p in q], [p.transpose(1, 2) for p in k]
    if layout == "feature_strided":
        q = cuda(series((B, T, H, 2 * D), n, seed, dtype))
        return [p[..., ::2] for p in q], cuda(series((B, T, K, D), n, seed + 1, dtype))
    return cuda(series((B, T, H, D), n, seed, dtype)), cuda(series((B, T, K, D), n, seed + 1, dtype))


def weights(D, n, dtype, seed, kind):
    if kind == "none":
        return None
    w = [0.2 * t for t in series((D,), n, seed, F64)]
    w[0] += 1.0
    return cuda([t.to(dtype) for t in w][:n + 1 if kind == "series" else 1])


def pad(w, n):
    return None if w is None else wide(w) + [torch.zeros(w[0].shape, dtype=F64)] * (n + 1 - len(w))


def check_qk(B, T, H, K, D, n, dtype, rotary=None, interleaved=False, weight="series", layout="dense", positions=None,
             train=True, eps=1e-6, rows=None):
    rotary = D - D % 2 if rotary is None else rotary
    q, k = heads(B, T, H, K, D, n, dtype, layout=layout)
    qw, kw = weights(D, n, dtype, 5, weight), weights(D, n, dtype, 6, weight)
    rows = rows or max(T, 40)
    cos, sin = tables(rows, rotary // 2, dtype)
    if positions == "shared":
        positions = (torch.arange(T) * 7 + 3) % rows
    elif positions == "own":
        positions = (torch.arange(B * T).view(B, T) * 11 + 1) % rows
    at = torch.arange(T).expand(B, T) if positions is None else positions.expand(B, T)
    angle = [t.double()[at][:, :, None] for t in (cos, sin)]
    gq, gk = cuda(series((B, H, T, D), n, 8, dtype)), cuda(series((B, K, T, D), n, 9, dtype))
    leaves = [variable(q, train), variable(k, train)] + [None if w is None else variable(w, train) for w in (qw, kw)]
    if weight == "plain" and train:
        leaves[2:] = [w[0].detach().requires_grad_() for w in (qw, kw)]
    y = api().qk_norm_rope(*leaves, cos.cuda(), sin.cuda(), positions=None if positions is None else positions.cuda(),
                           eps=eps, interleaved=interleaved)
    chain = D + 40 * (n + 1)
    c = COMPUTE[dtype]
    args = (*angle, interleaved, eps)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        assert y[i].is_contiguous()
        X, W = wide(x), pad(w, n)
        R.check(planes_of(y[i]), R.norm_rope(X, W, *args), R.norm_rope(X, W, *args, sign=1), chain, c, dtype, f"y{i}")
    if not train:
        return
    used = [v for v in leaves if v is not None]
    grads = torch.autograd.grad(y, used, (variable(gq), variable(gk)))
    for i, (x, w, g, H_) in enumerate(((q, qw, gq, H), (k, kw, gk, K))):
        X, W, G = wide(x), pad(w, n), wide(g)
        fn = (lambda a, b: R.norm_rope(a, b, *args)) if W is not None else (lambda a: R.norm_rope(a, None, *args))
        exact = polyref.series_vjp(fn, [X] if W is None else [X, W], G)
        mx, mw = R.norm_rope_grad(X, W, G, *args, sign=1)
        R.check(planes_of(grads[i]), exact[0], mx, chain + 40 * (n + 1), c, dtype, f"dx{i}")
        if W is not None:
            got = planes_of(grads[2 + i])
            R.check(got, exact[1][:len(got)], mw[:len(got)], chain + B * T * H_, c, dtype, f"dw{i}")


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("n", [0, 1, 2, 3, 4])
def test_qk_types_and_degrees(dtype, n):
    check_qk(2, 19, 6, 2, 64, n, dtype)


@pytest.mark.parametrize("n", [5, 7, 8, 11, 15])
def test_qk_high_degree(n):
    check_qk(1, 5, 3, 1, 32, n, F64)
    check_qk(1, 5, 2, 2, 16, n, F32)


@pytest.mark.parametrize("n", [5, 7, 11, 15])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_qk_high_degree_16_bit(n, dtype):
    check_qk(1, 5, 3, 1, 32, n, dtype)


@pytest.mark.parametrize("D,rotary", [(20, 20), (36, 36), (12, 4), (68, 36), (124, 124)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
def test_qk_narrow_vectors(D, rotary, interleaved, dtype):
    """Head dimensions that only vectors of four or eight bytes fit."""
    check_qk(2, 7, 3, 2, D, 1, dtype, rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("D", [1, 2, 7, 10, 33, 48, 80, 96, 128, 192, 256, 320, 520, 1024])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_qk_head_dimensions(D, dtype):
    check_qk(2, 3, 3, 1, D, 1, dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rotary", [(64, 32), (64, 0), (64, 62), (96, 24), (7, 4), (128, 64), (40, 8)])
@pytest.mark.parametrize("n,dtype", [(0, F16), (2, F32)])
def test_qk_partial_rotation(D, rotary, interleaved, n, dtype):
    check_qk(2, 5, 4, 2, D, n, dtype, rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("layout", ["packed", "odd", "head_major", "feature_strided"])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 128), (F64, 64), (F16, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_layouts(layout, dtype, D, interleaved):
    check_qk(2, 9, 4, 2, D, 1, dtype, layout=layout, interleaved=interleaved)


@pytest.mark.parametrize("weight", ["none", "plain", "series"])
@pytest.mark.parametrize("n", [0, 3])
def test_qk_weights(weight, n):
    check_qk(2, 9, 4, 2, 64, n, F32, weight=weight)


@pytest.mark.parametrize("positions", ["shared", "own"])
@pytest.mark.parametrize("T", [1, 6])
def test_qk_positions(positions, T):
    check_qk(5, T, 4, 2, 64, 1, BF16, positions=positions, rows=100)
    check_qk(5, T, 4, 2, 64, 0, F32, positions=positions, rows=100, train=False)


@pytest.mark.parametrize("B,T,H,K", [(1, 1, 1, 1), (1, 1, 32, 8), (3, 333, 1, 1), (1, 700, 5, 3)])
def test_qk_sizes(B, T, H, K):
    check_qk(B, T, H, K, 64, 1, F32)


@pytest.mark.parametrize("B,T,H,K", [(0, 4, 2, 2), (2, 0, 2, 2)])
def test_qk_empty(B, T, H, K):
    q, k = heads(B, T, H, K, 8, 1, F32)
    w = weights(8, 1, F32, 5, "series")
    leaves = [variable(q, True), variable(k, True), variable(w, True)]
    cos, sin = (t.cuda() for t in tables(4, 4, F32))
    y = api().qk_norm_rope(leaves[0], leaves[1], leaves[2], None, cos, sin)
    assert y[0].shape == (B, H, T, 8) and y[1].shape == (B, K, T, 8)
    grads = torch.autograd.grad(y, leaves, tuple(variable([torch.ones_like(p) for p in t.coeffs]) for t in y))
    assert grads[0].shape == q[0].shape and all(not t.any() for t in grads[2].coeffs)


def test_qk_zero_rows_and_no_eps():
    """A head of zeros stays zero under eps; without eps the definition gives NaN there, and only there."""
    q, k = heads(1, 3, 2, 1, 64, 1, F32)
    q[0][0, 1, 0] = 0
    cos, sin = (t.cuda() for t in tables(3, 32, F32))
    y = api().qk_norm_rope(variable(q), variable(k), None, None, cos, sin, eps=1e-6)[0]
    assert not y.coeffs[0][0, 0, 1].any() and torch.isfinite(y.coeffs[1]).all()
    y = api().qk_norm_rope(variable(q), variable(k), None, None, cos, sin, eps=0.0)[0]
    bad = torch.isnan(y.coeffs[0])
    assert bad[0, 0, 1].all() and bad.sum() == 64


def test_qk_positions_out_of_range():
    q, k = heads(2, 4, 2, 1, 64, 1, F32)
    cos, sin = (t.cuda() for t in tables(10, 32, F32))
    bad = torch.tensor([3, 10, 2, -1]).cuda()
    with pytest.raises(IndexError, match="position"):
        api().qk_norm_rope(variable(q), variable(k), None, None, cos, sin, positions=bad)
    y = api().qk_norm_rope(variable(q), variable(k), None, None, cos, sin, positions=bad, check_indices=False)
    for t in y:
        for p in t.coeffs:
            assert torch.isnan(p[:, :, [1, 3]]).all() and torch.isfinite(p[:, :, [0, 2]]).all()
    with pytest.raises(IndexError, match="table rows"):
        api().qk_norm_rope(variable(q), variable(k), None, None, cos[:3], sin[:3])


def test_qk_one_output_used():
    q, k = heads(2, 5, 4, 2, 64, 2, F32)
    w = weights(64, 2, F32, 5, "series")
    cos, sin = (t.cuda() for t in tables(5, 32, F32))
    gq, gk = cuda(series((2, 4, 5, 64), 2, 8, F32)), cuda(series((2, 2, 5, 64), 2, 9, F32))

    def grads(use):
        leaves = [variable(q, True), variable(k, True), variable(w, True), variable(w, True)]
        y = api().qk_norm_rope(*leaves, cos, sin)
        outs, seeds = zip(*[(y[i], variable((gq, gk)[i])) for i in use])
        return torch.autograd.grad(outs, leaves, seeds, allow_unused=True)

    both, only_q, only_k = grads((0, 1)), grads((0,)), grads((1,))
    assert only_q[1] is None and only_q[3] is None and only_k[0] is None and only_k[2] is None
    for one, i in ((only_q, 0), (only_q, 2), (only_k, 1), (only_k, 3)):
        # the weight sums run over another number of blocks when one side is alone
        for a, b in zip(one[i].coeffs, both[i].coeffs):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_qk_gradient_by_differences():
    """d objective / d x_(n-j) = gradient plane j (objective: sum_k <G_k, y_(n-k)>); central differences
    in float64: h^2 truncation and 2^-53 / h rounding, far below 1e-6."""
    n, h = 2, 1e-5
    q, k = heads(1, 3, 2, 1, 16, n, F64)
    w = weights(16, n, F64, 5, "series")
    cos, sin = (t.cuda() for t in tables(3, 6, F64))
    g = cuda(series((1, 2, 3, 16), n, 8, F64))
    leaf = [variable(q, True), variable(w, True)]
    y = api().qk_norm_rope(leaf[0], variable(k), leaf[1], None, cos, sin)[0]
    grads = torch.autograd.grad(y, leaf, variable(g))

    def objective(x, w_):
        out = api().qk_norm_rope(variable(x), variable(k), variable(w_), None, cos, sin)[0]
        return sum((a * b).sum() for a, b in zip(g, reversed(out.coeffs))).item()

    for which, base in enumerate((q, w)):
        for j in range(n + 1):
            v = series(tuple(base[0].shape), 0, 40 + j, F64)[0].cuda()
            moved = [[p + (s * h * v if i == n - j else 0) for i, p in enumerate(base)] for s in (1, -1)]
            up, down = (objective(*((m, w) if which == 0 else (q, m))) for m in moved)
            want = (grads[which].coeffs[j] * v).sum().item()
            assert abs((up - down) / (2 * h) - want) <= 1e-6 * max(1.0, abs(want)), (which, j)


def test_qk_broadcast_heads():
    """One key head expanded over the groups (stride 0): its gradient is the sum over them."""
    q, k = heads(2, 5, 4, 1, 64, 0, F64)
    cos, sin = (t.cuda() for t in tables(5, 32, F64))
    shared = k[0].clone().requires_grad_()
    y = api().qk_norm_rope(q[0], shared.expand(2, 5, 4, 64), None, None, cos, sin)[1]
    g = series((2, 4, 5, 64), 0, 8, F64)[0].cuda()
    (d,) = torch.autograd.grad(y, shared, g)
    dense = k[0].expand(2, 5, 4, 64).contiguous().requires_grad_()
    (e,) = torch.autograd.grad(api().qk_norm_rope(q[0], dense, None, None, cos, sin)[1], dense, g)
    torch.testing.assert_close(d, e.sum(2, keepdim=True), rtol=1e-13, atol=1e-13)


def test_qk_far_rows():
    """Rows more than 2^31 elements apart."""
    gap = (1 << 31) + 64
    base = torch.empty(gap + 64, dtype=BF16, device="cuda")
    x = base.as_strided((2, 1, 1, 64), (gap, 64, 64, 1))
    near = series((2, 1, 1, 64), 0, 3, BF16)[0].cuda()
    x.copy_(near)
    cos, sin = (t.cuda() for t in tables(1, 32, BF16))
    far = api().qk_norm_rope(x, x, None, None, cos, sin)[0]
    assert torch.equal(far, api().qk_norm_rope(near, near, None, None, cos, sin)[0])


def test_qk_repeats_and_streams():
    """Bit for bit the same on every run, and on a stream of its own."""
    q, k = heads(3, 100, 6, 2, 64, 3, F32)
    w = weights(64, 3, F32, 5, "series")
    cos, sin = (t.cuda() for t in tables(100, 32, F32))
    gq, gk = cuda(series((3, 6, 100, 64), 3, 8, F32)), cuda(series((3, 2, 100, 64), 3, 9, F32))

    def once():
        leaves = [variable(q, True), variable(k, True), variable(w, True), variable(w, True)]
        y = api().qk_norm_rope(*leaves, cos, sin)
        d = torch.autograd.grad(y, leaves, (variable(gq), variable(gk)))
        return [p.detach() for t in (*y, *d) for p in t.coeffs]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, once()):
        assert torch.equal(a, b) and torch.equal(a, c)


# ======================================================================================
# dropout

def check_dropout(shape, n, dtype, p, seed=7, offset=1, residual=True, layout="dense"):
    keep = R.keep_mask(shape, p, seed, offset)
    size = math.prod(shape)

    def make(s):
        if layout == "odd":
            return [t[1:].view(shape) for t in cuda(series((size + 1,), n, s, dtype))]
        if layout == "transposed":
            return [t.t() for t in cuda(series(shape[::-1], n, s, dtype))]
        return cuda(series(shape, n, s, dtype))

    x, res, g = make(1), make(2) if residual else None, make(3)
    leaves = [variable(x, True)] + ([variable(res, True)] if residual else [])
    y = api().dropout(leaves[0], p, seed=seed, offset=offset, residual=leaves[1] if residual else None)
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    drop = lambda t: torch.where(keep, t * scale, torch.zeros_like(t))  # noqa: E731
    want = [drop(t) for t in wide(x)]
    big = [t.abs() for t in want]
    if residual:
        want = [a + b for a, b in zip(want, wide(res))]
        big = [a + b.abs() for a, b in zip(big, wide(res))]
    # scale, product and sum: three roundings before the last one
    R.check(planes_of(y), want, big, 4, COMPUTE[dtype], dtype, "y")
    grads = torch.autograd.grad(y, leaves, variable(g))
    want = [drop(t) for t in wide(g)]
    R.check(planes_of(grads[0]), want, [t.abs() for t in want], 4, COMPUTE[dtype], dtype, "dx")
    if residual:
        for a, b in zip(planes_of(grads[1]), g):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("n", [0, 1, 3, 4, 8])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_types_and_degrees(dtype, n, residual):
    check_dropout((17, 96), n, dtype, 0.25, residual=residual)


@pytest.mark.parametrize("size", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 63, 1023, 4099])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["dense", "odd"])
def test_dropout_sizes(size, dtype, layout):
    check_dropout((size,), 1, dtype, 0.5, layout=layout)


def test_dropout_layouts():
    check_dropout((33, 20), 2, F32, 0.3, layout="transposed")
    check_dropout((33, 20), 0, F16, 0.3, layout="odd")


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.1, 0.999, 1.0])
def test_dropout_rates(p):
    check_dropout((40, 33), 1, F32, p)


@pytest.mark.parametrize("seed,offset", [(0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (1 << 40, 3), (3, 1 << 40)])
def test_dropout_seeds(seed, offset):
    check_dropout((64,), 0, F32, 0.5, seed=seed, offset=offset)


def test_dropout_known_answer():
    """The published test vector of Philox4x32-10 for counter 0 and key 0: words 0x6627e8d5, 0xe169c58d,
    0xbc57ac4c, 0x9b00dbd8, seen through the thresholds on either side of each word."""
    words = (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert R.philox4x32_10((0, 0, 0, 0), (0, 0)) == list(words)
    x = torch.ones(4, dtype=F64, device="cuda")
    for i, w in enumerate(words):
        assert api().dropout(x, w / 2.0 ** 32, seed=0)[i] != 0
        assert api().dropout(x, (w + 1) / 2.0 ** 32, seed=0)[i] == 0


def test_dropout_mask_ignores_layout_and_values():
    """The mask goes by the logical index, and a dropped element is 0 whatever stood there."""
    x = torch.full((64, 48), math.nan, device="cuda")
    keep = R.keep_mask((64, 48), 0.5, 9, 0).cuda()
    y = api().dropout(x, 0.5, seed=9)
    assert torch.equal(torch.isnan(y), keep) and not y[~keep].any()
    x = torch.ones(48, 64, device="cuda").t()
    assert torch.equal(api().dropout(x, 0.5, seed=9) != 0, keep)
    x.fill_(math.inf)
    assert torch.equal(api().dropout(x, 1.0, seed=9), torch.zeros_like(x))


def test_dropout_constants_and_degrees():
    """An ordinary residual under a series input, and an ordinary input under a series residual."""
    n, shape = 2, (9, 11)
    x, r = cuda(series(shape, n, 1, F32)), cuda(series(shape, n, 2, F32))
    y = api().dropout(variable(x), 0.3, seed=4, residual=r[0]).coeffs
    bare = api().dropout(variable(x), 0.3, seed=4).coeffs
    assert torch.equal(y[1], bare[1]) and torch.equal(y[2], bare[2]) and not torch.equal(y[0], bare[0])
    lead = x[0].clone().requires_grad_()
    series_r = variable(r, True)
    y = api().dropout(lead, 0.3, seed=4, residual=series_r)
    assert torch.equal(y.coeffs[1], r[1]) and torch.equal(y.coeffs[2], r[2])
    g = cuda(series(shape, n, 3, F32))
    dx, dr = torch.autograd.grad(y, (lead, series_r), variable(g))
    assert not hasattr(dx, "coeffs") and torch.equal(dx, api().dropout(g[0], 0.3, seed=4))
    assert all(torch.equal(a, b) for a, b in zip(dr.coeffs, g))


def test_dropout_second_derivative_and_empty():
    x = torch.randn(50, device="cuda", requires_grad=True)
    y = api().dropout(x, 0.5, seed=3)
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.sum(), x)
    keep = R.keep_mask((50,), 0.5, 3, 0).cuda()
    torch.testing.assert_close(gg, torch.where(keep, 8.0, 0.0))
    assert api().dropout(torch.empty(0, 4, device="cuda"), 0.5, seed=1).shape == (0, 4)


# ======================================================================================
# token log probabilities

def logits(rows, V, n, dtype, seed=0, std=2.0, layout="dense"):
    z = [std * t for t in series((rows, V), n, seed, F64)]
    z = cuda([t.to(dtype) for t in z])
    if layout == "columns":          # every row starts off the alignment of the last
        full = cuda([torch.zeros(rows, V + 5).to(dtype) for _ in z])
        for f, t in zip(full, z):
            f[:, 3:3 + V] = t
        return [f[:, 3:3 + V] for f in full]
    if layout == "strided":
        full = cuda([torch.zeros(rows, 2 * V).to(dtype) for _ in z])
        for f, t in zip(full, z):
            f[:, ::2] = t
        return [f[:, ::2] for f in full]
    return z


def order(z0):
    """Stable falling order, NaN first."""
    return torch.sort(z0.double().cpu(), dim=-1, descending=True, stable=True).indices


def check_log_probs(z, tokens, top=0, temperature=1.0, ignore=-100, grads="ab", seed=50):
    n, dtype = len(z) - 1, z[0].dtype
    rows, V = z[0].shape
    out = F64 if dtype == F64 else F32
    leaf = variable(z, True)
    got = api().token_log_probs(leaf, tokens.cuda(), top=top, temperature=temperature, ignore_index=ignore)
    Z = wide(z)
    exact, major = R.LogProbs(Z, temperature), R.LogProbs(Z, temperature, sign=1)
    read = tokens != ignore
    at = torch.where(read, tokens, 0)[:, None]
    row = lambda t: torch.where(read, t, torch.zeros_like(t))  # noqa: E731
    # sums of V terms by threads and their join, exponentials of arguments up to the spread of a row
    spread = torch.where(exact.open, (Z[0] / temperature).abs(), 0.0).clamp(max=200.0).amax().item()
    chain = V / 32 + 60 * (n + 1) + 4 * spread
    c = COMPUTE[dtype]
    chosen = [row(t.gather(1, at)[:, 0]) for t in exact.logp]
    R.check(planes_of(got.log_probs), chosen, [row(t.gather(1, at)[:, 0]) for t in major.logp], chain, c, out, "logp")
    R.check(planes_of(got.entropy), [row(t) for t in exact.entropy], [row(t) for t in major.entropy], chain, c, out,
            "entropy")
    best = None
    if top:
        best = order(z[0])[:, :top]
        assert torch.equal(got.top_tokens.cpu(), torch.where(read[:, None], best, -1))
        pick = lambda t: torch.where(read[:, None], t.gather(1, best), 0.0)  # noqa: E731
        R.check(planes_of(got.top_log_probs), [pick(t) for t in exact.logp], [pick(t) for t in major.logp], chain, c,
                out, "top")
    else:
        assert got.top_log_probs is None and got.top_tokens is None
    seeds = {"a": series((rows,), n, seed, out), "b": series((rows,), n, seed + 1, out),
             "c": series((rows, top), n, seed + 2, out)}
    outs, gs = [], []
    for name, t in (("a", got.log_probs), ("b", got.entropy), ("c", got.top_log_probs)):
        if name in grads:
            outs.append(t)
            gs.append(variable(cuda(seeds[name])))
    (d,) = torch.autograd.grad(outs, leaf, gs)
    zero = [torch.zeros(rows, dtype=F64)] * (n + 1)
    ga = [row(t.double()) for t in seeds["a"]] if "a" in grads else zero
    gb = [row(t.double()) for t in seeds["b"]] if "b" in grads else None
    gc = [torch.where(read[:, None], t.double(), 0.0) for t in seeds["c"]] if "c" in grads else None
    want = exact.gradient(at[:, 0], ga, gb, best, gc)
    R.check(planes_of(d), want, major.gradient(at[:, 0], ga, gb, best, gc), chain + top + 60 * (n + 1), c, dtype, "dz")
    return got, d


def random_tokens(rows, V, seed=3):
    return torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("n", [0, 1, 2, 3, 4])
def test_log_probs_types_and_degrees(dtype, n):
    check_log_probs(logits(5, 1000, n, dtype), random_tokens(5, 1000), top=3, grads="abc")


@pytest.mark.parametrize("n", [5, 7, 8, 11, 15])
def test_log_probs_high_degree(n):
    check_log_probs(logits(2, 50, n, F64, std=0.5), random_tokens(2, 50), top=2, grads="abc")
    check_log_probs(logits(2, 50, n, F32, std=0.5), random_tokens(2, 50), top=2, grads="abc")


@pytest.mark.parametrize("V", [1, 2, 3, 4, 5, 7, 8, 31, 32, 33, 127, 257, 1023, 1025, 4096, 5003, 20011])
@pytest.mark.parametrize("dtype,n", [(F32, 1), (BF16, 0), (F16, 2)])
@pytest.mark.parametrize("layout", ["dense", "columns"])
def test_log_probs_vocabularies(V, dtype, n, layout):
    check_log_probs(logits(3, V, n, dtype, layout=layout), random_tokens(3, V), top=min(V, 4), grads="abc")


@pytest.mark.parametrize("rows", [1, 2, 17, 300, 2500])
@pytest.mark.parametrize("top", [0, 2])
def test_log_probs_rows(rows, top):
    check_log_probs(logits(rows, 301, 1, F32), random_tokens(rows, 301), top=top)


@pytest.mark.parametrize("V,rows", [(60001, 1), (130003, 2), (130003, 5)])
@pytest.mark.parametrize("dtype,n", [(F32, 1), (BF16, 0)])
def test_log_probs_wide(V, rows, dtype, n):
    check_log_probs(logits(rows, V, n, dtype), random_tokens(rows, V), top=20, grads="abc")


@pytest.mark.parametrize("temperature", [0.1, 0.7, 5.0])
def test_log_probs_temperature(temperature):
    check_log_probs(logits(4, 333, 2, F32), random_tokens(4, 333), top=2, temperature=temperature, grads="abc")


@pytest.mark.parametrize("grads", ["a", "b", "c", "ac", "bc"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_gradients_apart(grads, dtype):
    check_log_probs(logits(4, 777, 2, dtype), random_tokens(4, 777), top=3, grads=grads)


def test_log_probs_strided_and_shaped():
    check_log_probs(logits(4, 100, 1, F32, layout="strided"), random_tokens(4, 100), top=2)
    z = logits(6, 50, 1, F32)
    flat = api().token_log_probs(variable(z), random_tokens(6, 50).cuda(), top=3)
    shaped = api().token_log_probs(variable([t.view(2, 3, 50) for t in z]), random_tokens(6, 50).view(2, 3).cuda(), top=3)
    assert shaped.log_probs.shape == (2, 3) and shaped.top_tokens.shape == (2, 3, 3)
    assert torch.equal(shaped.entropy.coeffs[1].flatten(), flat.entropy.coeffs[1])
    one = api().token_log_probs(z[0][0], random_tokens(6, 50)[0].cuda())
    assert one.log_probs.shape == () and torch.equal(one.log_probs, flat.log_probs.coeffs[0][0])


@pytest.mark.parametrize("dtype", [F32, BF16, F64])
@pytest.mark.parametrize("value", ["inf", "lowest"])
@pytest.mark.parametrize("V", [9, 700, 4099])
def test_log_probs_masked(dtype, value, V):
    """Masked words (also the token, also all but one), with directions at masked places that must not
    count under -inf; a row of the type's lowest value throughout is uniform."""
    z = logits(6, V, 2, dtype)
    low = -math.inf if value == "inf" else torch.finfo(dtype).min
    tokens = random_tokens(6, V)
    g = torch.Generator().manual_seed(1)
    off = torch.rand(6, V, generator=g) < 0.3
    off[1] = True
    off[1, V // 2] = False           # one open word
    off[2, tokens[2]] = True         # the token itself
    off[3, tokens[3]] = False
    if value == "lowest":
        off[4] = True
        for t in z[1:]:
            t[4] = 0
    z[0][off.cuda()] = low
    if value == "inf":
        for t in z[1:]:
            t[off.cuda()] = math.nan
    check_log_probs(z, tokens, top=5, grads="abc")


def test_log_probs_empty_rows():
    """A row with no open word: log probabilities -inf, entropy 0, alternatives in index order, no gradient."""
    z = logits(3, 40, 1, F32)
    z[0][1] = -math.inf
    got, d = check_log_probs(z, random_tokens(3, 40), top=3, grads="abc")
    assert got.log_probs.coeffs[0][1] == -math.inf and got.entropy.coeffs[0][1] == 0
    assert got.top_tokens[1].tolist() == [0, 1, 2] and not d.coeffs[0][1].any() and not d.coeffs[1][1].any()


def test_log_probs_nan_and_inf():
    """NaN and +inf make their row's results NaN, and no other row's; NaN counts as the largest logit."""
    z = logits(4, 90, 1, F32)
    z[0][1, 17] = math.nan
    z[0][2, 5] = math.inf
    leaf = variable(z, True)
    got = api().token_log_probs(leaf, torch.tensor([1, 2, 3, 4]).cuda(), top=2)
    for t in (got.log_probs, got.entropy):
        for p in t.coeffs:
            assert torch.isnan(p).tolist() == [False, True, True, False]
    assert got.top_tokens[1, 0] == 17 and got.top_tokens[2, 0] == 5
    (d,) = torch.autograd.grad(got.log_probs, leaf, variable([torch.ones(4, device="cuda")] * 1 + [torch.zeros(4, device="cuda")]))
    assert torch.isnan(d.coeffs[0]).any(1).tolist() == [False, True, True, False]


def test_log_probs_only_nan():
    z = torch.full((2, 3), math.nan, device="cuda")
    z[1] = 1.0
    got = api().token_log_probs(z, torch.tensor([0, 0]).cuda(), top=2)
    assert torch.isnan(got.entropy).tolist() == [True, False] and got.top_tokens[0].tolist() == [0, 1]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,top", [(33, 32), (32, 32), (1000, 32), (5000, 7)])
def test_log_probs_ties(dtype, V, top):
    """Few distinct values: ties go to the lowest index; +0 and -0 tie."""
    g = torch.Generator().manual_seed(4)
    z = (torch.randint(-2, 3, (5, V), generator=g).to(dtype) * 0.5)
    z[0] = torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0)
    z[1] = torch.arange(V).to(dtype)                # rising: every word is the best so far
    z[2] = -torch.arange(V).to(dtype)
    check_log_probs([z.cuda()], random_tokens(5, V), top=top, grads="abc")


def test_log_probs_large_values():
    """Logits of 1e4 and more: the row's maximum is taken out before anything is summed."""
    z = logits(4, 500, 1, F32)
    z[0] += torch.tensor([[1e4], [-1e4], [3e38], [-1e38]], device="cuda")
    z[0][2, 7] = -3e38
    z[0][3, 7] = 1e38
    check_log_probs(z, random_tokens(4, 500), top=1)


def test_log_probs_ignored_rows():
    z = logits(5, 64, 1, F32)
    z[0][1] = math.nan               # an ignored row is not read
    tokens = random_tokens(5, 64)
    tokens[1] = tokens[3] = -100
    for t in z:
        t[3] = 0
    leaf = variable(z, True)
    got = api().token_log_probs(leaf, tokens.cuda(), top=2)
    for p in (*got.log_probs.coeffs, *got.entropy.coeffs):
        assert not p[[1, 3]].any() and torch.isfinite(p).all()
    assert (got.top_tokens[[1, 3]] == -1).all() and (got.top_tokens[[0, 2, 4]] >= 0).all()
    ones = lambda t: variable([torch.ones_like(p) for p in t.coeffs])  # noqa: E731
    (d,) = torch.autograd.grad((got.log_probs, got.entropy), leaf, (ones(got.log_probs), ones(got.entropy)))
    assert all(not p[[1, 3]].any() and p[[0, 2, 4]].any() for p in d.coeffs)
    tokens[3] = 7
    check_log_probs([torch.nan_to_num(t) for t in z], torch.where(tokens < 0, 63, tokens), ignore=63, top=1)


def test_log_probs_tokens_out_of_range():
    z = logits(3, 20, 1, F32)
    bad = torch.tensor([3, 20, -1]).cuda()
    with pytest.raises(IndexError, match="token"):
        api().token_log_probs(variable(z), bad)
    leaf = variable(z, True)
    got = api().token_log_probs(leaf, bad, check_indices=False)
    assert torch.isnan(got.log_probs.coeffs[0]).tolist() == [False, True, True]
    assert torch.isfinite(got.entropy.coeffs[1]).all()
    (d,) = torch.autograd.grad(got.log_probs, leaf, variable([torch.ones(3, device="cuda"), torch.zeros(3, device="cuda")]))
    assert torch.isnan(d.coeffs[0]).all(1).tolist() == [False, True, True]


def test_log_probs_broadcast_rows():
    """One row of logits for several tokens (row stride 0), and tokens of a narrower integer type."""
    z = logits(1, 333, 0, F64)[0]
    one = z.clone().requires_grad_()
    tokens = random_tokens(4, 333).cuda()
    got = api().token_log_probs(one.expand(4, 333), tokens.to(torch.int32), top=2)
    want = api().token_log_probs(z.expand(4, 333).contiguous(), tokens, top=2)
    assert torch.equal(got.log_probs, want.log_probs) and torch.equal(got.top_tokens, want.top_tokens)
    (d,) = torch.autograd.grad(got.log_probs.sum(), one)
    expected = torch.zeros(333, dtype=F64, device="cuda").index_add_(0, tokens, torch.ones(4, dtype=F64, device="cuda"))
    torch.testing.assert_close(d[0], expected - 4 * torch.softmax(z[0], -1), rtol=1e-12, atol=1e-14)


def test_log_probs_changed_logits_are_noticed():
    """Logits changed in place between forward and backward are an error, not a wrong gradient."""
    z = logits(2, 50, 1, F32)
    leaf = variable(z, True)
    got = api().token_log_probs(leaf, random_tokens(2, 50).cuda())
    z[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(got.entropy, leaf, variable([torch.ones(2, device="cuda")] + [torch.zeros(2, device="cuda")]))


def test_log_probs_no_rows():
    leaf = variable([torch.empty(0, 7, device="cuda"), torch.empty(0, 7, device="cuda")], True)
    got = api().token_log_probs(leaf, torch.empty(0, dtype=torch.int64, device="cuda"), top=2)
    assert got.log_probs.shape == (0,) and got.top_tokens.shape == (0, 2)
    zero = variable([torch.empty(0, device="cuda")] * 1 + [torch.empty(0, device="cuda")])
    assert torch.autograd.grad(got.entropy, leaf, zero)[0].shape == (0, 7)


def test_log_probs_far_rows():
    """Rows more than 2^31 elements apart."""
    gap, V = (1 << 31) + 8, 1000
    base = torch.empty(gap + V, dtype=BF16, device="cuda")
    z = base.as_strided((2, V), (gap, 1))
    near = logits(2, V, 0, BF16)[0]
    z.copy_(near)
    tokens = random_tokens(2, V).cuda()
    far, want = api().token_log_probs(z, tokens, top=3), api().token_log_probs(near, tokens, top=3)
    assert torch.equal(far.entropy, want.entropy) and torch.equal(far.top_tokens, want.top_tokens)
    assert torch.equal(far.log_probs, want.log_probs)


def test_log_probs_repeats_and_streams():
    z, tokens = logits(3, 32000, 1, F32), random_tokens(3, 32000).cuda()

    def once():
        leaf = variable(z, True)
        got = api().token_log_probs(leaf, tokens, top=5)
        d = torch.autograd.grad((got.log_probs, got.entropy), leaf,
                                (variable([p.detach() for p in got.entropy.coeffs]),
                                 variable([p.detach() for p in got.log_probs.coeffs])))[0]
        return [p.detach() for t in (got.log_probs, got.entropy, got.top_log_probs, d) for p in t.coeffs]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_log_probs_gradient_by_differences():
    """Central differences in float64 of sum_k <G_k, y_(n-k)> over log probability, entropy and the best
    alternative (alone by a clear margin): far below 1e-6."""
    n, V, h = 2, 12, 1e-5
    z = logits(1, V, n, F64, std=1.0)
    z[0][0, 5] += 4.0
    tokens = torch.tensor([3]).cuda()
    g = [cuda(series(s, n, 60 + i, F64)) for i, s in enumerate(((1,), (1,), (1, 1)))]

    def results(x):
        return api().token_log_probs(x, tokens, top=1, temperature=0.8)[:3]

    leaf = variable(z, True)
    (d,) = torch.autograd.grad(results(leaf), leaf, [variable(t) for t in g])

    def objective(planes):
        return sum((a * b).sum() for t, gs in zip(results(variable(planes)), g)
                   for a, b in zip(gs, reversed(t.coeffs))).item()

    for j in range(n + 1):
        for i in range(V):
            step = torch.zeros(1, V, dtype=F64, device="cuda")
            step[0, i] = h
            up, down = (objective([p + (s * step if k == n - j else 0) for k, p in enumerate(z)]) for s in (1, -1))
            want = d.coeffs[j][0, i].item()
            assert abs((up - down) / (2 * h) - want) <= 1e-6 * max(1.0, abs(want)), (j, i)


# ======================================================================================
# all of them

def test_calls_in_a_graph():
    """The forward calls of a decoding step captured in a CUDA graph and replayed on new inputs."""
    q, k = heads(3, 1, 4, 2, 64, 0, BF16)
    cos, sin = (t.cuda() for t in tables(50, 32, BF16))
    positions = torch.tensor([[3], [40], [7]]).cuda()
    z, tokens = logits(3, 5000, 0, BF16)[0], random_tokens(3, 5000).cuda()

    def step():
        a, b = api().qk_norm_rope(q[0], k[0], None, None, cos, sin, positions=positions, check_indices=False)
        got = api().token_log_probs(z, tokens, top=3, check_indices=False)
        return [a, b, api().dropout(a, 0.5, seed=2), got.log_probs, got.entropy, got.top_log_probs, got.top_tokens]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in (q[0], z):
        t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(12)).to(t.dtype))
    positions.add_(5)
    tokens.copy_(random_tokens(3, 5000, seed=9))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_launches_per_call():
    """One launch forward; backward one, and one more for the weights' sums."""
    from polytensors_b200 import _lib

    q, k = heads(2, 9, 4, 2, 64, 1, F32)
    w = weights(64, 1, F32, 5, "series")
    cos, sin = (t.cuda() for t in tables(9, 32, F32))
    leaves = [variable(q, True), variable(k, True), variable(w, True), variable(w, True)]
    counts = []

    def counted(fn):
        _lib.launch_count(reset=True)
        out = fn()
        counts.append(_lib.launch_count())
        return out

    y = counted(lambda: api().qk_norm_rope(*leaves, cos, sin))
    seeds = tuple(variable([torch.ones_like(p) for p in t.coeffs]) for t in y)
    counted(lambda: torch.autograd.grad(y, leaves, seeds))
    z = variable(logits(3, 100, 1, F32), True)
    got = counted(lambda: api().token_log_probs(z, random_tokens(3, 100).cuda(), top=2, check_indices=False))
    ones = variable([torch.ones(3, device="cuda"), torch.zeros(3, device="cuda")])
    counted(lambda: torch.autograd.grad(got.entropy, z, ones))
    d = counted(lambda: api().dropout(z, 0.5, seed=1))
    counted(lambda: torch.autograd.grad(d, z, variable([torch.ones_like(p) for p in d.coeffs])))
    assert counts == [1, 2, 1, 1, 1, 1]
