"""Token operators on the GPU at the edges of their inputs."""

import pytest
import torch

from gpu_util import cuda, series
from polytensors_b200 import PolyTensor

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


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
