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
