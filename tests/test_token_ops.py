"""Refusals of the token operators that need no GPU: argument checks of the public calls and of the C
entry points (nothing is launched)."""

import ctypes

import pytest
import torch

from polytensors_b200 import PolyTensor, _lib


def head(B=1, T=2, H=2, D=8, dtype=torch.float32):
    return torch.zeros(B, T, H, D, dtype=dtype)


TABLE = torch.zeros(4, 4)


def test_qk_refusals():
    call = PolyTensor.qk_norm_rope
    with pytest.raises(NotImplementedError, match="CUDA"):
        call(head(), head(), None, None, TABLE, TABLE)
    with pytest.raises(ValueError, match="batch, tokens, heads, features"):
        call(torch.zeros(2, 8), head(), None, None, TABLE, TABLE)
    with pytest.raises(ValueError, match="beyond their heads"):
        call(head(), head(T=3), None, None, TABLE, TABLE)
    with pytest.raises(ValueError, match="query_weight"):
        call(head(), head(), torch.ones(7), None, TABLE, TABLE)
    with pytest.raises(NotImplementedError, match="head dimension"):
        call(head(D=1026), head(D=1026), None, None, TABLE, TABLE)
    with pytest.raises(NotImplementedError, match="differing types"):
        call(head(), head(dtype=torch.bfloat16), None, None, TABLE, TABLE)
    with pytest.raises(NotImplementedError, match="not supported"):
        call(head(dtype=torch.complex64), head(), None, None, TABLE, TABLE)
    with pytest.raises(ValueError, match="same degree"):
        call(PolyTensor((head(),), degree=1), PolyTensor((head(),), degree=2), None, None, TABLE, TABLE)
    with pytest.raises(NotImplementedError, match="degree"):
        call(PolyTensor((head(),), degree=16), head(), None, None, TABLE, TABLE)
    with PolyTensor.coefficient_autograd(), pytest.raises(NotImplementedError, match="coefficient_autograd"):
        call(head(), head(), None, None, TABLE, TABLE)


def test_dropout_refusals():
    call, x = PolyTensor.dropout, torch.zeros(3)
    with pytest.raises(NotImplementedError, match="CUDA"):
        call(x, 0.5, seed=1)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="p must"):
            call(x, p, seed=1)
    with pytest.raises(ValueError, match="seed"):
        call(x, 0.5, seed=-1)
    with pytest.raises(ValueError, match="offset"):
        call(x, 0.5, seed=1, offset=1 << 64)
    with pytest.raises(TypeError):
        call(x, 0.5, seed=1.5)
    with pytest.raises(TypeError):
        call(x, 0.5, seed=True)
    with pytest.raises(ValueError, match="residual"):
        call(x, 0.5, seed=1, residual=torch.zeros(4))
    with pytest.raises(NotImplementedError, match="differing types"):
        call(x, 0.5, seed=1, residual=torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ValueError, match="same degree"):
        call(PolyTensor((x,), degree=1), 0.5, seed=1, residual=PolyTensor((x,), degree=2))


def test_token_log_probs_refusals():
    call, z, t = PolyTensor.token_log_probs, torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="CUDA"):
        call(z, t)
    with pytest.raises(ValueError, match="V >= 1"):
        call(torch.zeros(2, 0), t)
    with pytest.raises(NotImplementedError, match="not supported"):
        call(torch.zeros(2, 5, dtype=torch.int32), t)


def pointers(n, base=0x10000):
    arr = (ctypes.c_void_p * n)(*[base * (i + 1) for i in range(n)])
    return ctypes.cast(arr, ctypes.POINTER(ctypes.c_void_p)), arr


def test_c_entry_refusals():
    lib = _lib.load()
    p, keep = pointers(2)
    qk = lambda dtype=0, degree=1, D=8, rotary=8, q=p, nw=0: lib.pk_qk_norm_rope_fwd(  # noqa: E731
        dtype, degree, 1, 1, 1, 1, D, rotary, 0, q, 8, 8, 8, p, 8, 8, 8, p, nw, p, 0, 0x1000, 0x1000, 4, None, 0, 1e-6,
        p, p, None)
    assert qk(dtype=4) == -2 and qk(degree=16) == -2 and qk(degree=-1) == -2 and qk(D=1025) == -2
    assert qk(rotary=7) == -1 and qk(rotary=10) == -1 and qk(q=None) == -1 and qk(nw=3) == -1
    assert lib.pk_qk_norm_rope_bwd(0, 1, 1, 1, 1, 1, 8, 8, 0, p, 8, 8, 8, p, 8, 8, 8, p, 2, p, 2, 0x1000, 0x1000, 4,
                                   None, 0, 1e-6, p, 8, 8, 8, p, 8, 8, 8, p, p, p, p, None, 0, None) == -4
    drop = lambda degree=1, n=4, nx=2, threshold=0, x=p: lib.pk_dropout(  # noqa: E731
        0, degree, n, x, nx, None, 0, threshold, 1.0, 0, 0, p, None)
    assert drop(degree=16) == -2 and drop(n=-1) == -1 and drop(nx=3) == -1 and drop(nx=0) == -1
    assert drop(threshold=(1 << 32) + 1) == -1 and drop(x=None) == -1 and drop(n=0) == 0
    assert lib.pk_dropout(4, 1, 4, p, 2, None, 0, 0, 1.0, 0, 0, p, None) == -2
    logp = lambda dtype=0, degree=1, rows=1, cols=5, top=0, z=p: lib.pk_token_log_probs_fwd(  # noqa: E731
        dtype, degree, rows, cols, z, cols, 0x1000, -100, 1.0, top, p, p, p, 0x1000, 0x1000, None)
    assert logp(dtype=4) == -2 and logp(degree=16) == -2 and logp(cols=0) == -1 and logp(rows=-1) == -1
    assert logp(top=33, cols=50) == -1 and logp(top=6) == -1 and logp(z=None) == -1 and logp(rows=0) == 0
    assert "null" in _lib.last_error() or _lib.last_error()


def test_constructor_separates_planes_of_one_buffer():
    """Planes that are views of one buffer, overlapping or not, get memory of their own; separate ones stay."""
    buffer = torch.randn(4, 6)
    x = PolyTensor((buffer[0], buffer[1], buffer[1]))
    assert x.coeffs[0].data_ptr() == buffer[0].data_ptr()
    assert len({c.untyped_storage().data_ptr() for c in x.coeffs}) == 3
    apart = (torch.randn(6), torch.randn(6))
    assert all(a is b for a, b in zip(PolyTensor(apart).coeffs, apart))
    with pytest.raises(TypeError):
        PolyTensor((torch.randn(3), "x"))


@pytest.mark.parametrize("same", [False, True])
def test_constructor_inside_function_transforms(same):
    """torch.func's tensors have no storage to compare; series of them are built as of any others."""
    x, y = torch.randn(3, 4), torch.randn(3, 4)
    build = lambda a, b: PolyTensor((a, a if same else b)).coeffs[1] * 2  # noqa: E731
    want = 2 * (x if same else y)
    assert torch.equal(torch.func.vmap(build)(x, y), want)
    assert torch.equal(torch.func.vmap(torch.func.vmap(build))(x, y), want)
    dx, dy = torch.func.grad(lambda a, b: build(a, b).sum(), argnums=(0, 1))(x, y)
    assert torch.equal(dx, torch.full_like(x, 2.0 if same else 0.0))
    assert torch.equal(dy, torch.full_like(x, 0.0 if same else 2.0))
    value, tangent = torch.func.jvp(build, (x, y), (torch.ones_like(x), 3 * torch.ones_like(y)))
    assert torch.equal(value, want) and torch.equal(tangent, torch.full_like(x, 2.0 if same else 6.0))


def test_c_dropout_refuses_a_type_before_anything_else():
    """Before its timing events are taken, as the other entry points do; so also without elements."""
    lib = _lib.load()
    p, keep = pointers(2)
    for n in (0, 4):
        assert lib.pk_dropout(4, 1, n, p, 2, None, 0, 0, 1.0, 0, 0, p, None) == -2
