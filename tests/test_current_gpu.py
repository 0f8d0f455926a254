"""Kernels launch on the thread's current GPU, so calls make their tensors' GPU current first.  Stand-in devices
and a stand-in for torch.cuda.device: no GPU is used and nothing is launched."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from polytensors_b200 import PolyTensor, _dispatch, _fused, _kernels, _token_ops


@pytest.fixture
def gpus(monkeypatch):
    """GPU 0 is current; the list of GPUs made current since."""
    now, entered = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            entered.append(self.index)
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    monkeypatch.setattr(_kernels, "several_gpus", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index)
    return entered


def test_a_stream_of_another_gpu_is_refused(gpus):
    assert _kernels._stream(torch.device("cuda:0")) == 100 and _kernels._stream(torch.device("cuda")) == 100
    with pytest.raises(ValueError, match="current GPU is 0"):
        _kernels._stream(torch.device("cuda:1"))
    with torch.cuda.device("cuda:1"):
        assert _kernels._stream(torch.device("cuda:1")) == 101


def test_token_operators_enter_their_tensors_gpu(gpus, monkeypatch):
    seen = []
    monkeypatch.setattr(_token_ops, "_wants_grad", lambda *_: False)
    for name, result in (("qk_norm_rope_fwd", ([None], [None])), ("dropout", [None]), ("token_log_probs_fwd", [[None]] * 4)):
        monkeypatch.setattr(_kernels, name, lambda *_, r=result: (seen.append(torch.cuda.current_device()), r)[1])
    for index in (0, 1):
        with FakeTensorMode():
            on = {"device": f"cuda:{index}"}
            x, table = torch.empty(1, 2, 2, 8, **on), torch.empty(4, 4, **on)
            PolyTensor.qk_norm_rope(x, x, None, None, table, table)
            PolyTensor.dropout(x, 0.5, seed=1)
            PolyTensor.dropout(input=x, p=0.5, seed=1)
            PolyTensor.token_log_probs(table, torch.empty(4, dtype=torch.int64, **on), check_indices=False)
        assert seen == [index] * 4
        seen.clear()
    assert gpus == [1] * 4 and torch.cuda.current_device() == 0


def test_series_operations_enter_their_tensors_gpu(gpus, monkeypatch):
    seen = []

    def record(*_, **__):
        seen.append(torch.cuda.current_device())
        return "done"

    monkeypatch.setitem(_dispatch._RULES, torch.ops.aten.add.Tensor, record)
    monkeypatch.setattr(_fused, "maybe_fused", record)
    monkeypatch.setattr(_fused, "cross_entropy_eligible", lambda *_: True)
    monkeypatch.setattr(_fused, "fused_cross_entropy", record)
    with FakeTensorMode(), PolyTensor.plain_range():
        x = PolyTensor((torch.empty(3, 4, device="cuda:1"), torch.empty(3, 4, device="cuda:1")))
        _dispatch.dispatch(torch.ops.aten.add.Tensor, (x, x), {})
        torch.nn.functional.rms_norm(x, (4,))
        PolyTensor.cross_entropy(x, torch.empty(3, dtype=torch.int64, device="cuda:1"))
    assert seen == [1, 1, 1] and gpus == [1, 1, 1] and torch.cuda.current_device() == 0
