"""Checks of the Python entry points of the block-scaled linear and the head norm that end in an answer before any
tensor is read: tensors of another device, outputs whose rows lie on one another."""
from types import SimpleNamespace

import pytest
import torch


def _on(index, shape, dtype):
    """What the checks see of a CUDA tensor; there may be no such device here."""
    t = torch.empty(shape, dtype=dtype, device="meta")
    return SimpleNamespace(is_cuda=True, device=torch.device("cuda", index), dtype=dtype, shape=t.shape, dim=t.dim,
                           stride=t.stride, numel=t.numel, data_ptr=lambda: 0)


@pytest.mark.parametrize("x,w,s", [(0, 0, 1), (1, 1, 0), (0, 1, 1)])
def test_linear_refuses_a_weight_or_scale_of_another_device(x, w, s):
    import qlin
    q, sc = _on(w, (256, 128), torch.float8_e4m3fn), _on(s, (2, 1), torch.float32)
    with pytest.raises(ValueError, match="cuda:1"):
        qlin.fp8_linear(_on(x, (4, 128), torch.float32), q, sc)
    with pytest.raises(ValueError, match="cuda:1"):
        qlin.fp8_linear_grad_input(_on(x, (4, 256), torch.float32), q, sc)
