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


def _out(q, k, out):
    import qlin
    table = _on(0, (5, 8, 2), torch.float32)
    table.contiguous = lambda: table
    return qlin.qk_norm_rotary(q, k, None, None, table, out=out)


@pytest.mark.parametrize("shape,stride", [((2, 5, 3, 16), (0, 48, 16, 1)), ((2, 5, 3, 16), (240, 0, 16, 1)),
                                          ((2, 5, 3, 16), (240, 48, 0, 1)), ((2, 5, 3, 16), (240, 48, 8, 1)),
                                          ((2, 5, 3, 16), (200, 48, 16, 1)), ((2, 5, 3, 16), (16, 16, 160, 1))])
def test_head_norm_refuses_outputs_that_overlap_themselves(shape, stride):
    def strided(st):
        t = _on(0, shape, torch.float32)
        t.stride = lambda i=None: st if i is None else st[i]
        return t
    x, plain = _on(0, shape, torch.float32), (240, 48, 16, 1)
    for out in ((strided(stride), strided(plain)), (strided(plain), strided(stride))):
        with pytest.raises(ValueError, match="overlap"):
            _out(x, x, out)


def test_slices_of_joint_buffers_do_not_overlap_themselves():
    from qlin._rotary import _overlaps_itself
    joint, first = torch.empty(2, 9, 6, 16), torch.empty(2, 6, 9, 16).transpose(1, 2)
    for t in (joint, joint[:, 4:], joint[:, ::2, 1:3], joint[:1], joint[:, :1], joint[:, :, :1], joint[..., :8], first,
              first[:, 2:, ::3], joint.transpose(0, 1), torch.empty(1, 1, 1, 16).as_strided((1, 1, 1, 16), (0, 0, 0, 1))):
        assert not _overlaps_itself(t), t.stride()
