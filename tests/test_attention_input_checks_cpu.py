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


class _Native:
    """The native path's functions, here on the CPU, with a count of their calls."""

    def __init__(self):
        self.calls = []

    def fp8_linear(self, x, qdata, scale, bias):
        self.calls.append("fp8_linear")
        return (x.float() @ qdata.float().t()).to(x.dtype).detach()

    def fp8_linear_grad_input(self, dy, qdata, scale):
        self.calls.append("fp8_linear_grad_input")
        return (dy.float() @ qdata.float()).to(dy.dtype).detach()

    def qk_norm_rotary(self, q, k, *args):
        return (q * 2).detach(), (k * 3).detach()

    def qk_norm_rotary_backward(self, dq, dk, q, k, q_weight, k_weight, *args):
        return (dq * 2).detach(), (dk * 3).detach(), q_weight.detach() * 0, k_weight.detach() * 0


@pytest.fixture
def native(monkeypatch):
    from qlin import _fp8, _rotary
    n = _Native()
    monkeypatch.setattr(_fp8, "native", n)
    monkeypatch.setattr(_rotary, "native", n)
    return n


def test_an_output_type_equal_to_the_inputs_takes_the_native_path(native):
    import qlin
    x, w, s = torch.randn(3, 128).bfloat16(), torch.randn(64, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    assert qlin.fp8_linear(x, w, s, out_dtype=torch.bfloat16).shape == (3, 64)
    assert qlin.fp8_linear_grad_input(x[:, :64], w, s, out_dtype=torch.bfloat16).shape == (3, 128)
    assert native.calls == ["fp8_linear", "fp8_linear_grad_input"]
    with pytest.raises(NotImplementedError):  # another type is the general path's
        qlin.fp8_linear(x, w, s, out_dtype=torch.float32)
    assert len(native.calls) == 2


def test_training_takes_the_native_path_in_both_directions(native):
    import qlin
    x = torch.randn(3, 128).bfloat16().requires_grad_(True)
    w = torch.randn(64, 128).to(torch.float8_e4m3fn)
    y = qlin.fp8_linear_trainable(x, w, torch.ones(1, 1))
    y.backward(torch.ones_like(y))
    assert native.calls == ["fp8_linear", "fp8_linear_grad_input"]
    assert torch.equal(x.grad, w.float().sum(0).bfloat16().expand(3, 128))


def test_gradients_of_gradients_are_refused(native):
    """The gradients are the kernels', without a graph: a penalty on them would be left out of the loss unseen."""
    import qlin
    x = torch.randn(3, 128, requires_grad=True)
    w = torch.randn(64, 128).to(torch.float8_e4m3fn)
    loss = qlin.fp8_linear_trainable(x, w, torch.ones(1, 1)).square().sum()
    (gx,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (loss + gx.square().sum()).backward()
    q, k = (torch.randn(1, 2, 1, 8, requires_grad=True) for _ in range(2))
    qw, kw = torch.ones(8, requires_grad=True), torch.ones(8, requires_grad=True)
    a, b = qlin.qk_norm_rotary_trainable(q, k, qw, kw, torch.zeros(2, 4, 2))
    loss = a.square().sum() + b.square().sum()
    (gq,) = torch.autograd.grad(loss, q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (loss + gq.square().sum()).backward()
    # the first derivatives stay what they are
    loss = qlin.fp8_linear_trainable(x, w, torch.ones(1, 1)).sum()
    loss.backward()
    assert torch.equal(x.grad, w.float().sum(0).expand(3, 128))


@pytest.mark.parametrize("shape,n", [((3, 128), 0), ((0, 128), 64), ((2, 0, 128), 64), ((128,), 64), ((2, 3, 128), 64)])
def test_bias_gradient_of_any_shape(native, shape, n):
    import qlin
    x, w = torch.randn(shape, requires_grad=True), torch.randn(n, 128).to(torch.float8_e4m3fn)
    b = torch.zeros(n, requires_grad=True)
    y = qlin.fp8_linear_trainable(x, w, torch.ones(-(-n // 128), 1), b)
    y.backward(torch.ones_like(y))
    rows = y.numel() // n if n else 0
    assert torch.equal(b.grad, torch.full((n,), float(rows))) and x.grad.shape == shape
