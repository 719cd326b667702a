"""CPU checks of the block-scaled 8-bit linear, the rotary tables and the head norm at the C ABI: sizes and types that
the host refuses before anything is launched, workspace sizes, and the Python entry points' refusal of CPU tensors.
Pointers are never read here: every call ends in an answer of the host."""
import ctypes

import pytest
import torch

from oracle import attention_input as A

I64x3 = ctypes.c_int64 * 3
F32, F16, I32 = 0, 1, 5
SOME = 1 << 20  # a 16-byte aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    from qlin import _lib
    return _lib.lib


def test_workspaces(lib):
    assert lib.qlin_fp8_linear_workspace(0, 64, 128) == 0 and lib.qlin_fp8_linear_workspace(16, 64, 128) == 0 and lib.qlin_fp8_linear_workspace(4, 64, 0) == 0
    assert lib.qlin_fp8_linear_workspace(300, 64, 200) >= 300 * 256 + 2 * 300 * 4
    assert lib.qlin_fp8_linear_grad_input_workspace(300, 200, 64) >= 300 * 256 + 2 * 300 * 4
    assert lib.qlin_qk_norm_rotary_backward_workspace(0, 5, 2, 2, 64) == 0
    assert lib.qlin_qk_norm_rotary_backward_workspace(2, 500, 8, 2, 64) % (64 * 4) == 0


def _linear(lib, m=4, k=128, ldx=128, ldq=128, n=8, ld_scale=1, x=SOME, q=SOME, y=SOME, xd=F32, yd=F32, bd=F32, bias=None,
            ldy=8, ws=SOME, wsb=1 << 20):
    return lib.qlin_fp8_linear(x, xd, m, k, ldx, q, ldq, n, SOME, ld_scale, bias, bd, y, yd, ldy, ws, wsb, None)


@pytest.mark.parametrize("change,code", [
    (dict(m=-1), 2), (dict(k=-16), 2), (dict(n=-1), 2), (dict(ldx=64), 2), (dict(ldq=112), 2), (dict(ldy=4), 2),
    (dict(n=300, ldy=300, k=256, ldx=256, ldq=256, ld_scale=1), 2), (dict(m=1 << 31), 2), (dict(xd=I32), 1),
    (dict(yd=I32), 1), (dict(bias=SOME, bd=I32), 1), (dict(k=120, ldx=120), 1), (dict(ldq=136), 1),
    (dict(q=SOME + 8), 1), (dict(y=None), 2), (dict(x=None), 2), (dict(q=None), 2), (dict(m=100, ws=None), 2),
    (dict(m=100, wsb=100), 2), (dict(m=0), 0), (dict(n=0), 0)])
def test_linear_refusals(lib, change, code):
    assert _linear(lib, **change) == code
    if code:
        assert b"qlin_fp8_linear" in lib.qlin_last_error()


def test_grad_and_quantizer_refusals(lib):
    assert lib.qlin_fp8_linear_grad_input(SOME, F32, 4, 100, 100, SOME, 120, 120, SOME, 1, SOME, F32, 120, SOME, 1 << 20,
                                          None) == 1
    assert lib.qlin_fp8_linear_grad_input(SOME, F32, 100, 100, 100, SOME, 128, 128, SOME, 1, SOME, F32, 128, SOME, 16,
                                          None) == 2
    assert lib.qlin_fp8_linear_grad_input(SOME, F32, 4, 100, 99, SOME, 128, 128, SOME, 1, SOME, F32, 128, SOME, 1 << 20,
                                          None) == 2
    q = lib.qlin_quantize_rows_fp8
    assert q(SOME, F32, 4, 100, 100, SOME, 100, SOME, 4, None) == 2  # rows of out end before the block
    assert q(SOME, F32, 4, 100, 100, SOME, 128, SOME, 3, None) == 2
    assert q(SOME, I32, 4, 100, 100, SOME, 128, SOME, 4, None) == 1
    assert q(SOME, F32, 4, 100, 100, SOME + 4, 128, SOME, 4, None) == 1
    assert q(None, F32, 4, 100, 100, SOME, 128, SOME, 4, None) == 2
    assert q(None, F32, 0, 100, 100, None, 128, None, 4, None) == 0


def test_table_refusals(lib):
    dims = (ctypes.c_int32 * 3)(4, 6, 8)
    t = lib.qlin_rotary_table
    assert t(SOME, F32, -1, 3, dims, 1e4, SOME, None) == 2
    assert t(SOME, F32, 4, 0, dims, 1e4, SOME, None) == 2
    assert t(SOME, F32, 4, 3, None, 1e4, SOME, None) == 2
    assert t(SOME, F32, 4, 3, dims, 0.0, SOME, None) == 2
    assert t(SOME, F32, 4, 3, dims, float("nan"), SOME, None) == 2
    assert t(SOME, F16, 4, 3, dims, 1e4, SOME, None) == 1
    assert t(None, F32, 4, 3, dims, 1e4, SOME, None) == 2
    assert t(SOME, F32, 4, 3, dims, 1e4, SOME + 4, None) == 2
    assert t(SOME, F32, 4, 2, (ctypes.c_int32 * 2)(3, 4), 1e4, SOME, None) == 2
    assert t(SOME, F32, 4, 2, (ctypes.c_int32 * 2)(300, 300), 1e4, SOME, None) == 1
    assert t(SOME, F32, 0, 3, dims, 1e4, SOME, None) == 0


def _qk(lib, q=SOME, qs=I64x3(1024, 128, 64), dtype=F32, batch=1, tokens=8, hq=2, hk=2, dim=64, wd=F32, table=SOME, tb=0,
        pairs=32, out=SOME):
    st = I64x3(1024, 128, 64)
    return lib.qlin_qk_norm_rotary(q, qs, SOME, st, dtype, batch, tokens, hq, hk, dim, SOME, SOME, wd, table, tb, pairs,
                                   1e-6, 1, out, st, SOME, st, None)


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 2), (dict(tokens=-1), 2), (dict(hq=-1), 2), (dict(dim=0), 2), (dict(pairs=33), 2),
    (dict(pairs=-1), 2), (dict(batch=2, tb=16), 2), (dict(dtype=I32), 1), (dict(wd=I32), 1), (dict(dim=2048), 1),
    (dict(table=SOME + 4), 1), (dict(qs=None), 2), (dict(q=None), 2), (dict(out=None), 2), (dict(table=None), 2),
    (dict(batch=0), 0), (dict(tokens=0), 0)])
def test_head_norm_refusals(lib, change, code):
    assert _qk(lib, **change) == code


def test_head_norm_backward_refusals(lib):
    st = I64x3(1024, 128, 64)

    def call(dq=SOME, ws=SOME, wsb=1 << 20, gs=st):
        return lib.qlin_qk_norm_rotary_backward(dq, gs, SOME, st, SOME, st, SOME, st, F32, 1, 8, 2, 2, 64, SOME, SOME,
                                                F32, SOME, 0, 32, 1e-6, 1, SOME, st, SOME, st, SOME, SOME, ws, wsb,
                                                None)
    assert call(dq=None) == 2 and call(ws=None) == 2 and call(wsb=64) == 2 and call(gs=None) == 2


def test_cpu_tensors_are_refused():
    import qlin
    x = torch.zeros(2, 128)
    w = torch.zeros(64, 128).to(torch.float8_e4m3fn)
    h = torch.zeros(1, 2, 1, 8)
    t = torch.zeros(2, 4, 2)
    for call in (lambda: qlin.fp8_linear(x, w, torch.ones(1, 1)), lambda: qlin.quantize_fp8_rowwise(x),
                 lambda: qlin.fp8_linear_grad_input(torch.zeros(2, 64), w, torch.ones(1, 1)),
                 lambda: qlin.rotary_table(torch.zeros(3, 1), [8]),
                 lambda: qlin.qk_norm_rotary(h, h, None, None, t),
                 lambda: qlin.qk_norm_rotary_backward(h, h, h, h, None, None, t)):
        with pytest.raises(NotImplementedError):
            call()


# ------------------------------------------------------------------------------------------------ the oracle itself
def test_oracle_quantizer_reconstructs_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 300, generator=g) * 3
    x[2, 128:256] = 0
    q, s = A.quantize(x)
    amax = torch.stack([x[:, i:i + 128].abs().amax(1) for i in (0, 128, 256)], 1)
    err = (A.dequantize(q, s) - x.double()).abs()
    # e4m3 keeps 4 significant bits down to 2^-6 of its own scale, 2^-10 steps below
    limit = torch.maximum(x.double().abs() * 2.0 ** -4, (amax / 448.0).double().repeat_interleave(128, 1)[:, :300] * 2.0 ** -10)
    assert bool((err <= limit * 1.001 + 1e-30).all())
    assert bool((s[2, 1] == torch.tensor(2.0 ** -100) / torch.tensor(448.0)))


@pytest.mark.parametrize("inter", [True, False])
def test_oracle_gradients_against_autograd(inter):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 2, 20, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(20, generator=g, dtype=torch.float64, requires_grad=True)
    a = torch.randn(3, 8, generator=g, dtype=torch.float64)
    t = torch.stack([a.cos(), a.sin()], -1)
    dy = torch.randn(2, 3, 2, 20, generator=g, dtype=torch.float64)
    A.norm_rotary(x, w, t, 1e-6, inter).backward(dy)
    dx, dw, _, _ = A.norm_rotary_backward(dy, x.detach(), w.detach(), t, 1e-6, inter)
    assert torch.allclose(dx, x.grad, rtol=1e-12, atol=1e-13) and torch.allclose(dw, w.grad, rtol=1e-12, atol=1e-13)


def test_oracle_rotation_keeps_lengths_and_turns_by_the_angle():
    t = A.table(torch.tensor([[3, 5]]), [2, 4], 100.0)
    assert t.shape == (1, 3, 2)
    expect = torch.tensor([3.0, 5.0, 0.5], dtype=torch.float64)
    assert torch.allclose(t[0, :, 0], expect.cos()) and torch.allclose(t[0, :, 1], expect.sin())
    v = torch.randn(1, 1, 1, 8, dtype=torch.float64)
    for inter in (True, False):
        r = A.rotate(v, t, inter)
        assert torch.allclose(r.square().sum(), v.square().sum()) and torch.equal(r[..., 6:], v[..., 6:])
