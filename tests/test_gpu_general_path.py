"""The block-scaled linear, the rotary table and the head norm without the native call path's module: the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_results_without_the_module(monkeypatch, m, dtype):
    import qlin
    from qlin import _fast, _fp8, _rotary
    g = torch.Generator(device="cuda").manual_seed(m)
    w = (torch.randn(200, 272, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(2, 3, generator=g, device="cuda")
    x = torch.randn(m, 272, generator=g, device="cuda").to(dtype)
    b = torch.randn(200, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 90, (m, 2), generator=g, device="cuda")
    q, k = (torch.randn(2, m, h, 64, generator=g, device="cuda").to(dtype) for h in (4, 2))
    wt = torch.rand(64, generator=g, device="cuda").to(dtype)

    def all_of():
        t = qlin.rotary_table(pos, (32, 32))
        return [qlin.fp8_linear(x, w, s, b), qlin.fp8_linear(x, w, s), qlin.fp8_linear_grad_input(x[:, :200], w, s), t,
                *qlin.qk_norm_rotary(q, k, wt, None, t), *qlin.qk_norm_rotary_backward(q, k, q, k, wt, wt, t)]
    ref = all_of()
    for module in (_fp8, _rotary):
        assert not isinstance(module.native, _fast._Missing), "the module is built for the tests"
        monkeypatch.setattr(module, "native", _fast._Missing(None))
    for a, r in zip(all_of(), ref):
        assert torch.equal(a, r)
