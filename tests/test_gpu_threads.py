"""Operators as the first CUDA work of a thread, as autograd's threads and servers call them: the thread has no current
context then, and outputs come from memory that the allocator already holds."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_fill():
    """Without the fills of fresh allocations, whose launches would make a context current."""
    was = torch.utils.deterministic.fill_uninitialized_memory
    torch.utils.deterministic.fill_uninitialized_memory = False
    yield
    torch.utils.deterministic.fill_uninitialized_memory = was


def _in_a_thread(call):
    got = []

    def body():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001  (raised again below)
            got.append(e)
    t = threading.Thread(target=body)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


def _calls(m):
    import qlin
    g = torch.Generator(device="cuda").manual_seed(m)
    w = torch.randn(256, 384, generator=g, device="cuda").mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(2, 3, generator=g, device="cuda") * 1e-3
    x = torch.randn(m, 384, generator=g, device="cuda").bfloat16()
    dy = torch.randn(m, 256, generator=g, device="cuda").bfloat16()
    h = dy.view(1, m, 4, 64)
    wi = torch.randint(-127, 128, (256, 384), generator=g, device="cuda").to(torch.int8)
    si = torch.rand(256, generator=g, device="cuda") * 1e-3
    pos = torch.arange(m, device="cuda").unsqueeze(1)
    tab = qlin.rotary_table(pos, [64])
    return {"linear": lambda: qlin.fp8_linear(x, w, s), "grad": lambda: qlin.fp8_linear_grad_input(dy, w, s),
            "to f32": lambda: qlin.fp8_linear(x, w, s, out_dtype=torch.float32),
            "quantize": lambda: qlin.quantize_fp8_rowwise(x)[1], "table": lambda: qlin.rotary_table(pos, [64]),
            "norm": lambda: qlin.qk_norm_rotary(h, h, None, None, tab)[0],
            "norm grad": lambda: qlin.qk_norm_rotary_backward(h, h, h, h, None, None, tab)[0],
            "int8": lambda: qlin.int8_linear(x, wi, si)}


@pytest.mark.parametrize("name", ["linear", "grad", "to f32", "quantize", "table", "norm", "norm grad", "int8"])
@pytest.mark.parametrize("m", [3, 200])
def test_first_call_of_a_thread(name, m):
    call = _calls(m)[name]
    ref = call()
    del ref  # the thread's call takes this memory
    ref = call().clone()
    torch.cuda.synchronize()
    got = _in_a_thread(call)
    torch.cuda.synchronize()
    assert torch.equal(got, ref)


@pytest.mark.parametrize("m", [3, 200])
def test_backward_that_begins_with_the_gradient(m):
    import qlin
    g = torch.Generator(device="cuda").manual_seed(m)
    w = torch.randn(256, 384, generator=g, device="cuda").to(torch.float8_e4m3fn)
    s = torch.rand(2, 3, generator=g, device="cuda")
    x = torch.randn(m, 384, generator=g, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(m, 256, generator=g, device="cuda").bfloat16()
    ref = qlin.fp8_linear_grad_input(dy, w, s)
    y = _in_a_thread(lambda: qlin.fp8_linear_trainable(x, w, s))
    assert torch.equal(_in_a_thread(lambda: torch.autograd.grad(y, x, dy))[0], ref)
