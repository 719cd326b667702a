"""The two ways to the block-scaled linear, the rotary table and the head norm: the native call path takes the calls
that need no copy, gives what the general path gives bit for bit, and leaves every other call to it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qlin():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import qlin as q
    return q


def _weight(n, k):
    g = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn(n, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return w, torch.rand(-(-n // 128), -(-k // 128), generator=g, device="cuda"), g


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear(qlin, m):
    from qlin._fast import native
    w, s, g = _weight(200, 272)
    x = torch.randn(m, 272, generator=g, device="cuda").to(torch.bfloat16)
    b = torch.randn(200, generator=g, device="cuda")
    y = native.fp8_linear(x, w, s, b)
    assert torch.equal(y, qlin.fp8_linear(x, w, s, b, out_dtype=x.dtype))
    dx = native.fp8_linear_grad_input(x[:, :200], w, s)
    assert torch.equal(dx, qlin.fp8_linear_grad_input(x[:, :200], w, s, out_dtype=x.dtype))
    # a parameter and a tensor that requires grad come out the same, without a graph
    p = torch.nn.Parameter(x.clone())
    got = native.fp8_linear(p, w, s, b)
    assert torch.equal(got, y) and not got.requires_grad
    for args in ((x.cpu(), w, s, b), (x.double(), w, s, b), (x, w.float(), s, b), (x, w, s.double(), b), (x, w, s, b[:9]),
                 (x[:, ::2], w[:, :136], s, b), (x[:0], w, s, b), (x, w, s[:1], b), ([1.0], w, s, b)):
        assert native.fp8_linear(*args) is None


def test_table_and_head_norm(qlin):
    from qlin._fast import native
    pos = torch.randint(0, 60, (12, 3), device="cuda")
    t = native.rotary_table(pos, [16, 24, 24], 10000.0)
    assert torch.equal(t, qlin.rotary_table(pos.t().contiguous().t(), (16, 24, 24)))
    for args in ((pos.cpu(), [16, 24, 24], 1e4), (pos.half(), [16, 24, 24], 1e4), (pos, [16, 24], 1e4), (pos, [16, 24, 23], 1e4),
                 (pos, [16, 24, 24], 10000), (pos[:0], [16, 24, 24], 1e4), (pos, [0, 0, 0], 1e4)):
        assert native.rotary_table(*args) is None
    q, k = torch.randn(2, 12, 4, 64, device="cuda"), torch.randn(2, 12, 2, 64, device="cuda")
    w = torch.rand(64, device="cuda")
    got = native.qk_norm_rotary(q, k, w, None, t, 1e-6, True)
    ref = qlin.qk_norm_rotary(q, k, w, None, t[None], 1e-6, True)  # a table with a batch takes the general path
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    got = native.qk_norm_rotary_backward(q, k, q, k, w, None, t, 1e-6, False)
    ref = qlin.qk_norm_rotary_backward(q, k, q, k, w, None, t[None], 1e-6, False)
    assert got[3] is None and ref[3] is None and all(torch.equal(a, b) for a, b in zip(got[:3], ref[:3]))
    for args in ((q.cpu(), k, w, w, t, 1e-6, True), (q, k.half(), w, w, t, 1e-6, True), (q, k, w, w.half(), t, 1e-6, True),
                 (q, k, w[:9], w, t, 1e-6, True), (q, k, w, w, t[:5], 1e-6, True), (q, k, w, w, t, 0, True),
                 (q[..., ::2], k[..., ::2], None, None, t[:, :16], 1e-6, True), (q[:0], k[:0], w, w, t, 1e-6, True)):
        assert native.qk_norm_rotary(*args) is None


def test_empty_contraction_at_the_c_abi(qlin):
    """k = 0: the bias, rounded to y's type, for few and for many tokens."""
    b = torch.randn(300, device="cuda")
    w, s = torch.zeros(512, dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda")
    for m in (3, 200):
        y = torch.full((m, 300), 7.0, dtype=torch.float16, device="cuda")
        rc = qlin.lib.qlin_fp8_linear(w.data_ptr(), 0, m, 0, 0, w.data_ptr(), 16, 300, s.data_ptr(), 1, b.data_ptr(), 0,
                                      y.data_ptr(), 1, 300, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(y, b.half().expand(m, 300))
