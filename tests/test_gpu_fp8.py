"""GPU parity of the block-scaled 8-bit linear, its input gradient and the row quantizer through the C ABI, against
the 64-bit oracle.  Codes and scales are equal; outputs lie within the bound that oracle.attention_input.linear_bound
derives from the roundings that the kernel makes."""
import pytest
import torch

from oracle import attention_input as A

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def qlin():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import qlin as q
    return q


def _weights(n, k, g):
    q = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (torch.rand(-(-n // 128), -(-k // 128), generator=g) + 0.5) * 2e-4
    return q, s


def _status(qlin):
    code, where = qlin.device_status(reset=True)
    assert code == 0, f"a kernel timed out waiting (where={where:#x})"


def _check(got, ref, size, depth):
    bound = A.linear_bound(ref, size, depth, got.dtype)
    assert A.finite(got)
    excess = A.max_excess(got, ref, bound)
    assert excess <= 1.0, excess


SHAPES = [(1, 16, 16), (1, 5, 256), (2, 130, 272), (3, 128, 128), (7, 1, 1040), (16, 200, 4096), (17, 129, 384),
          (31, 640, 144), (33, 256, 2048), (64, 384, 2048), (65, 300, 528), (77, 1000, 1552), (128, 130, 640),
          (129, 129, 400), (200, 512, 1024), (256, 256, 128), (257, 300, 512), (300, 1000, 768), (520, 777, 1168)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_linear_matches_64_bits(qlin, m, n, k, dtype):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    q, s = _weights(n, k, g)
    x = torch.randn(m, k, generator=g).to(dtype)
    b = (torch.randn(n, generator=g) * 0.1).to(dtype)
    y = qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda(), b.cuda())
    assert y.dtype == dtype and y.shape == (m, n)
    _check(y, *A.linear(x, q, s, b), k)
    _status(qlin)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_grad_input_matches_64_bits(qlin, m, n, k, dtype):
    g = torch.Generator().manual_seed(m * 5 + n + k)
    q, s = _weights(n, k, g)
    dy = torch.randn(m, n, generator=g).to(dtype)
    dx = qlin.fp8_linear_grad_input(dy.cuda(), q.cuda(), s.cuda())
    assert dx.dtype == dtype and dx.shape == (m, k)
    _check(dx, *A.linear(dy, q, s, transposed=True), n)
    _status(qlin)


@pytest.mark.parametrize("x_dtype,y_dtype,b_dtype", [(BF16, F32, F16), (F32, F16, BF16), (F16, BF16, F32),
                                                     (BF16, F16, None)])
@pytest.mark.parametrize("m", [2, 40, 150])
def test_linear_types_mix(qlin, x_dtype, y_dtype, b_dtype, m):
    n, k = 264, 656
    g = torch.Generator().manual_seed(m)
    q, s = _weights(n, k, g)
    x = torch.randn(m, k, generator=g).to(x_dtype)
    b = None if b_dtype is None else torch.randn(n, generator=g).to(b_dtype)
    y = qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda(), None if b is None else b.cuda(), out_dtype=y_dtype)
    assert y.dtype == y_dtype
    _check(y, *A.linear(x, q, s, b), k)
    dx = qlin.fp8_linear_grad_input(x[:, :n].contiguous().cuda(), q.cuda(), s.cuda(), out_dtype=y_dtype)
    assert dx.dtype == y_dtype
    _check(dx, *A.linear(x[:, :n], q, s, transposed=True), n)


@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 130), (9, 1000), (40, 4096), (130, 2049)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantizer_is_exact(qlin, m, k, dtype):
    g = torch.Generator().manual_seed(m + k)
    x = (torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-12, 8, (m, 1), generator=g).float())).to(dtype)
    x[:, ::7] = 0
    if k > 300:
        x[0, 128:256] = 0  # a block of zeros
    q, s = qlin.quantize_fp8_rowwise(x.cuda())
    q_ref, s_ref = A.quantize(x)
    assert torch.equal(s.cpu(), s_ref)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), q_ref.contiguous().view(torch.uint8))
    # rows that start off a 16-byte boundary, and a transposed input
    wide = torch.zeros(m, k + 3, dtype=dtype, device="cuda")
    wide[:, 3:] = x.cuda()
    q2, s2 = qlin.quantize_fp8_rowwise(wide[:, 3:])
    assert torch.equal(s2, s) and torch.equal(q2.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))
    q3, s3 = qlin.quantize_fp8_rowwise(x.t().contiguous().cuda().t())
    assert torch.equal(s3, s) and torch.equal(q3.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))


def test_quantizer_extremes(qlin):
    tiny = torch.full((2, 128), 1e-38)
    tiny[1] = 1e-44
    q, s = qlin.quantize_fp8_rowwise(tiny.cuda())
    q_ref, s_ref = A.quantize(tiny)
    assert torch.equal(s.cpu(), s_ref) and bool((s > 0).all())
    assert torch.equal(q.cpu().view(torch.uint8), q_ref.view(torch.uint8))
    big = torch.full((1, 128), 3e38)
    big[0, ::2] = -1e30
    q, s = qlin.quantize_fp8_rowwise(big.cuda())
    q_ref, s_ref = A.quantize(big)
    assert torch.equal(s.cpu(), s_ref) and torch.equal(q.cpu().view(torch.uint8), q_ref.view(torch.uint8))


@pytest.mark.parametrize("m", [4, 40, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_inputs_stay_in_their_rows(qlin, m, bad):
    n, k = 200, 400
    g = torch.Generator().manual_seed(1)
    q, s = _weights(n, k, g)
    x = torch.randn(m, k, generator=g).to(BF16)
    clean = qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda())
    x[1, 390] = bad
    y = qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda())
    assert not bool(torch.isfinite(y[1].float()).any())
    keep = [i for i in range(m) if i != 1]
    assert torch.equal(y[keep], clean[keep])
    dy = torch.randn(m, n, generator=g).to(BF16)
    clean = qlin.fp8_linear_grad_input(dy.cuda(), q.cuda(), s.cuda())
    dy[m - 1, 0] = bad
    dx = qlin.fp8_linear_grad_input(dy.cuda(), q.cuda(), s.cuda())
    assert not bool(torch.isfinite(dx[m - 1].float()).any())
    assert torch.equal(dx[:m - 1], clean[:m - 1])


@pytest.mark.parametrize("m", [5, 50, 140])
def test_strided_operands(qlin, m):
    n, k = 144, 336
    g = torch.Generator().manual_seed(m)
    q, s = _weights(n, k, g)
    x = torch.randn(m, k, generator=g).to(F16)
    ref = qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda())
    big = torch.zeros(n + 2, k + 48, dtype=torch.uint8)
    big[1:n + 1, 16:16 + k] = q.view(torch.uint8)
    qv = big.cuda().view(torch.float8_e4m3fn)[1:n + 1, 16:16 + k]    # aligned slice: read in place
    qo = torch.zeros(n, k + 5, dtype=torch.uint8).cuda()
    qo[:, 5:] = q.view(torch.uint8).cuda()
    qo = qo.view(torch.float8_e4m3fn)[:, 5:]                          # misaligned slice: copied
    wide = torch.zeros(s.shape[0], s.shape[1] + 2).cuda()
    wide[:, 1:-1] = s.cuda()
    odd = torch.zeros(m, k + 1, dtype=F16).cuda()
    odd[:, 1:] = x.cuda()
    for w in (qv, qo):
        for sc in (wide[:, 1:-1], s.t().contiguous().cuda().t(), s.double().cuda()):
            assert torch.equal(qlin.fp8_linear(x.cuda(), w, sc), ref)
    assert torch.equal(qlin.fp8_linear(odd[:, 1:], q.cuda(), s.cuda()), ref)
    assert torch.equal(qlin.fp8_linear(x.t().contiguous().cuda().t(), q.cuda(), s.cuda()), ref)
    assert torch.equal(qlin.fp8_linear(x.cuda()[:1].expand(m, k), q.cuda(), s.cuda()), ref[:1].expand(m, n))
    y3 = qlin.fp8_linear(x.cuda().view(1, m, 1, k), q.cuda(), s.cuda())
    assert y3.shape == (1, m, 1, n) and torch.equal(y3.view(m, n), ref)
    dref = qlin.fp8_linear_grad_input(x.cuda()[:, :n].contiguous(), q.cuda(), s.cuda())
    assert torch.equal(qlin.fp8_linear_grad_input(x.cuda()[:, :n], qv, wide[:, 1:-1]), dref)
    assert torch.equal(qlin.fp8_linear_grad_input(odd[:, 1:n + 1], qo, s.cuda()), dref)


def test_rows_past_32_bit_offsets(qlin):
    n, k, m = 144, 272, 3
    g = torch.Generator().manual_seed(4)
    q, s = _weights(n, k, g)
    x = torch.randn(m, k, generator=g).to(F16)
    store = torch.empty(2 * (2 ** 30 + 8) + 2 ** 20, dtype=F16, device="cuda")
    far = store.as_strided((m, k), (2 ** 30 + 8, 1), 0)
    far.copy_(x)
    assert torch.equal(qlin.fp8_linear(far, q.cuda(), s.cuda()), qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda()))
    far8 = torch.empty(0, device="cuda")
    del far, store, far8
    torch.cuda.empty_cache()


def test_empty_sizes(qlin):
    g = torch.Generator().manual_seed(0)
    q, s = _weights(130, 256, g)
    q, s = q.cuda(), s.cuda()
    assert qlin.fp8_linear(torch.empty(0, 256, dtype=F16, device="cuda"), q, s).shape == (0, 130)
    assert qlin.fp8_linear_grad_input(torch.empty(2, 0, 130, device="cuda"), q, s).shape == (2, 0, 256)
    e = torch.empty(0, 256, device="cuda").to(torch.float8_e4m3fn)
    assert qlin.fp8_linear(torch.ones(4, 256, device="cuda"), e, torch.empty(0, 2, device="cuda")).shape == (4, 0)
    z = qlin.fp8_linear_grad_input(torch.empty(4, 0, device="cuda"), e, torch.empty(0, 2, device="cuda"))
    assert z.shape == (4, 256) and bool((z == 0).all())
    e = torch.empty(5, 0, device="cuda").to(torch.float8_e4m3fn)
    b = torch.arange(5.0, device="cuda")
    y = qlin.fp8_linear(torch.empty(3, 0, device="cuda"), e, torch.empty(1, 0, device="cuda"), b)
    assert torch.equal(y, b.expand(3, 5))
    q0, s0 = qlin.quantize_fp8_rowwise(torch.empty(0, 40, device="cuda"))
    assert q0.shape == (0, 40) and s0.shape == (0, 1)


def _exact_points(rows, cols, g):
    """Rows whose quantization is exact: e4m3 values with a 448 in every block of 128."""
    v = (torch.randn(rows, cols, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    v[:, ::128] = 448.0
    return v


@pytest.mark.parametrize("m,n,k", [(6, 200, 336), (150, 300, 512)])
def test_gradient_against_differences(qlin, m, n, k):
    """Where the quantization is exact, the linear is linear in x: the change of <dy, y> between two points
    is <dx, the step> to the fp32 sums' bound."""
    g = torch.Generator().manual_seed(m)
    q, s = _weights(n, k, g)
    x0, x1, dy = _exact_points(m, k, g), _exact_points(m, k, g), _exact_points(m, n, g)
    y0, y1 = (qlin.fp8_linear(x.cuda(), q.cuda(), s.cuda()).double().cpu() for x in (x0, x1))
    dx = qlin.fp8_linear_grad_input(dy.cuda(), q.cuda(), s.cuda()).double().cpu()
    lhs = (dy.double() * (y1 - y0)).sum(1)
    rhs = (dx * (x1 - x0).double()).sum(1)
    wd = A.weight(q, s).abs()
    size = (dy.double().abs() * ((x0.abs() + x1.abs()).double() @ wd.t())).sum(1)
    blocks = -(-max(n, k) // 128)
    assert bool(((lhs - rhs).abs() <= size * 2 * (2.0 ** -16 + (blocks + 4) * 2.0 ** -23)).all())


def test_trainable_gradients(qlin):
    m, n, k = 70, 192, 512
    g = torch.Generator().manual_seed(9)
    q, s = _weights(n, k, g)
    q, s = q.cuda(), s.cuda()
    x = torch.randn(2, m, k, generator=g).to(BF16).cuda().requires_grad_(True)
    b = (torch.randn(n, generator=g) * 0.01).to(BF16).cuda().requires_grad_(True)
    y = qlin.fp8_linear_trainable(x, q, s, b)
    assert torch.equal(y.detach(), qlin.fp8_linear(x.detach(), q, s, b.detach()))
    dy = torch.randn(2, m, n, generator=g).to(BF16).cuda()
    y.backward(dy)
    assert torch.equal(x.grad, qlin.fp8_linear_grad_input(dy, q, s))
    assert torch.equal(b.grad, dy.view(-1, n).float().sum(0).to(BF16))
    y = qlin.fp8_linear_trainable(x, q, s, b)
    y.sum().backward()  # an expanded gradient
    assert A.finite(x.grad)


def test_repeatable_on_side_stream_and_in_a_graph(qlin):
    for m in (3, 60, 300):
        n, k = 520, 1040
        g = torch.Generator().manual_seed(m)
        q, s = _weights(n, k, g)
        q, s = q.cuda(), s.cuda()
        x = torch.randn(m, k, generator=g).to(BF16).cuda()
        ref, dref = qlin.fp8_linear(x, q, s), qlin.fp8_linear_grad_input(x[:, :n], q, s)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y = qlin.fp8_linear(x, q, s)
        side.synchronize()
        assert torch.equal(y, ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = qlin.fp8_linear(x, q, s)
            dx = qlin.fp8_linear_grad_input(x[:, :n], q, s)
        for _ in range(3):
            y.zero_()
            dx.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ref) and torch.equal(dx, dref)
        del graph
    _status(qlin)


def test_refusals(qlin):
    q = torch.zeros(64, 128, device="cuda").to(torch.float8_e4m3fn)
    s = torch.ones(1, 1, device="cuda")
    x = torch.zeros(2, 128, device="cuda")
    with pytest.raises(ValueError):
        qlin.fp8_linear(x[:, :64], q, s)
    with pytest.raises(ValueError):
        qlin.fp8_linear(x, q, torch.ones(1, 2, device="cuda"))
    with pytest.raises(ValueError):
        qlin.fp8_linear(x, q, s, torch.zeros(3, device="cuda"))
    with pytest.raises(qlin.QlinDecline):
        qlin.fp8_linear(x, q.float(), s)
    with pytest.raises(qlin.QlinDecline):
        qlin.fp8_linear(x.double(), q, s)
    with pytest.raises(qlin.QlinDecline):
        qlin.fp8_linear(x, q, s, out_dtype=torch.int32)
    with pytest.raises(qlin.QlinDecline):  # K not a multiple of 16
        qlin.fp8_linear(x[:, :24], torch.zeros(64, 24, device="cuda").to(torch.float8_e4m3fn), s)
    with pytest.raises(ValueError):
        qlin.fp8_linear_grad_input(x, q, s)
    with pytest.raises(NotImplementedError):
        qlin.fp8_linear(x.cpu(), q, s)
    with pytest.raises(NotImplementedError):
        qlin.fp8_linear(x, q.cpu(), s.cpu())
    with pytest.raises(qlin.QlinDecline):
        qlin.quantize_fp8_rowwise(x.int())
    _status(qlin)
