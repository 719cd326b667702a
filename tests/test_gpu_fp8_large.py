"""The forms of the block-scaled linear that only larger sizes reach: CTA pairs, CTAs that take several tiles, several
token groups, and the contraction shared by 2 or 8 CTAs; ragged in every direction, outputs on and off 16-byte rows.

Operands are whole numbers and scales powers of two, so that every product and every sum is exact in fp32 in any order
(each element's products add up to less than 2^24 units in magnitude): outputs are compared bit for bit.  A form
whose sums held fewer bits would show.  A second test takes ordinary values against 64 bits."""
import json
import re

import pytest
import torch

from oracle import attention_input as A

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIR, ONE = "fp8_gemm_kernel<2, 256, {}>", "fp8_gemm_kernel<1, 128, {}>"
# tokens, outputs, contraction, kernel, its CTAs on 148 SMs
FORMS = [
    (1700, 1650, 272, PAIR, 98),      # 7 x 7 tiles, the last ones half empty
    (1700, 1664, 272, PAIR, 98),
    (2200, 2203, 400, PAIR, 148),     # 81 tiles for 74 pairs
    (2200, 2208, 400, PAIR, 148),
    (2700, 1111, 16400, PAIR, 110),   # groups of 6 and 5 token tiles
    (2700, 1120, 16400, PAIR, 110),
    (1050, 3709, 144, ONE, 148),      # 261 tiles for 148 CTAs
    (1050, 3712, 144, ONE, 148),
    (2333, 135, 2784, ONE, 76),       # 2 CTAs to a tile
    (140, 270, 9008, ONE, 48),        # 8 CTAs to a tile
    (3725, 144, 10896, ONE, 120),     # 2 CTAs to a tile, two groups
]


@pytest.fixture(scope="module")
def qlin():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import qlin as q
    yield q
    torch.cuda.empty_cache()


def _launches(call, path):
    """The call's result and the (name, CTAs) of its kernels."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        got = call()
        torch.cuda.synchronize()
    prof.export_chrome_trace(str(path))
    events = json.loads(path.read_text())["traceEvents"]
    return got, [(e["name"], e["args"]["grid"][0]) for e in events if e.get("cat") == "kernel"]


def _expect(launches, kernel, trans, ctas):
    ours = [(re.sub(r"\((int|bool)\)", "", n).replace("false", "0").replace("true", "1"), c) for n, c in launches if "fp8_" in n]
    assert len(ours) == 2 and "quant_rows_fp8_kernel" in ours[0][0], launches
    assert kernel.format(int(trans)) in ours[1][0] and ours[1][1] == ctas, ours


def _whole(rows, cols, g):
    """Activations that the quantizer leaves as they are: whole numbers up to 4, and a 448 in every block of 128."""
    v = torch.randint(-4, 5, (rows, cols), generator=g, device="cuda").float()
    v[:, ::128] = 448.0
    return v


def _weight(n, k, g):
    """e4m3 whole numbers from 1 to 240 and scales of 2^-10 or 2^-9."""
    q = torch.randn(n, k, generator=g, device="cuda").mul_(60).clamp_(-240, 240).round_().to(torch.float8_e4m3fn)
    s = torch.exp2(torch.randint(-10, -8, (-(-n // 128), -(-k // 128)), generator=g, device="cuda").float())
    return q, s


def _dense(q, s):
    n, k = q.shape
    return q.double() * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _exact(x, wd, bias):
    """The 64-bit result, after a check that the sum of the magnitudes stays below 2^24 units of 2^-10."""
    y, size = x.double() @ wd, x.double().abs() @ wd.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    assert float(size.max()) < 2.0 ** 14
    return y


def _clean(qlin):
    code, where = qlin.device_status(reset=True)
    assert code == 0, hex(where)


@pytest.mark.parametrize("m,n,k,kernel,ctas", FORMS)
def test_linear_is_exact(qlin, tmp_path, m, n, k, kernel, ctas):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, (q, s) = _whole(m, k, g), _weight(n, k, g)
    b = torch.randint(-99, 99, (n,), generator=g, device="cuda").float()
    ref = _exact(x, _dense(q, s).t(), b).float()
    y, launches = _launches(lambda: qlin.fp8_linear(x, q, s, b), tmp_path / "trace.json")
    _expect(launches, kernel, False, ctas)
    assert torch.equal(y, ref)
    for dtype in (F16, BF16):
        y = qlin.fp8_linear(x.to(dtype), q, s, b.to(dtype))
        assert torch.equal(y, ref.to(dtype)), dtype
    _clean(qlin)


@pytest.mark.parametrize("m,k,n,kernel,ctas", [f for f in FORMS if f[1] % 16 == 0] + [
    (1700, 1664, 275, PAIR, 98), (2200, 2208, 333, PAIR, 148), (140, 272, 9001, ONE, 48), (2333, 144, 2777, ONE, 76)])
def test_grad_input_is_exact(qlin, tmp_path, m, k, n, kernel, ctas):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    dy, (q, s) = _whole(m, n, g), _weight(n, k, g)
    ref = _exact(dy, _dense(q, s), None).float()
    dx, launches = _launches(lambda: qlin.fp8_linear_grad_input(dy, q, s), tmp_path / "trace.json")
    _expect(launches, kernel, True, ctas)
    assert torch.equal(dx, ref)
    for dtype in (F16, BF16):
        assert torch.equal(qlin.fp8_linear_grad_input(dy.to(dtype), q, s), ref.to(dtype)), dtype
    _clean(qlin)


@pytest.mark.parametrize("m,n,k", [(1, 1000, 256), (2, 300, 5120), (5, 200, 400), (9, 1008, 4096), (16, 130, 1552),
                                   (17, 300, 640), (77, 1000, 1552), (128, 650, 2048), (333, 1027, 4096)])
def test_smaller_forms_are_exact(qlin, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, dy, (q, s) = _whole(m, k, g), _whole(m, n, g), _weight(n, k, g)
    b = torch.randint(-99, 99, (n,), generator=g, device="cuda").float()
    ref, dref = _exact(x, _dense(q, s).t(), b).float(), _exact(dy, _dense(q, s), None).float()
    for dtype in (F32, F16, BF16):
        assert torch.equal(qlin.fp8_linear(x.to(dtype), q, s, b.to(dtype)), ref.to(dtype)), dtype
        assert torch.equal(qlin.fp8_linear_grad_input(dy.to(dtype), q, s), dref.to(dtype)), dtype
    _clean(qlin)


@pytest.mark.parametrize("m,k,n", [(1700, 1664, 272), (2200, 2208, 400), (1050, 3712, 144), (140, 272, 9008)])
@pytest.mark.parametrize("dtype,code", [(F32, 0), (F16, 1), (BF16, 2)])
@pytest.mark.parametrize("gap,first", [(1, 0), (3, 1), (8, 0)])
def test_grad_input_into_rows_of_any_pitch(qlin, m, k, n, dtype, code, gap, first):
    """Outputs inside a wider buffer, at every alignment; what lies between the rows stays."""
    g = torch.Generator(device="cuda").manual_seed(m)
    dy, (q, s) = _whole(m, n, g).to(dtype), _weight(n, k, g)
    ref = _exact(dy, _dense(q, s), None).float().to(dtype)
    wide = torch.full((m + 2, k + gap), 7.0, dtype=dtype, device="cuda")
    dx = wide.view(-1)[k + gap + first:][:m * (k + gap)].view(m, k + gap)[:, :k]
    nws = qlin.lib.qlin_fp8_linear_grad_input_workspace(m, n, k)
    ws = torch.empty(nws, dtype=torch.uint8, device="cuda")
    rc = qlin.lib.qlin_fp8_linear_grad_input(dy.data_ptr(), code, m, n, n, q.data_ptr(), k, k, s.data_ptr(), s.stride(0),
                                             dx.data_ptr(), code, k + gap, ws.data_ptr(), nws,
                                             torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(dx, ref)
    dx.fill_(7.0)
    assert bool((wide == 7.0).all())
    _clean(qlin)


@pytest.mark.parametrize("m,n,k", [(1700, 1651, 272), (2700, 1120, 16400), (1050, 3712, 144), (140, 270, 9008)])
def test_ordinary_values(qlin, m, n, k):
    """Both directions against 64 bits, and the same bits at every repeat."""
    g = torch.Generator().manual_seed(m)
    q = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (torch.rand(-(-n // 128), -(-k // 128), generator=g) + 0.5) * 2e-4
    wd, qc, sc = _dense(q.cuda(), s.cuda()), q.cuda(), s.cuda()
    for x, w, call, depth in ((torch.randn(m, k, generator=g), wd.t(), qlin.fp8_linear, k),
                              (torch.randn(m, n, generator=g), wd, qlin.fp8_linear_grad_input, n)):
        xd = A.dequantize(*A.quantize(x)).cuda()
        ref, size = (xd @ w).cpu(), (xd.abs() @ w.abs()).cpu()
        xc = x.cuda()
        y = call(xc, qc, sc)
        assert A.finite(y) and A.max_excess(y, ref, A.linear_bound(ref, size, depth, F32)) <= 1.0
        for _ in range(5):
            assert torch.equal(call(xc, qc, sc), y)
    _clean(qlin)


def test_non_finite_inputs_stay_in_their_rows(qlin):
    m, n, k = 1700, 1650, 272
    g = torch.Generator(device="cuda").manual_seed(0)
    x, (q, s) = torch.randn(m, k, generator=g, device="cuda").to(BF16), _weight(n, k, g)
    clean = qlin.fp8_linear(x, q, s)
    x[300, 5], x[m - 1, k - 1] = float("nan"), float("inf")
    y = qlin.fp8_linear(x, q, s)
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[300] = keep[m - 1] = False
    assert torch.equal(y[keep], clean[keep]) and not bool(torch.isfinite(y[~keep].float()).any())
    _clean(qlin)
