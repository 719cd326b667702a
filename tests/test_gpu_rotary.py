"""GPU parity of the rotary tables and of the head norm with rotation, forward and backward, against the 64-bit
oracle.  Bounds: the table's angle keeps at most half a unit of the last place of 2^-1 turns plus sincospif's
two units; a normed and rotated value takes at most 16 fp32 roundings of its two terms (the mean of up to 1024 squares
among them), a gradient at most 32 of its terms, and one rounding to the output's type comes on top."""
import itertools

import pytest
import torch

from oracle import attention_input as A

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-6


@pytest.fixture(scope="module")
def qlin():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import qlin as q
    return q


def _table(l, pairs, g, batch=None):
    shape = (l, pairs) if batch is None else (batch, l, pairs)
    a = torch.randn(*shape, generator=g) * 20
    return torch.stack([a.cos(), a.sin()], -1)


# ------------------------------------------------------------------------------------------------ table
@pytest.mark.parametrize("axes", [[64], [16, 56, 56], [44, 42, 42], [2, 0, 6, 8], [256, 256]])
@pytest.mark.parametrize("dtype", [F32, torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [1, 7, 1500])
def test_table_matches_64_bits(qlin, axes, dtype, tokens):
    g = torch.Generator().manual_seed(tokens)
    pos = torch.randint(-200, 20000, (tokens, len(axes)), generator=g)
    pos[0] = 0
    pos = (pos.float() * 0.25 if dtype == F32 else pos).to(dtype)
    got = qlin.rotary_table(pos.cuda(), axes, 10000.0)
    assert got.shape == (tokens, sum(axes) // 2, 2) and got.dtype == F32
    assert float((got.double().cpu() - A.table(pos, axes, 10000.0)).abs().max()) <= 2 * torch.pi * 2.0 ** -25 + 2.0 ** -22
    assert torch.equal(got[0].cpu(), torch.tensor([1.0, 0.0]).expand(sum(axes) // 2, 2))


def test_table_shapes_and_refusals(qlin):
    pos = torch.arange(24, device="cuda").view(2, 4, 3)
    got = qlin.rotary_table(pos, (4, 6, 8), 500.0)
    assert got.shape == (2, 4, 9, 2)
    assert torch.equal(got.view(8, 9, 2), qlin.rotary_table(pos.view(8, 3), [4, 6, 8], 500.0))
    assert torch.equal(qlin.rotary_table(pos.transpose(0, 1), (4, 6, 8), 500.0), got.transpose(0, 1))
    far = qlin.rotary_table(torch.tensor([[2 ** 40 + 1]], device="cuda"), [8])
    ref = A.table(torch.tensor([[2 ** 40 + 1]]), [8], 10000.0)
    # the frequency itself has 53 bits: 2^40 positions leave 2^-13 of a turn times its roundings
    assert float((far.double().cpu() - ref).abs().max()) <= 2 * torch.pi * 2.0 ** (40 - 51)
    nan = qlin.rotary_table(torch.tensor([[float("nan")], [float("inf")], [1.0]], device="cuda"), [4])
    assert bool(torch.isnan(nan[:2]).all()) and A.finite(nan[2])
    assert qlin.rotary_table(torch.empty(0, 2, device="cuda"), [4, 4]).shape == (0, 4, 2)
    assert qlin.rotary_table(torch.zeros(5, 1, device="cuda"), [0]).shape == (5, 0, 2)
    with pytest.raises(ValueError):
        qlin.rotary_table(pos, [4, 4])
    with pytest.raises(ValueError):
        qlin.rotary_table(pos, [4, 5, 4])
    with pytest.raises(qlin.QlinDecline):
        qlin.rotary_table(pos.half(), [4, 4, 4])
    with pytest.raises(qlin.QlinDecline):
        qlin.rotary_table(pos, [400, 400, 4])
    with pytest.raises(qlin.QlinError):
        qlin.rotary_table(pos, [4, 4, 4], theta=-1.0)
    with pytest.raises(NotImplementedError):
        qlin.rotary_table(pos.cpu(), [4, 4, 4])


# ------------------------------------------------------------------------------------------------ forward, backward
# (batch, tokens, q heads, k heads, head dim, pairs): whole and ragged lane groups, part of a head rotated, shared key
# heads, no rotation, heads that only the general kernel takes
SHAPES = [(1, 1, 1, 1, 64, 32), (2, 7, 3, 1, 128, 64), (1, 77, 24, 24, 64, 32), (2, 33, 5, 2, 96, 32), (1, 20, 4, 4, 80, 20),
          (1, 9, 40, 8, 128, 32), (3, 5, 2, 2, 256, 128), (1, 6, 3, 3, 32, 16), (1, 5, 2, 1, 8, 4), (1, 4, 3, 2, 72, 0),
          (1, 6, 2, 2, 100, 50), (2, 3, 2, 1, 30, 15), (1, 3, 2, 2, 512, 256), (1, 2, 1, 2, 1024, 256), (1, 3, 1, 1, 7, 2),
          (1, 300, 17, 3, 128, 64)]


def _case(shape, dtype, seed, weights=True):
    b, l, hq, hk, d, pairs = shape
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, l, hq + 2 * hk, d, generator=g).to(dtype)
    qkv[:, -1, 0] = 0  # a row of zeros
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) if weights else None for _ in range(2)]
    dq, dk = torch.randn(b, l, hq, d, generator=g).to(dtype), torch.randn(b, l, hk, d, generator=g).to(dtype)
    return qkv, q, k, w, dq, dk, g


def _gpu_views(qkv, hq, hk):
    c = qkv.cuda()
    return c[:, :, :hq], c[:, :, hq:hq + hk]


def _forward_check(got, x, w, tab, inter, dtype):
    ref = A.norm_rotary(x, w, tab, EPS, inter)
    xd = x.double()
    v = xd / (xd.square().mean(-1, keepdim=True) + EPS).sqrt() * (1.0 if w is None else w.double())
    bound = A.rotate_abs(v, tab, inter) * 16 * 2.0 ** -23 + A.rounding(ref, dtype) * 1.01
    assert got.dtype == dtype and got.shape == x.shape
    assert A.max_excess(got, ref, bound) <= 1.0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("inter", [True, False])
def test_forward_matches_64_bits(qlin, shape, dtype, inter):
    b, l, hq, hk, d, pairs = shape
    qkv, q, k, w, _, _, g = _case(shape, dtype, 11)
    tab = _table(l, pairs, g)
    qc, kc = _gpu_views(qkv, hq, hk)
    qo, ko = qlin.qk_norm_rotary(qc, kc, w[0].cuda(), w[1].cuda(), tab.cuda(), EPS, inter)
    _forward_check(qo, q, w[0], tab, inter, dtype)
    _forward_check(ko, k, w[1], tab, inter, dtype)


def _backward_check(got, dy, x, w, tab, inter, dtype):
    dx, dw = got
    rdx, rdw, sdx, sdw = A.norm_rotary_backward(dy, x, w, tab, EPS, inter)
    assert dx.dtype == dtype and dx.shape == x.shape
    assert A.max_excess(dx, rdx, sdx * 32 * 2.0 ** -23 + A.rounding(rdx, dtype) * 1.01) <= 1.0
    if w is None:
        assert dw is None
        return
    # a lane sums at most 64 of these shapes' rows one after the other, then 16 lanes' and 32 rows' sums
    assert dw.dtype == w.dtype and dw.shape == w.shape
    assert A.max_excess(dw, rdw, sdw * 128 * 2.0 ** -23 + A.rounding(rdw, w.dtype) * 1.01 + 1e-30) <= 1.0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("inter", [True, False])
def test_backward_matches_64_bits(qlin, shape, dtype, inter):
    b, l, hq, hk, d, pairs = shape
    qkv, q, k, w, dq, dk, g = _case(shape, dtype, 12)
    tab = _table(l, pairs, g)
    qc, kc = _gpu_views(qkv, hq, hk)
    gq, gk, gqw, gkw = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc, kc, w[0].cuda(), w[1].cuda(), tab.cuda(),
                                                    EPS, inter)
    _backward_check((gq, gqw), dq, q, w[0], tab, inter, dtype)
    _backward_check((gk, gkw), dk, k, w[1], tab, inter, dtype)


@pytest.mark.parametrize("inter,d,pairs", [(True, 64, 32), (False, 48, 16), (True, 10, 4)])
def test_gradients_against_differences(qlin, inter, d, pairs):
    """Central differences of the 64-bit forward, step 1e-6: their own error is below 1e-7 of values of order one."""
    b, l, h = 1, 3, 2
    qkv, q, k, w, dq, dk, g = _case((b, l, h, h, d, pairs), F32, 5)
    qkv[:, -1, 0] += 0.5
    tab = _table(l, pairs, g)
    gq, _, gqw, _ = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), q.cuda(), k.cuda(), w[0].cuda(), w[1].cuda(),
                                                 tab.cuda(), EPS, inter)
    f = lambda x, wt: float((A.norm_rotary(x, wt, tab, EPS, inter) * dq.double()).sum())  # noqa: E731
    step = 1e-6
    for hh, i in itertools.product(range(h), range(0, d, 5)):
        e = torch.zeros(b, l, h, d, dtype=torch.float64)
        e[0, 1, hh, i] = step
        num = (f(q.double() + e, w[0]) - f(q.double() - e, w[0])) / (2 * step)
        assert abs(num - float(gq[0, 1, hh, i])) <= 1e-4
    for i in range(0, d, 5):
        e = torch.zeros(d, dtype=torch.float64)
        e[i] = step
        num = (f(q, w[0].double() + e) - f(q, w[0].double() - e)) / (2 * step)
        assert abs(num - float(gqw[i])) <= 1e-4


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("inter", [True, False])
def test_layouts(qlin, dtype, inter):
    """Heads before tokens, one value off every boundary, tables per batch, expanded inputs, given outputs, no
    weights: all as the plain layout."""
    b, l, hq, hk, d, pairs = 2, 19, 6, 3, 64, 24
    qkv, q, k, w, dq, dk, g = _case((b, l, hq, hk, d, pairs), dtype, 3)
    tab = _table(l, pairs, g)
    wc = [x.cuda() for x in w]
    args = (wc[0], wc[1], tab.cuda(), EPS, inter)
    qc, kc = q.contiguous().cuda(), k.contiguous().cuda()
    ref = qlin.qk_norm_rotary(qc, kc, *args)
    bref = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc, kc, *args)

    def same(a, b_, tol):
        for x, y in zip(a, b_):
            assert float((x.float() - y.float()).abs().max()) <= tol * float(y.float().abs().max())

    tol = 2.0 ** -20 if dtype == F32 else 2.0 ** -7
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (qc, kc)]
    same(qlin.qk_norm_rotary(*heads_first, *args), ref, tol)
    gf = [x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (dq, dk)]
    same(qlin.qk_norm_rotary_backward(*gf, *heads_first, *args), bref, tol)
    off = []
    for x in (qc, kc, dq.cuda(), dk.cuda()):
        wide = torch.zeros(*x.shape[:3], d + 1, dtype=dtype, device="cuda")
        wide[..., 1:] = x
        off.append(wide[..., 1:])
    same(qlin.qk_norm_rotary(off[0], off[1], *args), ref, tol)
    same(qlin.qk_norm_rotary_backward(off[2], off[3], off[0], off[1], *args), bref, tol)
    spread = [torch.stack([x, x], -1)[..., 0] for x in (qc, kc)]  # no unit inner stride
    same(qlin.qk_norm_rotary(*spread, *args), ref, tol)
    # tables per batch, shared through a size or a stride of one
    per = _table(l, pairs, g, b)
    for t in (per.cuda(), torch.stack([per, per], 1).cuda()[:, 1]):
        got = qlin.qk_norm_rotary(qc, kc, wc[0], wc[1], t, EPS, inter)
        _forward_check(got[0], q, w[0], per, inter, dtype)
        gb = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc, kc, wc[0], wc[1], t, EPS, inter)
        _backward_check((gb[0], gb[2]), dq, q, w[0], per, inter, dtype)
    for t in (tab.cuda()[None], tab.cuda()[None].expand(b, -1, -1, -1)):
        got = qlin.qk_norm_rotary(qc, kc, wc[0], wc[1], t, EPS, inter)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    # expanded inputs and gradients
    one = qlin.qk_norm_rotary(qc[:1].expand(b, -1, -1, -1), kc[:, :, :1].expand(-1, -1, hk, -1), *args)
    assert torch.equal(one[0][1], ref[0][0]) and torch.equal(one[1][:, :, 2], ref[1][:, :, 0])
    flat = qlin.qk_norm_rotary_backward(torch.ones((), dtype=dtype, device="cuda").expand(b, l, hq, d), dk.cuda(), qc, kc,
                                        *args)
    full = qlin.qk_norm_rotary_backward(torch.ones(b, l, hq, d, dtype=dtype, device="cuda"), dk.cuda(), qc, kc, *args)
    for x, y in zip(flat, full):
        assert float((x.float() - y.float()).abs().max()) <= tol * float(y.float().abs().max())
    # outputs inside a joint buffer; what lies around them stays
    joint = torch.full((b, l + 5, hq, d), 7.0, dtype=dtype, device="cuda")
    jk = torch.full((b, hk, l + 5, d), 7.0, dtype=dtype, device="cuda")
    got = qlin.qk_norm_rotary(qc, kc, *args, out=(joint[:, 5:], jk.transpose(1, 2)[:, :l]))
    assert torch.equal(joint[:, 5:], ref[0]) and torch.equal(jk[:, :, :l].transpose(1, 2), ref[1])
    assert got[0].data_ptr() == joint[:, 5:].data_ptr()
    assert bool((joint[:, :5] == 7).all()) and bool((jk[:, :, l:] == 7).all())
    # no weights, one weight, weights of another type
    got = qlin.qk_norm_rotary(qc, kc, None, None, tab.cuda(), EPS, inter)
    _forward_check(got[0], q, None, tab, inter, dtype)
    gb = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc, kc, None, wc[1], tab.cuda(), EPS, inter)
    _backward_check((gb[0], gb[2]), dq, q, None, tab, inter, dtype)
    _backward_check((gb[1], gb[3]), dk, k, w[1], tab, inter, dtype)
    mixed = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc, kc, wc[0].float(), wc[1].half(), tab.cuda(), EPS, inter)
    assert mixed[2].dtype == F32 and mixed[3].dtype == F16
    _backward_check((mixed[0], mixed[2]), dq, q, w[0].float(), tab, inter, dtype)


def test_empty_sizes_give_empty_outputs_and_zero_weight_gradients(qlin):
    w = torch.ones(64, device="cuda")
    for b, l, hq, hk in ((0, 4, 2, 2), (2, 0, 2, 2), (1, 3, 0, 2), (1, 3, 2, 0), (1, 3, 0, 0)):
        q, k = torch.randn(b, l, hq, 64, device="cuda"), torch.randn(b, l, hk, 64, device="cuda")
        t = _table(l, 32, torch.Generator().manual_seed(0)).cuda()
        qo, ko = qlin.qk_norm_rotary(q, k, w, w, t)
        assert qo.shape == q.shape and ko.shape == k.shape and A.finite(qo) and A.finite(ko)
        gq, gk, gqw, gkw = qlin.qk_norm_rotary_backward(q, k, q, k, w, w, t)
        assert gq.shape == q.shape and A.finite(gk)
        if b * l * hq == 0:
            assert bool((gqw == 0).all())
        if b * l * hk == 0:
            assert bool((gkw == 0).all())


def test_non_finite_rows_stay_alone(qlin):
    q = torch.randn(1, 8, 4, 128, device="cuda")
    k = torch.randn(1, 8, 4, 128, device="cuda")
    w = torch.ones(128, device="cuda")
    t = _table(8, 64, torch.Generator().manual_seed(0)).cuda()
    ref = qlin.qk_norm_rotary(q, k, w, w, t)
    q2 = q.clone()
    q2[0, 3, 1, 5] = float("inf")
    q2[0, 4, 2, 7] = float("nan")
    got = qlin.qk_norm_rotary(q2, k, w, w, t)
    keep = torch.ones(1, 8, 4, dtype=torch.bool, device="cuda")
    keep[0, 3, 1] = keep[0, 4, 2] = False
    assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[1], ref[1])
    assert bool(torch.isnan(got[0][0, 3, 1]).any()) and bool(torch.isnan(got[0][0, 4, 2]).all())


def test_tokens_past_32_bit_offsets(qlin):
    g = torch.Generator().manual_seed(0)
    l, h, d = 3, 2, 64
    x = torch.randn(1, l, h, d, generator=g).to(BF16).cuda()
    w = torch.ones(d, dtype=BF16, device="cuda")
    t = _table(l, 32, g).cuda()
    store = torch.empty(2 * (2 ** 30 + 64) + 2 ** 20, dtype=BF16, device="cuda")
    far = store.as_strided((1, l, h, d), (0, 2 ** 30 + 64, d, 1), 0)
    far.copy_(x)
    for inter in (True, False):
        ref = qlin.qk_norm_rotary(x, x, w, w, t, EPS, inter)
        got = qlin.qk_norm_rotary(far, far, w, w, t, EPS, inter)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        bref = qlin.qk_norm_rotary_backward(x, x, x, x, w, w, t, EPS, inter)
        back = qlin.qk_norm_rotary_backward(far, x, far, x, w, w, t, EPS, inter)
        assert all(torch.equal(a, b) for a, b in zip(back, bref))
    del store, far
    torch.cuda.empty_cache()


def test_trainable_stream_and_repeats(qlin):
    b, l, hq, hk, d, pairs = 2, 500, 8, 2, 128, 64
    qkv, q, k, w, dq, dk, g = _case((b, l, hq, hk, d, pairs), BF16, 8)
    tab = _table(l, pairs, g).cuda()
    qc, kc = (x.contiguous().cuda().requires_grad_(True) for x in (q, k))
    wc = [x.cuda().requires_grad_(True) for x in w]
    qo, ko = qlin.qk_norm_rotary_trainable(qc, kc, wc[0], wc[1], tab)
    torch.autograd.backward([qo, ko], [dq.cuda(), dk.cuda()])
    ref = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc.detach(), kc.detach(), wc[0].detach(), wc[1].detach(), tab)
    for a, r in zip((qc.grad, kc.grad, wc[0].grad, wc[1].grad), ref):
        assert torch.equal(a, r)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = qlin.qk_norm_rotary_backward(dq.cuda(), dk.cuda(), qc.detach(), kc.detach(), wc[0].detach(),
                                             wc[1].detach(), tab)
    side.synchronize()
    for a, r in zip(again, ref):
        assert torch.equal(a, r)
    # one output unused: its gradient arrives as zeros
    qc.grad = kc.grad = None
    qlin.qk_norm_rotary_trainable(qc, kc, wc[0], wc[1], tab)[0].float().sum().backward()
    assert bool((kc.grad == 0).all()) and A.finite(qc.grad)


def test_refusals(qlin):
    q = torch.zeros(1, 4, 2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    t = torch.zeros(4, 32, 2, device="cuda")
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q[:, :3], w, w, t)
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q.half(), w, w, t)
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q, w[:32], w, t)
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q, w, w, t[:3])
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q, w, w, torch.zeros(4, 33, 2, device="cuda"))
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q, w, w, t.double())
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary(q, q, w, w, t, out=(torch.empty(1, 4, 2, 32, device="cuda"), torch.empty_like(q)))
    with pytest.raises(ValueError):
        qlin.qk_norm_rotary_backward(q[:, :, :1], q, q, q, w, w, t)
    with pytest.raises(qlin.QlinDecline):
        qlin.qk_norm_rotary(q[0], q[0], w, w, t)
    with pytest.raises(qlin.QlinDecline):
        qlin.qk_norm_rotary(q.double(), q.double(), w, w, t)
    with pytest.raises(qlin.QlinDecline):
        qlin.qk_norm_rotary(torch.zeros(1, 4, 1, 2048, device="cuda"), torch.zeros(1, 4, 1, 2048, device="cuda"), None,
                            None, t)
    with pytest.raises(NotImplementedError):
        qlin.qk_norm_rotary(q.cpu(), q.cpu(), w.cpu(), w.cpu(), t.cpu())
