"""Chains of small calls, each reading what the one before it wrote, over buffers that the allocator and in-place
updates recycle: kernels that are set up while earlier ones still run give what they give when every call is waited for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qlin():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import qlin as q
    return q


@pytest.fixture(autouse=True)
def _no_fill():
    """Without the fills of fresh allocations, which would stand between the calls of a chain."""
    was = torch.utils.deterministic.fill_uninitialized_memory
    torch.utils.deterministic.fill_uninitialized_memory = False
    yield
    torch.utils.deterministic.fill_uninitialized_memory = was


def _weight(n, k, g):
    q = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.cuda(), (torch.rand(-(-n // 128), -(-k // 128), generator=g) * 4e-4 + 1e-4).cuda()


def _chain(qlin, m, steps, dtype, wait):
    """Products, tables, head norms and their gradients in turn; what every tenth step leaves."""
    g = torch.Generator().manual_seed(m)
    d, heads = 64, 4
    w1, w2 = _weight(heads * d, heads * d, g), _weight(2 * heads * d, heads * d, g)
    x = torch.randn(m, heads * d, generator=g).to(dtype).cuda()
    norm = (1 + 0.1 * torch.randn(d, generator=g)).to(dtype).cuda()
    pos = torch.randint(0, 60, (m, 2), generator=g).cuda()
    fixed = torch.empty(2, 1, m, heads, d, dtype=dtype, device="cuda")  # written again by every step
    step = (lambda: torch.cuda.synchronize()) if wait else (lambda: None)
    kept = []
    for i in range(steps):
        table = qlin.rotary_table(pos, (32, 32))
        step()
        h = qlin.fp8_linear(x, *w2)
        step()
        qk = h.view(1, m, 2, heads, d)
        q, k = qlin.qk_norm_rotary(qk[:, :, 0], qk[:, :, 1], norm, None, table)
        step()
        y = qlin.fp8_linear(q.view(m, -1), *w1)
        step()
        qlin.qk_norm_rotary(y.view(1, m, heads, d), k, None, norm, table, out=(fixed[0], fixed[1]))
        step()
        gq, gk, gw, _ = qlin.qk_norm_rotary_backward(fixed[0], fixed[1], q, k, norm, None, table)
        step()
        x = qlin.fp8_linear_grad_input(gq.view(m, -1), *w1)
        step()
        x, _ = (t.view(m, -1) for t in qlin.qk_norm_rotary(x.view(1, m, heads, d), gk, None, None, table))
        step()
        pos += 1
        step()
        if i % 10 == 0:
            kept.append((x.clone(), gw.clone(), table.clone()))
    torch.cuda.synchronize()
    return kept


@pytest.mark.parametrize("m,dtype", [(1, torch.bfloat16), (9, torch.float16), (77, torch.bfloat16), (333, torch.float32)])
def test_chains_over_recycled_buffers(qlin, m, dtype):
    waited = _chain(qlin, m, 60, dtype, True)
    assert all(bool(torch.isfinite(t.float()).all()) for kept in waited for t in kept)
    for _ in range(3):
        for a, b in zip(_chain(qlin, m, 60, dtype, False), waited):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    code, where = qlin.device_status(reset=True)
    assert code == 0, hex(where)
