"""CPU oracle, in 64 bits, of the block-scaled 8-bit linear, its input gradient, the rotary tables and the head norm
with rotation.  Only the quantizer works in fp32, because its definition does: a stored code is what fp32
arithmetic makes of the input."""
import math

import torch

BLOCK = 128
FLOOR = 2.0 ** -100


def quantize(x):
    """(e4m3 codes [M, K], fp32 scales [M, blocks]): per row and 128 columns, a = max(max |x|, 2^-100),
    q = e4m3(x * (448 / a)), scale = a / 448, each step rounded to fp32 once."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    f = torch.zeros(m, blocks * BLOCK, dtype=torch.float32)
    f[:, :k] = x.float()
    f = f.view(m, blocks, BLOCK)
    a = torch.maximum(f.abs().amax(2), torch.tensor(FLOOR, dtype=torch.float32))
    top = torch.tensor(448.0, dtype=torch.float32)
    q = (f * (top / a).unsqueeze(2)).to(torch.float8_e4m3fn)
    return q.view(m, -1)[:, :k], a / top


def dequantize(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def weight(q, scale):
    n, k = q.shape
    return q.double() * scale.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def linear(x, q, scale, bias=None, transposed=False):
    """(y, sum of the products' magnitudes): x . W^T + bias, or x . W."""
    xd, wd = dequantize(*quantize(x)), weight(q, scale)
    wd = wd if transposed else wd.t()
    y, size = xd @ wd, xd.abs() @ wd.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def table(positions, axes_dim, theta):
    out = []
    for a, dim in enumerate(axes_dim):
        omega = torch.tensor([theta ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
        angle = positions[..., a].double().unsqueeze(-1) * omega
        out.append(torch.stack([angle.cos(), angle.sin()], -1))
    return torch.cat(out, -2)


def pair_index(dim, pairs, interleaved):
    i = torch.arange(pairs)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)


def rotate(v, tab, interleaved):
    """v [B, L, H, D] in 64 bits, tab [L, P, 2] or [B, L, P, 2]."""
    pairs = tab.shape[-2]
    tab = (tab if tab.dim() == 4 else tab.unsqueeze(0)).double().unsqueeze(3)  # [B or 1, L, P, 1, 2]
    c, s = tab[..., 0].transpose(2, 3), tab[..., 1].transpose(2, 3)  # [., L, 1, P]
    a, b = pair_index(v.shape[-1], pairs, interleaved)
    out = v.clone()
    out[..., a] = v[..., a] * c - v[..., b] * s
    out[..., b] = v[..., a] * s + v[..., b] * c
    return out


def norm_rotary(x, w, tab, eps, interleaved):
    x = x.double()
    v = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return rotate(v if w is None else v * w.double(), tab, interleaved)


def norm_rotary_backward(dy, x, w, tab, eps, interleaved):
    """(dx, dw, size of dx's terms, size of dw's terms)."""
    x, d = x.double(), x.shape[-1]
    back = tab.double().clone()
    back[..., 1] = -back[..., 1]
    g = rotate(dy.double(), back, interleaved)
    gabs = rotate_abs(dy.double(), tab, interleaved)
    w = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    rstd = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    dot = (g * w * x).sum(-1, keepdim=True)
    dx = rstd * (g * w - x * rstd ** 2 * dot / d)
    dw = (g * x * rstd).sum((0, 1, 2))
    dx_size = rstd * (gabs * w.abs() + x.abs() * rstd ** 2 * (gabs * w.abs() * x.abs()).sum(-1, keepdim=True) / d)
    return dx, dw, dx_size, (gabs * x.abs() * rstd).sum((0, 1, 2))


def rotate_abs(v, tab, interleaved):
    """The sum of the magnitudes of the two terms of every rotated value."""
    pairs = tab.shape[-2]
    tab = (tab if tab.dim() == 4 else tab.unsqueeze(0)).double().abs().unsqueeze(3)
    c, s = tab[..., 0].transpose(2, 3), tab[..., 1].transpose(2, 3)
    a, b = pair_index(v.shape[-1], pairs, interleaved)
    out = v.abs().clone()
    out[..., a] = v[..., a].abs() * c + v[..., b].abs() * s
    out[..., b] = v[..., a].abs() * s + v[..., b].abs() * c
    return out


HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rounding(y, dtype):
    """What one rounding to dtype may move each value of y by."""
    return y.abs() * HALF_ULP[dtype] + SMALLEST[dtype]


def linear_bound(y, size, depth, dtype):
    """Products of e4m3 values are exact in fp32.  A block's 128 are summed by the tensor core, whose partial sums
    may lose up to one unit of the last place of 24 bits with each of them (2^-17 of the magnitudes); each of the
    blocks' sums is then scaled and added with two fp32 roundings, and the scales' product has a third."""
    blocks = -(-depth // BLOCK)
    return size * (2.0 ** -16 + (blocks + 3) * 2.0 ** -23) + rounding(y, dtype) * 1.01


def max_excess(got, ref, bound):
    """The largest |got - ref| / bound."""
    d = (got.double().cpu() - ref).abs()
    return float((d / bound).max()) if d.numel() else 0.0


def finite(x):
    return bool(torch.isfinite(x.float()).all()) and not math.isnan(float(x.float().sum())) if x.numel() else True
