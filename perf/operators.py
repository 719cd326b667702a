"""The attention-input path of a diffusion transformer on block-scaled 8-bit weights, as measured cases:

  linear       y = x . W^T (+ bias) with W in e4m3 and one fp32 scale per 128 x 128 block, x brought to e4m3
               with one scale per row and 128 columns
  linear_grad  dx = dy . W for the same frozen weight, dy brought to e4m3 the same way along its N columns
  table        cosines and sines of rotary positions with several axes (time, height, width)
  qk           RMS norm of every head of q and k with the position rotation in the same pass
  qk_grad      its gradients: dq, dk and those of the two norm weights

`run` computes them in elementary torch operations in fp32, or, where `own` is true, through the package.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100  # rows of zeros: the block's scale stays a normal number
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-kernels-public_b200")


def _qlin():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import qlin
    return qlin


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one timestep embedding through its first projection: the smallest call, all latency
        {"name": "linear_embed_m1", "op": "linear", "m": 1, "k": 256, "n": 5120, "dtype": "bf16", "bias": True},
        # two samples' modulation vectors (six of them at once): the weight's bytes are everything
        {"name": "linear_modulation_m2", "op": "linear", "m": 2, "k": 5120, "n": 30720, "dtype": "bf16", "bias": True},
        # a text prompt of odd length through a context projection
        {"name": "linear_text_m333", "op": "linear", "m": 333, "k": 4096, "n": 5120, "dtype": "f16", "bias": True},
        # image tokens plus text through an MLP's first matrix: the large product
        {"name": "linear_image_m4608", "op": "linear", "m": 4608, "k": 6144, "n": 16384, "dtype": "bf16", "bias": False},
        # adapter training on a short odd batch, ragged widths
        {"name": "linear_grad_m77", "op": "linear_grad", "m": 77, "k": 1552, "n": 1000, "dtype": "f32"},
        # adapter training at image length
        {"name": "linear_grad_m4608", "op": "linear_grad", "m": 4608, "k": 6144, "n": 16384, "dtype": "bf16"},
        # positions of one 512-pixel image behind 512 text tokens, once per sampling run
        {"name": "table_image", "op": "table", "text": 512, "grid": "1x32x32", "axes": "16,56,56", "pos": "f32"},
        # positions of a 480p video clip
        {"name": "table_video", "op": "table", "text": 0, "grid": "21x30x52", "axes": "44,42,42", "pos": "i64"},
        # two short prompts, halves rotated, heads of 64
        {"name": "qk_text_l77", "op": "qk", "b": 2, "l": 77, "hq": 24, "hk": 24, "d": 64, "r": 64, "dtype": "f16",
         "interleaved": False},
        # every token of a 480p clip, forty heads of 128, adjacent pairs rotated: the large pass over memory
        {"name": "qk_video_l32760", "op": "qk", "b": 1, "l": 32760, "hq": 40, "hk": 40, "d": 128, "r": 128,
         "dtype": "bf16", "interleaved": True},
        # training on a short odd length, shared key heads, part of each head rotated, fp32
        {"name": "qk_grad_l333", "op": "qk_grad", "b": 1, "l": 333, "hq": 24, "hk": 8, "d": 96, "r": 64, "dtype": "f32",
         "interleaved": False},
        # training at image length, two samples
        {"name": "qk_grad_l4608", "op": "qk_grad", "b": 2, "l": 4608, "hq": 48, "hk": 48, "d": 128, "r": 128,
         "dtype": "bf16", "interleaved": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "table", "qk", "qk", "qk_grad"])
    if op in ("linear", "linear_grad"):
        while True:
            m, n = _log_int(rng, 1, 8192), _log_int(rng, 100, 30720)
            k = 16 * _log_int(rng, 8, 1024)
            if m * n * k <= 4608 * 6144 * 16384 and n * k <= 5120 * 30720:
                break
        case = {"op": op, "m": m, "k": k, "n": n, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
        if op == "linear":
            case["bias"] = rng.random() < 0.5
        return case
    if op == "table":
        axes = [2 * rng.randint(1, 28) for _ in range(rng.randint(1, 4))]
        sides = [_log_int(rng, 1, 96) for _ in axes]
        while math.prod(sides) > 32760 or math.prod(sides) < 2:
            sides = [_log_int(rng, 1, 96) for _ in axes]
        return {"op": op, "text": rng.choice([0, _log_int(rng, 1, 512)]), "grid": "x".join(map(str, sides)),
                "axes": ",".join(map(str, axes)), "pos": rng.choice(["f32", "i64", "i32"])}
    while True:
        b, l = rng.randint(1, 4), _log_int(rng, 1, 32760)
        d = rng.choice([64, 80, 96, 128, 128, 256])
        hk = rng.randint(1, 48)
        hq = hk * rng.choice([1, 1, 2, 3])
        most = 32760 * 80 * 128 if op == "qk" else 2 * 4608 * 96 * 128
        if b * l * (hq + hk) * d <= most and hq <= 64:
            break
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if dtype == "f32" and b * l * (hq + hk) * d * 2 > most:
        dtype = "bf16"
    return {"op": op, "b": b, "l": l, "hq": hq, "hk": hk, "d": d, "r": rng.choice([d, d, d // 2]), "dtype": dtype,
            "interleaved": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _positions(case, gen):
    """Text tokens at the origin, then the grid's points in row order, each axis from an offset of its own (a crop
    or a continued clip)."""
    sides = [int(s) for s in case["grid"].split("x")]
    grid = torch.stack(torch.meshgrid(*[torch.arange(s, device="cuda") for s in sides], indexing="ij"), -1)
    grid = grid.reshape(-1, len(sides)) + torch.randint(0, 16, (len(sides),), generator=gen, device="cuda")
    text = torch.zeros(case["text"], len(sides), dtype=grid.dtype, device="cuda")
    return torch.cat([text, grid]).to({"f32": torch.float32, "i64": torch.int64, "i32": torch.int32}[case["pos"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] in ("linear", "linear_grad"):
        dt = DTYPES[case["dtype"]]
        n, k, m = case["n"], case["k"], case["m"]
        s["w"] = (randn(n, k) * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s["scale"] = (torch.rand(-(-n // BLOCK), -(-k // BLOCK), generator=gen, device="cuda") + 0.5) * (0.02 / 100)
        if case["op"] == "linear":
            # a few columns far above the rest, as the activations of these models have
            x = randn(m, k)
            x *= 1.0 + 20.0 * (torch.rand(k, generator=gen, device="cuda") < 0.01)
            s["x"] = x.to(dt)
            s["bias"] = (randn(n) * 0.1).to(dt) if case["bias"] else None
        else:
            s["dy"] = (randn(m, n) * 1e-3).to(dt)
    elif case["op"] == "table":
        s["positions"] = _positions(case, gen)
    else:
        dt = DTYPES[case["dtype"]]
        b, l, hq, hk, d, r = (case[x] for x in ("b", "l", "hq", "hk", "d", "r"))
        # queries, keys and values as one projection leaves them
        qkv = randn(b, l, hq + 2 * hk, d).to(dt)
        s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        s["q_weight"], s["k_weight"] = (1 + 0.2 * randn(d)).to(dt), (1 + 0.2 * randn(d)).to(dt)
        angle = randn(l, r // 2) * 20
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1)
        if case["op"] == "qk_grad":
            s["dq"], s["dk"] = (randn(b, l, hq, d) * 1e-2).to(dt), (randn(b, l, hk, d) * 1e-2).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _quantize(x):
    """(e4m3 values as fp32 [M, blocks, 128], scales [M, blocks, 1]) of the rows' 128-column blocks."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    xb = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    amax = xb.abs().amax(-1, keepdim=True).clamp_min(AMAX_FLOOR)
    top = torch.full_like(amax, E4M3_MAX)
    return (xb * (top / amax)).to(torch.float8_e4m3fn).float(), amax / top


def _blocks_of(scale, n, k):
    return scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_linear(x, w, scale, bias, transposed):
    n, k = w.shape
    q, sx = _quantize(x)
    xd = (q * sx).reshape(x.shape[0], -1)[:, :x.shape[1]]
    wd = w.float() * _blocks_of(scale, n, k)
    y = xd @ (wd if transposed else wd.t())
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _plain_table(positions, axes, theta):
    angles = []
    for a, dim in enumerate(axes):
        omega = theta ** (-torch.arange(0, dim, 2, device=positions.device, dtype=torch.float32) / dim)
        angles.append(positions[:, a:a + 1].float() * omega)
    angle = torch.cat(angles, -1)
    return torch.stack([angle.cos(), angle.sin()], -1)


def _pairs(x, r, interleaved):
    """The rotated part's pairs, as two halves."""
    return (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])


def _joined(a, b, rest, interleaved):
    rot = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([rot, rest], -1)


def _rotate(x, table, interleaved, back=False):
    r = 2 * table.shape[-2]
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    s = -s if back else s
    a, b = _pairs(x, r, interleaved)
    return _joined(a * c - b * s, a * s + b * c, x[..., r:], interleaved)


def _plain_qk(x, weight, table, eps, interleaved):
    xf = x.float()
    xn = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps) * weight.float()
    return _rotate(xn, table, interleaved).to(x.dtype)


def _plain_qk_grad(dy, x, weight, table, eps, interleaved):
    xf = x.float()
    rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps)
    xhat = xf * rstd
    g = _rotate(dy.float(), table, interleaved, back=True)
    gw = g * weight.float()
    dx = rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * xhat).sum((0, 1, 2)).to(weight.dtype)


EPS = 1e-6
THETA = 10000.0


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        qlin = _qlin()
        if op == "linear":
            return qlin.fp8_linear(s["x"], s["w"], s["scale"], s["bias"])
        if op == "linear_grad":
            return qlin.fp8_linear_grad_input(s["dy"], s["w"], s["scale"])
        if op == "table":
            return qlin.rotary_table(s["positions"], _axes(case), THETA)
        if op == "qk":
            return qlin.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], eps=EPS,
                                       interleaved=case["interleaved"])
        return qlin.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"],
                                            eps=EPS, interleaved=case["interleaved"])
    if op == "linear":
        return _plain_linear(s["x"], s["w"], s["scale"], s["bias"], False)
    if op == "linear_grad":
        return _plain_linear(s["dy"], s["w"], s["scale"], None, True)
    if op == "table":
        return _plain_table(s["positions"], _axes(case), THETA)
    if op == "qk":
        return (_plain_qk(s["q"], s["q_weight"], s["table"], EPS, case["interleaved"]),
                _plain_qk(s["k"], s["k_weight"], s["table"], EPS, case["interleaved"]))
    dq, dqw = _plain_qk_grad(s["dq"], s["q"], s["q_weight"], s["table"], EPS, case["interleaved"])
    dk, dkw = _plain_qk_grad(s["dk"], s["k"], s["k_weight"], s["table"], EPS, case["interleaved"])
    return dq, dk, dqw, dkw


def work(case):
    op = case["op"]
    if op in ("linear", "linear_grad"):
        m, n, k, size = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
        scales = 4 * -(-n // BLOCK) * -(-k // BLOCK)
        return {"bytes": m * (n + k) * size + n * k + scales + (n * size if case.get("bias") else 0),
                "flops": 2 * m * n * k}
    if op == "table":
        tokens = case["text"] + math.prod(int(g) for g in case["grid"].split("x"))
        axes = _axes(case)
        values = tokens * sum(axes)
        return {"bytes": 4 * values + tokens * len(axes) * (8 if case["pos"] == "i64" else 4), "flops": 2 * values}
    b, l, h, d, r, size = case["b"], case["l"], case["hq"] + case["hk"], case["d"], case["r"], SIZE[case["dtype"]]
    values = b * l * h * d
    if op == "qk":
        return {"bytes": 2 * values * size + l * r * 4 + 2 * d * size, "flops": values * 7}
    return {"bytes": 3 * values * size + l * r * 4 + 4 * d * size, "flops": values * 14}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_linear(s, transposed):
    """The stored e4m3 values and scales follow the definition in its own fp32 steps; the sum over them is in
    64 bits."""
    x = s["dy"] if transposed else s["x"]
    m, depth = x.shape
    pad = -depth % BLOCK
    groups = torch.cat([x.to(torch.float32), x.new_zeros((m, pad), dtype=torch.float32)], 1).reshape(m, -1, BLOCK)
    largest = torch.maximum(groups.abs().max(2).values, torch.tensor(AMAX_FLOOR, device="cuda"))
    top = torch.tensor(E4M3_MAX, device="cuda")
    up = torch.div(top.expand_as(largest), largest)
    values = (groups * up[:, :, None]).to(torch.float8_e4m3fn).double()
    step = torch.div(largest, top.expand_as(largest).contiguous()).double()
    xd = (values * step[:, :, None]).reshape(m, -1)[:, :depth]
    n, k = s["w"].shape
    rows, cols = torch.arange(n, device="cuda") // BLOCK, torch.arange(k, device="cuda") // BLOCK
    wd = s["w"].double()
    wd *= s["scale"].double()[rows][:, cols]
    if transposed:
        return torch.matmul(xd, wd)
    y = torch.matmul(xd, wd.T)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_rotation(table, r, d, interleaved):
    """For each of the d columns: its partner's column, the cosine, and the signed sine that the partner takes."""
    i = torch.arange(d, device="cuda")
    if interleaved:
        pair, first = i // 2, i % 2 == 0
        partner = torch.where(first, i + 1, i - 1)
    else:
        pair, first = i % (r // 2), i < r // 2
        partner = torch.where(first, i + r // 2, i - r // 2)
    turned = i < r
    partner = torch.where(turned, partner, i)
    pair = torch.where(turned, pair, torch.zeros_like(pair))
    c, sn = table[:, :, 0].double()[:, pair], table[:, :, 1].double()[:, pair]
    c = torch.where(turned, c, torch.ones_like(c))
    sn = torch.where(turned, torch.where(first, -sn, sn), torch.zeros_like(sn))
    return partner, c[None, :, None, :], sn[None, :, None, :]


def _exact_qk(x, weight, rotation):
    partner, c, sn = rotation
    xd = x.double()
    xd = xd / (xd.square().sum(-1, keepdim=True) / xd.shape[-1] + EPS).sqrt() * weight.double()
    return xd * c + xd[..., partner] * sn


def _exact_qk_grad(dy, x, weight, rotation):
    """With v = w xhat and y_i = c_i v_i + s_i v_p(i): dv_i = c_i dy_i + s_p(i) dy_p(i)."""
    partner, c, sn = rotation
    g = dy.double()
    g = g * c + (g * sn)[..., partner]
    xd, d = x.double(), x.shape[-1]
    rms = (xd.square().sum(-1, keepdim=True) / d + EPS).sqrt()
    dweight = (g * xd / rms).sum((0, 1, 2))
    g = g * weight.double()
    return g / rms - xd * (g * xd).sum(-1, keepdim=True) / (d * rms ** 3), dweight


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("linear", "linear_grad"):
        return _exact_linear(s, op == "linear_grad")
    if op == "table":
        p = s["positions"].double()
        exponent = [(a, j / dim) for a, dim in enumerate(_axes(case)) for j in range(0, dim, 2)]
        omega = torch.tensor([THETA ** -e for _, e in exponent], dtype=torch.float64, device="cuda")
        angle = p[:, [a for a, _ in exponent]] * omega
        return torch.stack([torch.cos(angle), torch.sin(angle)], 2)
    rotation = _exact_rotation(s["table"], case["r"], case["d"], case["interleaved"])
    if op == "qk":
        return _exact_qk(s["q"], s["q_weight"], rotation), _exact_qk(s["k"], s["k_weight"], rotation)
    dq, dqw = _exact_qk_grad(s["dq"], s["q"], s["q_weight"], rotation)
    dk, dkw = _exact_qk_grad(s["dk"], s["k"], s["k_weight"], rotation)
    return dq, dk, dqw, dkw
