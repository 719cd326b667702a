"""The attention block of a diffusion transformer on block-scaled 8-bit weights, sampled and trained.

    python examples/attention_input.py [--tokens 4096] [--text 512] [--heads 40] [--steps 3]

One block with random weights in e4m3 (one fp32 scale per 128 x 128): the timestep's vector through a projection to a
shift and a scale, the joint projection of text and image tokens to queries, keys and values, RMS norm and rotary
positions of every query and key head, attention (torch's), and the output projection.  The rotary table is built once,
from a text part at the origin and the image's rows and columns.  Sampling runs it forward; training fits an
adapter beside the frozen q/k/v projection, with gradients through the projections, the rotation and the norms.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mac-kernels-public_b200")
if PKG not in sys.path:
    sys.path.insert(0, PKG)

import qlin  # noqa: E402


def quantize_weight(w):
    """(e4m3 [N, K], fp32 [ceil(N/128), ceil(K/128)]) of a weight, once, when it is loaded."""
    n, k = w.shape
    pn, pk = -n % 128, -k % 128
    blocks = torch.nn.functional.pad(w.float(), (0, pk, 0, pn)).view((n + pn) // 128, 128, (k + pk) // 128, 128)
    scale = blocks.abs().amax((1, 3)).clamp_min(2.0 ** -100) / 448.0
    q = (blocks / scale[:, None, :, None]).reshape(n + pn, k + pk)[:n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scale


class Block:
    """Weights of one block; `rank` > 0 adds a trainable low-rank adapter beside the q/k/v projection."""

    def __init__(self, heads, head_dim, device, dtype=torch.bfloat16, rank=0, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * head_dim
        self.heads, self.head_dim, self.width = heads, head_dim, width

        def weight(n, k):
            return quantize_weight(torch.randn(n, k, generator=g, device=device) * k ** -0.5)

        self.modulation, self.qkv, self.out = weight(2 * width, 256), weight(3 * width, width), weight(width, width)
        self.modulation_bias = torch.zeros(2 * width, dtype=dtype, device=device)
        self.q_norm = torch.ones(head_dim, dtype=dtype, device=device)
        self.k_norm = torch.ones(head_dim, dtype=dtype, device=device)
        self.adapter = None
        if rank:
            down = (torch.randn(rank, width, generator=g, device=device) * width ** -0.5).to(dtype)
            self.adapter = [down.requires_grad_(True),
                            torch.zeros(3 * width, rank, dtype=dtype, device=device).requires_grad_(True)]
            self.q_norm.requires_grad_(True)
            self.k_norm.requires_grad_(True)

    def parameters(self):
        return [] if self.adapter is None else [*self.adapter, self.q_norm, self.k_norm]

    def forward(self, x, timestep, table):
        """x [B, L, width], timestep [B, 256] embeddings, table from positions()."""
        train = self.adapter is not None and torch.is_grad_enabled()
        linear = qlin.fp8_linear_trainable if train else qlin.fp8_linear
        norm_rotary = qlin.qk_norm_rotary_trainable if train else qlin.qk_norm_rotary
        shift, scale = linear(timestep, *self.modulation, self.modulation_bias).chunk(2, -1)
        h = torch.nn.functional.layer_norm(x, (self.width,)) * (1 + scale[:, None]) + shift[:, None]
        qkv = linear(h, *self.qkv)
        if self.adapter is not None:
            down, up = self.adapter
            qkv = qkv + (h @ down.t()) @ up.t()
        q, k, v = qkv.view(*x.shape[:2], 3, self.heads, self.head_dim).unbind(2)
        q, k = norm_rotary(q, k, self.q_norm, self.k_norm, table)
        a = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
        return x + linear(a.transpose(1, 2).reshape(x.shape), *self.out)


def positions(text, rows, cols, device):
    """[text + rows * cols, 3]: text at the origin, the image's tokens at (0, row, column)."""
    grid = torch.stack(torch.meshgrid(torch.arange(rows, device=device), torch.arange(cols, device=device), indexing="ij"),
                       -1).reshape(-1, 2)
    image = torch.nn.functional.pad(grid, (1, 0))
    return torch.cat([torch.zeros(text, 3, dtype=image.dtype, device=device), image])


def axes_of(head_dim):
    """A head's pairs over (time, row, column), about 1 : 3.5 : 3.5."""
    side = head_dim * 7 // 16 // 2 * 2
    return [head_dim - 2 * side, side, side]


def run(tokens=4096, text=512, heads=40, head_dim=128, steps=3, device="cuda", seed=0):
    """(sampled activations, losses of the training steps)."""
    g = torch.Generator(device=device).manual_seed(seed)
    rows = int(tokens ** 0.5)
    table = qlin.rotary_table(positions(text, rows, tokens // rows, device), axes_of(head_dim))
    length = table.shape[0]
    block = Block(heads, head_dim, device, seed=seed)
    x = torch.randn(1, length, block.width, generator=g, device=device).to(torch.bfloat16)
    timestep = torch.randn(1, 256, generator=g, device=device).to(torch.bfloat16)
    with torch.no_grad():
        y = x
        for _ in range(steps):
            y = block.forward(y, timestep, table)
    trained = Block(heads, head_dim, device, rank=16, seed=seed)
    target = y
    opt = torch.optim.SGD(trained.parameters(), lr=0.05)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (trained.forward(x, timestep, table).float() - target.float()).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return y, [float(v) for v in losses]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--text", type=int, default=512)
    ap.add_argument("--heads", type=int, default=40)
    ap.add_argument("--steps", type=int, default=3)
    a = ap.parse_args(argv)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    run(a.tokens, a.text, a.heads, steps=1)  # warm up
    start.record()
    y, losses = run(a.tokens, a.text, a.heads, steps=a.steps)
    end.record()
    torch.cuda.synchronize()
    print(f"{a.steps} sampling and {a.steps} training steps of {a.tokens} + {a.text} tokens, {a.heads} heads: "
          f"{start.elapsed_time(end):.1f} ms, rms {float(y.float().square().mean().sqrt()):.3f}, losses "
          + ", ".join(f"{v:.5f}" for v in losses))
    code, where = qlin.device_status()
    return 1 if code else 0


if __name__ == "__main__":
    sys.exit(main())
