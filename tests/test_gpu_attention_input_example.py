"""examples/attention_input.py: the block forward against the same block in fp32 torch, and its training steps."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def _plain(block, x, timestep, table):
    """The block in fp32, from dequantized weights and unquantized activations."""
    def weight(w):
        q, s = w
        n, k = q.shape
        return q.float() * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]

    def rotated(h):
        h = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        c, s = table[None, :, None, :, 0], table[None, :, None, :, 1]
        a, b = h[..., 0::2], h[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)

    x, timestep = x.float(), timestep.float()
    shift, scale = (timestep @ weight(block.modulation).t()).chunk(2, -1)
    h = torch.nn.functional.layer_norm(x, (block.width,)) * (1 + scale[:, None]) + shift[:, None]
    q, k, v = (h @ weight(block.qkv).t()).view(*x.shape[:2], 3, block.heads, block.head_dim).unbind(2)
    q, k = rotated(q), rotated(k)
    a = torch.softmax(torch.einsum("blhd,bmhd->bhlm", q, k) * block.head_dim ** -0.5, -1)
    return x + torch.einsum("bhlm,bmhd->blhd", a, v).reshape(x.shape) @ weight(block.out).t()


def test_block_matches_plain_torch():
    import attention_input as E
    import qlin
    g = torch.Generator(device="cuda").manual_seed(1)
    table = qlin.rotary_table(E.positions(13, 6, 9, "cuda"), E.axes_of(64))
    block = E.Block(4, 64, "cuda", seed=1)
    x = torch.randn(2, 67, 256, generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randn(2, 256, generator=g, device="cuda").to(torch.bfloat16)
    y, ref = block.forward(x, t, table).float(), _plain(block, x, t, table)
    # e4m3 keeps 4 significant bits: 2^-5 rms at most of each projection's input, three projections deep
    delta = (y - x.float()) - (ref - x.float())
    assert float(delta.norm() / (ref - x.float()).norm()) <= 3 * 2.0 ** -5


def test_example_runs_and_its_training_lowers_the_loss():
    import attention_input as E
    y, losses = E.run(tokens=256, text=20, heads=4, head_dim=128, steps=4)
    assert y.shape == (1, 276, 512) and bool(torch.isfinite(y.float()).all())
    assert losses[-1] < losses[0]
    import qlin
    code, where = qlin.device_status()
    assert code == 0, hex(where)
