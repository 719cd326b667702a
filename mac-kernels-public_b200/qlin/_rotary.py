"""Rotary positions with several axes, and the RMS norm of every query and key head with the position rotation in
the same pass: what a diffusion transformer's attention does between its quantized projections and the
attention itself.

  rotary_table(positions, axes_dim, theta)                       cosines and sines, once per sampling run
  qk_norm_rotary(q, k, q_weight, k_weight, table, ...)           one kernel for both
  qk_norm_rotary_backward(dq, dk, q, k, ...)                     gradients of q, k and the two weights
  qk_norm_rotary_trainable(q, k, q_weight, k_weight, table, ...) the two under autograd

No counterpart in the reference, whose hosts run these steps as separate framework ops.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from ._fast import native
from ._lib import QlinDecline, check, lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_POS = {torch.float32: 0, torch.int32: 5, torch.int64: 7}
_Strides = ctypes.c_int64 * 3


def rotary_table(positions, axes_dim, theta=10000.0):
    """fp32 [..., sum(axes_dim) / 2, 2], (cos, sin) of each pair's angle: positions [..., A] (float32, int32 or
    int64) holds a coordinate per axis, axis a turns axes_dim[a] / 2 pairs, pair i of it by
    positions[..., a] * theta ** (-2 i / axes_dim[a]); theta is at least 1."""
    out = native.rotary_table(positions, axes_dim, float(theta))
    if out is not None:
        return out
    if not positions.is_cuda:
        raise NotImplementedError("qlin runs on CUDA tensors only (there is no CPU path)")
    axes = len(axes_dim)
    if positions.dim() == 0 or positions.shape[-1] != axes or axes == 0:
        raise ValueError(f"rotary_table: positions need {axes} coordinates each, got {list(positions.shape)}")
    if positions.dtype not in _POS:
        raise QlinDecline(1, "rotary_table: positions must be float32, int32 or int64")
    if any(d < 0 or d % 2 for d in axes_dim):
        raise ValueError(f"rotary_table: every axis needs an even number of dimensions, got {list(axes_dim)}")
    pos = positions.contiguous()
    out = torch.empty(*pos.shape[:-1], sum(axes_dim) // 2, 2, dtype=torch.float32, device=pos.device)
    if out.numel():
        with torch.cuda.device(pos.device):
            check(lib.qlin_rotary_table(pos.data_ptr(), _POS[pos.dtype], pos.numel() // axes, axes,
                                        (ctypes.c_int32 * axes)(*axes_dim), float(theta), out.data_ptr(),
                                        torch.cuda.current_stream().cuda_stream), "qlin_rotary_table")
    return out


def _heads(what, name, x, like=None):
    """x checked as [B, L, H, D] with a unit inner stride (copied where it has none)."""
    if not x.is_cuda:
        raise NotImplementedError("qlin runs on CUDA tensors only (there is no CPU path)")
    if x.dim() != 4 or x.dtype not in _DT:
        raise QlinDecline(1, f"{what}: {name} must be [batch, tokens, heads, head_dim] in f32, f16 or bf16")
    if like is not None and (x.dtype != like.dtype or x.device != like.device or x.shape[:2] != like.shape[:2]
                             or x.shape[3] != like.shape[3]):
        raise ValueError(f"{what}: {name} {list(x.shape)} {x.dtype} on {x.device} does not go with "
                         f"{list(like.shape)} {like.dtype} on {like.device}")
    return x if x.stride(3) == 1 else x.contiguous()


def _weights(what, q, q_weight, k_weight):
    """The two weights contiguous and of one dtype (None stays None), and that dtype's code."""
    got = [w for w in (q_weight, k_weight) if w is not None]
    for w in got:
        if w.dtype not in _DT or w.device != q.device or w.shape != (q.shape[3],):
            raise ValueError(f"{what}: a weight needs {q.shape[3]} values in f32, f16 or bf16 on {q.device}, got "
                             f"{list(w.shape)} {w.dtype} on {w.device}")
    if not got:
        return None, None, 0
    if len(got) == 2 and got[0].dtype != got[1].dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    return (None if q_weight is None else q_weight.contiguous(), None if k_weight is None else k_weight.contiguous(),
            _DT[(k_weight if q_weight is None else q_weight).dtype])


def _table(what, q, table):
    """(table contiguous within each batch, floats between batches, pairs)."""
    b, l, _, d = q.shape
    ok = table.dtype == torch.float32 and table.device == q.device and table.dim() in (3, 4) and table.shape[-1] == 2 \
        and table.shape[-3] == l and 2 * table.shape[-2] <= d and (table.dim() == 3 or table.shape[0] in (1, b))
    if not ok:
        raise ValueError(f"{what}: the table must be fp32 [tokens, pairs, 2] or [batch, tokens, pairs, 2] for "
                         f"{list(q.shape)} on {q.device}, got {list(table.shape)} {table.dtype} on {table.device}")
    pairs = table.shape[-2]
    if table.dim() == 4 and table.shape[0] == 1:
        table = table[0]
    if table.dim() == 3:
        return table.contiguous(), 0, pairs
    if table.stride(3) != 1 or table.stride(2) != 2 or table.stride(1) != 2 * pairs or \
            (b > 1 and table.stride(0) != 0 and table.stride(0) < l * pairs * 2):
        table = table.contiguous()
    return table, table.stride(0) if b > 1 else 0, pairs


def _overlaps_itself(x):
    """Whether rows of x [B, L, H, D] share memory, by the strides from the smallest on (layouts whose rows interleave
    without nesting count as overlapping too)."""
    extent = x.shape[3]
    for step, size in sorted((x.stride(i), x.shape[i]) for i in range(3) if x.shape[i] > 1):
        if step < extent:
            return True
        extent += step * (size - 1)
    return False


def _st(x):
    return _Strides(*x.stride()[:3])


def qk_norm_rotary(q, k, q_weight, k_weight, table, eps=1e-6, interleaved=True, out=None):
    """(q', k'): every head's row times its inverse root mean square and the weight [D] (None: ones), then its
    pairs turned by the token's table entries, in fp32 with one rounding.  q [B, L, Hq, D] and k [B, L, Hk, D] may be
    views of one projection's output.  `table` from rotary_table, [L, P, 2] or [B, L, P, 2] with 2 P <= D; pair i is
    values (2 i, 2 i + 1), or (i, i + P) where interleaved is false; values past 2 P are normed only.  `out`: two
    tensors of the inputs' shapes and dtype to write to, e.g. slices of the buffers of a joint attention (their
    rows may not overlap, nor may they overlap the inputs)."""
    if out is None:
        got = native.qk_norm_rotary(q, k, q_weight, k_weight, table, eps, interleaved)
        if got is not None:
            return got
    what = "qk_norm_rotary"
    q = _heads(what, "q", q)
    k = _heads(what, "k", k, q)
    qw, kw, wdt = _weights(what, q, q_weight, k_weight)
    tab, tab_b, pairs = _table(what, q, table)
    if out is None:
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        qo, ko = out
        for o, x in ((qo, q), (ko, k)):
            if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device or (o.numel() and o.stride(3) != 1):
                raise ValueError(f"{what}: out must have the inputs' shapes, dtype and device and a unit inner stride")
            if o.numel() and _overlaps_itself(o):
                raise ValueError(f"{what}: rows of out overlap (strides {list(o.stride())} for {list(o.shape)})")
    if qo.numel() or ko.numel():
        b, l, hq, d = q.shape
        with torch.cuda.device(q.device):
            check(lib.qlin_qk_norm_rotary(q.data_ptr(), _st(q), k.data_ptr(), _st(k), _DT[q.dtype], b, l, hq,
                                          k.shape[2], d, None if qw is None else qw.data_ptr(),
                                          None if kw is None else kw.data_ptr(), wdt, tab.data_ptr(), tab_b, pairs, eps,
                                          1 if interleaved else 0, qo.data_ptr(), _st(qo), ko.data_ptr(), _st(ko),
                                          torch.cuda.current_stream().cuda_stream), "qlin_qk_norm_rotary")
    return qo, ko


def qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, table, eps=1e-6, interleaved=True):
    """(gradient of q, of k, of q_weight, of k_weight) for the gradients dq, dk of qk_norm_rotary's outputs; a
    weight that is None has None.  The weights' gradients are fp32 sums over all rows, in a fixed order."""
    got = native.qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, table, eps, interleaved)
    if got is not None:
        return got
    what = "qk_norm_rotary_backward"
    q = _heads(what, "q", q)
    k = _heads(what, "k", k, q)
    dq = _heads(what, "dq", dq, q)
    dk = _heads(what, "dk", dk, k)
    if dq.shape != q.shape or dk.shape != k.shape:
        raise ValueError(f"{what}: gradients {list(dq.shape)}, {list(dk.shape)} for {list(q.shape)}, {list(k.shape)}")
    qw, kw, wdt = _weights(what, q, q_weight, k_weight)
    tab, tab_b, pairs = _table(what, q, table)
    b, l, hq, d = q.shape
    hk = k.shape[2]
    gq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    gk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    gqw = None if qw is None else torch.empty_like(qw)
    gkw = None if kw is None else torch.empty_like(kw)
    if d:
        with torch.cuda.device(q.device):
            nws = lib.qlin_qk_norm_rotary_backward_workspace(b, l, hq, hk, d)
            ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
            check(lib.qlin_qk_norm_rotary_backward(
                dq.data_ptr(), _st(dq), dk.data_ptr(), _st(dk), q.data_ptr(), _st(q), k.data_ptr(), _st(k),
                _DT[q.dtype], b, l, hq, hk, d, None if qw is None else qw.data_ptr(),
                None if kw is None else kw.data_ptr(), wdt, tab.data_ptr(), tab_b, pairs, eps, 1 if interleaved else 0,
                gq.data_ptr(), _st(gq), gk.data_ptr(), _st(gk), None if gqw is None else gqw.data_ptr(),
                None if gkw is None else gkw.data_ptr(), None if ws is None else ws.data_ptr(), nws,
                torch.cuda.current_stream().cuda_stream), "qlin_qk_norm_rotary_backward")
    return (gq, gk, None if gqw is None else gqw.to(q_weight.dtype), None if gkw is None else gkw.to(k_weight.dtype))


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table)
        ctx.args = (eps, interleaved)
        return qk_norm_rotary(q, k, q_weight, k_weight, table, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, table = ctx.saved_tensors
        need = ctx.needs_input_grad
        gq, gk, gqw, gkw = qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, table, *ctx.args)
        return (gq if need[0] else None, gk if need[1] else None, gqw if need[2] else None, gkw if need[3] else None,
                None, None, None)


def qk_norm_rotary_trainable(q, k, q_weight, k_weight, table, eps=1e-6, interleaved=True):
    """qk_norm_rotary with autograd: gradients for q, k and the weights, none for the table."""
    return _QkNormRotary.apply(q, k, q_weight, k_weight, table, eps, interleaved)
