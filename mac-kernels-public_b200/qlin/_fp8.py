"""Block-scaled 8-bit floating point linears: W in e4m3 with one fp32 scale per block of 128 x 128.

  fp8_linear(x, qdata, scale, bias, out_dtype)             y = x . W^T + bias
  fp8_linear_grad_input(dy, qdata, scale, out_dtype)       dx = dy . W, the weight frozen
  fp8_linear_trainable(x, qdata, scale, bias)              the two under autograd
  quantize_fp8_rowwise(x)                                  the activations' quantizer on its own

The activations (and dy) are brought to e4m3 with one scale per row and block of 128 columns; each block's
products are summed in fp32 on the tensor cores and scaled into the fp32 sum over the blocks.  The
reference has no 8-bit floating point format; names and argument order follow its int8_linear family
(bench/bench_ck01_int8.py:57, bench/bench_int8_backward.py:52,70).
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from ._fast import native
from ._lib import QlinDecline, check, lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BLOCK = 128


def _weight(what, qdata, scale):
    """(qdata with aligned contiguous rows, scale fp32 with a unit inner stride) of a checked weight."""
    if not qdata.is_cuda or not scale.is_cuda:
        raise NotImplementedError("qlin runs on CUDA tensors only (there is no CPU path)")
    if scale.device != qdata.device:
        raise ValueError(f"{what}: weight on {qdata.device}, scale on {scale.device}")
    if qdata.dtype != torch.float8_e4m3fn or qdata.dim() != 2:
        raise QlinDecline(1, f"{what}: qdata must be a 2-D float8_e4m3fn tensor")
    n, k = qdata.shape
    if scale.dim() != 2 or scale.shape[0] != -(-n // _BLOCK) or scale.shape[1] != -(-k // _BLOCK):
        raise ValueError(f"{what}: scale must be [{-(-n // _BLOCK)}, {-(-k // _BLOCK)}] for a weight of [{n}, {k}], "
                         f"got {list(scale.shape)}")
    if qdata.stride(1) != 1 or qdata.stride(0) % 16 or qdata.stride(0) < k or qdata.data_ptr() % 16:
        qdata = qdata.clone(memory_format=torch.contiguous_format)
    if scale.dtype != torch.float32:
        scale = scale.float()
    if scale.stride(1) != 1 or scale.stride(0) < scale.shape[1]:
        scale = scale.contiguous()
    return qdata, scale


def _rows(x):
    """x as [rows, features] with a unit inner stride."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or x2.stride(0) < x2.shape[1]:
        x2 = x2.contiguous()
    return x2


def _same_device(what, x, qdata):
    if not x.is_cuda or not qdata.is_cuda:
        raise NotImplementedError("qlin runs on CUDA tensors only (there is no CPU path)")
    if x.device != qdata.device:
        raise ValueError(f"{what}: activations on {x.device}, weight on {qdata.device}")


def fp8_linear(x, qdata, scale, bias=None, out_dtype=None):
    """y = x . W^T + bias for the weight W = qdata (float8_e4m3fn [N, K]) times `scale` (fp32
    [ceil(N/128), ceil(K/128)], one per block).  x [..., K] in f32, f16 or bf16, quantized per row and block of
    128 columns; K a multiple of 16.  Returns [..., N] in out_dtype (default x's)."""
    if out_dtype is None or out_dtype == x.dtype:
        y = native.fp8_linear(x, qdata, scale, bias)
        if y is not None:
            return y
    _same_device("fp8_linear", x, qdata)
    q, sc = _weight("fp8_linear", qdata, scale)
    n, k = q.shape
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"fp8_linear: x has {x.shape[-1] if x.dim() else 0} features, weight has {k}")
    out_dtype = out_dtype or x.dtype
    if x.dtype not in _DT or out_dtype not in _DT:
        raise QlinDecline(1, "fp8_linear: x and y must be f32, f16 or bf16")
    if bias is not None:
        if bias.numel() != n or bias.device != x.device:
            raise ValueError(f"fp8_linear: the bias needs {n} values on {x.device}")
        bias = bias.reshape(n).contiguous()
        if bias.dtype not in _DT:
            bias = bias.float()
    y = torch.empty(*x.shape[:-1], n, dtype=out_dtype, device=x.device)
    if y.numel() == 0:
        return y
    if k == 0:
        return y.zero_() if bias is None else y.copy_(bias.expand_as(y))
    x2 = _rows(x)
    m = x2.shape[0]
    with torch.cuda.device(x.device):
        nws = lib.qlin_fp8_linear_workspace(m, n, k)
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws else None
        check(lib.qlin_fp8_linear(x2.data_ptr(), _DT[x2.dtype], m, k, x2.stride(0), q.data_ptr(), q.stride(0), n,
                                  sc.data_ptr(), sc.stride(0), None if bias is None else bias.data_ptr(),
                                  0 if bias is None else _DT[bias.dtype], y.data_ptr(), _DT[out_dtype], n,
                                  None if ws is None else ws.data_ptr(), nws,
                                  torch.cuda.current_stream().cuda_stream), "qlin_fp8_linear")
    return y


def fp8_linear_grad_input(dy, qdata, scale, out_dtype=None):
    """dx = dy . W for the frozen weight of fp8_linear; dy [..., N] float, quantized per row and block of 128 of
    its N columns, returns [..., K] in out_dtype (default dy's).  The weight is read as it is stored."""
    if out_dtype is None or out_dtype == dy.dtype:
        dx = native.fp8_linear_grad_input(dy, qdata, scale)
        if dx is not None:
            return dx
    _same_device("fp8_linear_grad_input", dy, qdata)
    q, sc = _weight("fp8_linear_grad_input", qdata, scale)
    n, k = q.shape
    if dy.dim() == 0 or dy.shape[-1] != n:
        raise ValueError(f"fp8_linear_grad_input: dy has {dy.shape[-1] if dy.dim() else 0} features, weight has {n} "
                         "rows")
    out_dtype = out_dtype or dy.dtype
    if dy.dtype not in _DT or out_dtype not in _DT:
        raise QlinDecline(1, "fp8_linear_grad_input: dy and dx must be f32, f16 or bf16")
    dx = torch.empty(*dy.shape[:-1], k, dtype=out_dtype, device=dy.device)
    if dx.numel() == 0:
        return dx
    if n == 0:
        return dx.zero_()
    dy2 = _rows(dy)
    m = dy2.shape[0]
    with torch.cuda.device(dy.device):
        nws = lib.qlin_fp8_linear_grad_input_workspace(m, n, k)
        ws = torch.empty(nws, dtype=torch.uint8, device=dy.device) if nws else None
        check(lib.qlin_fp8_linear_grad_input(dy2.data_ptr(), _DT[dy2.dtype], m, n, dy2.stride(0), q.data_ptr(),
                                             q.stride(0), k, sc.data_ptr(), sc.stride(0), dx.data_ptr(),
                                             _DT[out_dtype], k, None if ws is None else ws.data_ptr(), nws,
                                             torch.cuda.current_stream().cuda_stream), "qlin_fp8_linear_grad_input")
    return dx


def quantize_fp8_rowwise(x):
    """(q float8_e4m3fn [M, K], scale fp32 [M, ceil(K/128)]) of x [..., K]: per row and block of 128 columns, in
    fp32, a = max(max |x|, 2^-100), q = e4m3(x * (448 / a)), scale = a / 448.  The scales lie block by block
    (scale.t() is contiguous) and the rows of q 128-byte aligned."""
    if not x.is_cuda:
        raise NotImplementedError("qlin runs on CUDA tensors only (there is no CPU path)")
    if x.dim() == 0 or x.dtype not in _DT:
        raise QlinDecline(1, "quantize_fp8_rowwise: x must be rows of f32, f16 or bf16")
    k = x.shape[-1]
    m = x.numel() // k if k else 0
    blocks = -(-k // _BLOCK)
    q = torch.empty(m, blocks * _BLOCK, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(blocks, m, dtype=torch.float32, device=x.device)
    if q.numel():
        x2 = _rows(x)
        with torch.cuda.device(x.device):
            check(lib.qlin_quantize_rows_fp8(x2.data_ptr(), _DT[x2.dtype], m, k, x2.stride(0), q.data_ptr(),
                                             blocks * _BLOCK, s.data_ptr(), m,
                                             torch.cuda.current_stream().cuda_stream), "qlin_quantize_rows_fp8")
    return q[:, :k], s.t()


class _Fp8Trainable(torch.autograd.Function):
    """y = fp8_linear(x, ...); backward gives x (and a bias that requires grad) their gradients, the
    weight stays frozen."""

    @staticmethod
    def forward(ctx, x, qdata, scale, bias):
        ctx.save_for_backward(qdata, scale)
        ctx.x_dtype = x.dtype
        ctx.bias = None if bias is None else (bias.dtype, bias.shape)
        return fp8_linear(x, qdata, scale, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        qdata, scale = ctx.saved_tensors
        gx = gb = None
        if ctx.needs_input_grad[0]:
            gx = fp8_linear_grad_input(gy, qdata, scale, out_dtype=ctx.x_dtype)
        if ctx.bias is not None and ctx.needs_input_grad[3]:
            gb = gy.reshape(math.prod(gy.shape[:-1]), gy.shape[-1]).float().sum(0).to(ctx.bias[0]).reshape(ctx.bias[1])
        return gx, None, None, gb


def fp8_linear_trainable(x, qdata, scale, bias=None):
    """fp8_linear with autograd: gradients for x (and bias), none for the frozen weight."""
    return _Fp8Trainable.apply(x, qdata, scale, bias)
