"""Layer normalisation of node features on the library's kernels.

``layer_norm(x, layer)`` is the forward of an ``nn.LayerNorm`` over the last
axis, ``(x - mean) / sqrt(var + eps) * weight + bias``, with its backward
(dx, and the weight's and bias's gradients summed over all rows in a fixed
order) in ``egnn_layer_norm_fwd`` / ``egnn_layer_norm_bwd``.  It stands next
to ``linear`` (``nn.Linear`` on the library's node GEMM); ``EGNN`` calls it
between its layers when built with ``node_norm=True``.
"""
from __future__ import annotations

import functools

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _native as nat

DTYPES = {torch.float32: nat.DTYPE_F32, torch.bfloat16: nat.DTYPE_BF16, torch.float16: nat.DTYPE_F16}


@functools.lru_cache(maxsize=256)
def _workspace_size(rows, cols, device):
    return nat.lib().egnn_layer_norm_workspace_size(rows, cols)


def _forward(x, weight, bias, eps, stats):
    """y and, where asked for, the (rows, 2) mean and 1 / sqrt(var + eps)."""
    rows, cols = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    kept = x.new_empty((rows, 2), dtype=torch.float32) if stats else None
    p = weight if weight is not None else bias
    lib = nat.lib()
    with nat.device_of(x):
        nat.check(lib.egnn_layer_norm_fwd(rows, cols, x.data_ptr(), x.stride(0), DTYPES[x.dtype],
                                          None if weight is None else weight.data_ptr(),
                                          None if bias is None else bias.data_ptr(),
                                          nat.DTYPE_F32 if p is None else DTYPES[p.dtype], eps, y.data_ptr(),
                                          kept.data_ptr() if stats else None, nat.stream_ptr()), "egnn_layer_norm_fwd")
    return y, kept


def _backward(ctx, dy):
    x, weight, stats = ctx.saved_tensors
    rows, cols = x.shape
    dy = _rows(dy)
    need_x, need_w, need_b, _ = ctx.needs_input_grad
    pdt = weight.dtype if weight is not None else ctx.bias_dtype or torch.float32
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    dw = torch.empty_like(weight) if need_w else None
    db = x.new_empty(cols, dtype=pdt) if need_b else None
    lib, ws, nbytes = nat.lib(), None, 0
    with nat.device_of(x):
        if need_w or need_b:
            nbytes = _workspace_size(rows, cols, x.get_device())
            ws = x.new_empty(nbytes, dtype=torch.uint8)
        nat.check(lib.egnn_layer_norm_bwd(rows, cols, x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0),
                                          DTYPES[x.dtype], nat.ptr(weight), DTYPES[pdt], stats.data_ptr(), nat.ptr(dx),
                                          nat.ptr(dw), nat.ptr(db), nat.ptr(ws), nbytes, nat.stream_ptr()),
                  "egnn_layer_norm_bwd")
    return dx, dw, db, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        # grad mode is on only under create_graph, where a second derivative has to be refused
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _rows(t):
    """t itself where its rows are dense and do not overlap, else a copy."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def layer_norm(x: torch.Tensor, layer: nn.LayerNorm) -> torch.Tensor:
    """nn.LayerNorm forward (over the last axis) on the library's kernels.

    x: (..., C) float32, bfloat16 or float16 CUDA, C <= 8192; rows may be a
    slice of wider ones.  The layer's weight and bias (either may be absent)
    are float32 or of x's type, both of one type.  The result has x's type;
    statistics and sums are float32.
    """
    device = x.get_device()
    if device < 0:
        raise ValueError("layer_norm takes CUDA tensors (pymolecular_b200 has no CPU path)")
    dtype, size, shape = x.dtype, x.shape, tuple(layer.normalized_shape)
    if dtype not in DTYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {dtype}")
    if len(shape) != 1 or not size or size[-1] != shape[0]:
        raise ValueError(f"x must be (..., C) for a LayerNorm over its last axis alone, got {tuple(size)} and "
                         f"normalized_shape {shape}")
    params = layer._parameters   # spares nn.Module's lookup; a parametrised layer has none there
    weight = params["weight"] if "weight" in params else layer.weight
    bias = params["bias"] if "bias" in params else layer.bias
    needs_grad = x.requires_grad
    for p in (weight, bias):
        if p is None:
            continue
        if p.shape != shape:   # the kernels read C elements of each, and write as many of their gradients
            raise ValueError(f"the layer's parameters must be of its normalized_shape {shape}, got {tuple(p.shape)}")
        if p.get_device() != device:
            raise ValueError(f"the layer's parameters must be on {x.device}, got {p.device}")
        code = p.dtype
        if code is not torch.float32 and code is not dtype or weight is not None and code is not weight.dtype:
            raise TypeError(f"the layer's parameters must be float32 or {dtype}, both of one type, got {p.dtype}")
        needs_grad = needs_grad or p.requires_grad
    rows = x if len(size) == 2 else x.reshape(-1, shape[0])
    if not rows.is_contiguous():
        rows = _rows(rows)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    # Through autograd also what has to be recorded, or refused, without a gradient: dual tensors
    # of forward mode (the Function has no jvp), and tracing, which makes tensors of sizes.
    if needs_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 or type(size[-1]) is not int:
        y = _LayerNormFn.apply(rows, weight, bias, layer.eps)
    else:
        y = _forward(rows, weight, bias, layer.eps, False)[0]
    return y if len(size) == 2 else y.view(size)


__all__ = ["layer_norm"]
