"""Fused Linear: ``y = act(x W^T + b) [+ residual]`` on the tcgen05 GEMM engine.

Reference: ``autograd::linear`` -> ``torch::linear`` (flodl/src/autograd/ops.rs:576,
flodl-sys/ops_training.cpp:400-414). On CUDA the forward is one GEMM whose
epilogue adds the bias, applies GELU (keeping the pre-activation for backward)
and adds the residual; backward is two GEMMs (dgrad with the GELU derivative in
its epilogue, split-K wgrad accumulating into ``weight.grad``) plus the bias
column sum.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from ._common import (C, as_bf16_2d, bf16_shadow, grad_buffer, grad_ready, has_tangent, splitk_for,
                      use_kernels, wants_grad)


def gelu_op(y):
    from .misc import gelu
    return gelu(y)


def wgrad_accumulate(dy2: torch.Tensor, x2: torch.Tensor, weight: torch.Tensor,
                     alpha_t: Optional[torch.Tensor] = None) -> None:
    """weight.grad += dy2^T @ x2  (dy2 [T, N] bf16, x2 [T, K] bf16)."""
    T, N = dy2.shape
    K = x2.shape[1]
    g = grad_buffer(weight)
    ks = splitk_for(N, K, T)
    C().gemm(dy2, x2, g, N, K, T, True, True, flags=C().EPI_ACCUMULATE, k_splits=ks,
             alpha_t=alpha_t)


def bias_grad_accumulate(dy2: torch.Tensor, bias: torch.Tensor) -> None:
    C().colsum(dy2, grad_buffer(bias))


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        K = x.shape[-1]
        N = weight.shape[0]
        x2 = as_bf16_2d(x)
        T = x2.shape[0]
        w16 = bf16_shadow(weight)
        out_f32 = residual is not None
        out = torch.empty((T, N), device=x.device,
                          dtype=torch.float32 if out_f32 else torch.bfloat16)
        flags = 0
        aux = None
        if act == "gelu":
            flags |= C().EPI_GELU
            aux = torch.empty((T, N), device=x.device, dtype=torch.bfloat16)
        res2 = residual.reshape(T, N).float().contiguous() if residual is not None else None
        C().gemm(x2, w16, out, T, N, K, False, False, bias=bias.detach() if bias is not None else None,
                 residual=res2, aux=aux, flags=flags)
        ctx.save_for_backward(x2, weight, bias, aux)
        ctx.act = act
        ctx.x_shape = x.shape
        ctx.x_dtype = x.dtype
        ctx.has_res = residual is not None
        return out.reshape(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x2, weight, bias, aux = ctx.saved_tensors
        N, K = weight.shape
        dy2 = as_bf16_2d(dy)
        T = dy2.shape[0]
        if ctx.act == "gelu":
            # dy of the pre-activation: dy * GELU' (kept by the forward epilogue)
            dh = torch.empty((T, N), device=dy.device, dtype=torch.bfloat16)
            C().mul_bf16(dy2.contiguous(), aux, dh)
            dy2 = dh
        dx = None
        if ctx.needs_input_grad[0]:
            w16 = bf16_shadow(weight)
            out_dtype = torch.float32 if ctx.x_dtype == torch.float32 else torch.bfloat16
            dx2 = torch.empty((T, K), device=dy.device, dtype=out_dtype)
            C().gemm(dy2, w16, dx2, T, K, N, False, True)
            dx = dx2.reshape(ctx.x_shape)
        if wants_grad(weight):
            wgrad_accumulate(dy2, x2, weight)
            grad_ready(weight)
        if bias is not None and wants_grad(bias):
            bias_grad_accumulate(dy2, bias)
            grad_ready(bias)
        dres = dy if ctx.has_res else None
        return dx, None, None, None, dres


class _SmallLinearFn(torch.autograd.Function):
    """Forward and input gradient on the library GEMM (bf16 operands from the
    cached weight shadow, f32 accumulation); the weight and bias gradients
    accumulate into ``.grad`` through the split-K tcgen05 GEMM and fire the
    gradient-ready listeners, exactly as the fused path does."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = as_bf16_2d(x)
        w16 = bf16_shadow(weight)
        b16 = bf16_shadow(bias) if bias is not None else None
        out = F.linear(x2, w16, b16)
        ctx.save_for_backward(x2, weight, bias)
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        return out.reshape(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, weight, bias = ctx.saved_tensors
        dy2 = as_bf16_2d(dy)
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.mm(dy2, bf16_shadow(weight)).reshape(ctx.x_shape)
            if ctx.x_dtype == torch.float32:
                dx = dx.float()
        if wants_grad(weight):
            wgrad_accumulate(dy2, x2, weight)
            grad_ready(weight)
        if bias is not None and wants_grad(bias):
            bias_grad_accumulate(dy2, bias)
            grad_ready(bias)
        return dx, None, None


def _ceil8(n: int) -> int:
    return (n + 7) // 8 * 8


class _PaddedLinearFn(torch.autograd.Function):
    """Linear whose in/out features are not multiples of 8: the TMA-fed GEMMs
    need 16-byte row pitches, so operands are zero-padded to the next multiple
    of 8 (a copy of x, of the bf16 weight and of dy) and the results sliced."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        N, K = weight.shape
        Np, Kp = _ceil8(N), _ceil8(K)
        x2 = F.pad(as_bf16_2d(x), (0, Kp - K))
        w16 = F.pad(bf16_shadow(weight), (0, Kp - K, 0, Np - N))
        T = x2.shape[0]
        bias_p = F.pad(bias.detach().float(), (0, Np - N)) if bias is not None else None
        out = torch.empty((T, Np), device=x.device, dtype=torch.bfloat16)
        C().gemm(x2, w16, out, T, Np, Kp, False, False, bias=bias_p)
        ctx.save_for_backward(x2, w16, weight, bias)
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        return out[:, :N].reshape(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x2, w16, weight, bias = ctx.saved_tensors
        N, K = weight.shape
        Np, Kp = w16.shape
        dyp = F.pad(as_bf16_2d(dy), (0, Np - N)).contiguous()
        T = dyp.shape[0]
        dx = None
        if ctx.needs_input_grad[0]:
            dx2 = torch.empty((T, Kp), device=dy.device, dtype=torch.bfloat16)
            C().gemm(dyp, w16, dx2, T, Kp, Np, False, True)
            dx = dx2[:, :K].to(ctx.x_dtype if ctx.x_dtype == torch.float32 else torch.bfloat16)
            dx = dx.reshape(ctx.x_shape)
        if wants_grad(weight):
            gp = torch.zeros((Np, Kp), device=dy.device, dtype=torch.float32)
            C().gemm(dyp, x2, gp, Np, Kp, T, True, True, flags=C().EPI_ACCUMULATE,
                     k_splits=splitk_for(Np, Kp, T))
            grad_buffer(weight).add_(gp[:N, :K])
            grad_ready(weight)
        if bias is not None and wants_grad(bias):
            C().colsum(dyp[:, :N], grad_buffer(bias))
            grad_ready(bias)
        return dx, None, None


_SMALL = {"tiles": None}


def set_small_gemm_tiles(n: Optional[int]) -> None:
    """Problems with fewer output tiles than ``n`` use the library GEMM
    (``None``: a quarter of the SMs; ``0``: always the tcgen05 kernels)."""
    _SMALL["tiles"] = n


def _few_tiles(M: int, N: int) -> bool:
    """Fewer 128x256 output tiles than the threshold (default: SMs / 4)."""
    if _SMALL["tiles"] is None:
        _SMALL["tiles"] = max(1, C().num_sms() // 4)
    return ((M + 127) // 128) * ((N + 255) // 256) < _SMALL["tiles"]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           act: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    CUDA inputs run the fused tcgen05 path (bf16 operands, f32 accumulation;
    the output is bf16, or f32 when a residual is added). CPU inputs run the
    plain PyTorch composition in the input dtype.
    """
    if not use_kernels(x):
        y = F.linear(x, weight, bias)
        if act == "gelu":
            y = F.gelu(y)
        elif act == "relu":
            y = F.relu(y)
        elif act is not None:
            raise ValueError(f"unsupported fused activation {act!r}")
        if residual is not None:
            y = residual + y
        return y
    if (weight.shape[0] % 8 == 0 and weight.shape[1] % 8 == 0
            and _few_tiles(x.numel() // x.shape[-1], weight.shape[0])):
        # A handful of output tiles would occupy a handful of SMs: the library
        # GEMM's split-K / small-tile kernels spread such problems over the
        # whole GPU. Same precision as the fused path (bf16 operands, f32
        # accumulation, bf16 output).
        y = _SmallLinearFn.apply(x, weight, bias)
        if act == "gelu":
            y = gelu_op(y)
        elif act == "relu":
            y = F.relu(y)
        elif act is not None:
            raise ValueError(f"unsupported fused activation {act!r}")
        return y if residual is None else residual + y
    if weight.shape[0] % 8 or weight.shape[1] % 8:
        y = _PaddedLinearFn.apply(x, weight, bias)
        if act == "gelu":
            y = gelu_op(y)
        elif act == "relu":
            y = F.relu(y)
        elif act is not None:
            raise ValueError(f"unsupported fused activation {act!r}")
        return y if residual is None else residual + y
    if act not in (None, "gelu"):
        y = _LinearFn.apply(x, weight, bias, None, None)
        y = F.relu(y) if act == "relu" else y
        return y if residual is None else residual + y
    return _LinearFn.apply(x, weight, bias, act, residual)


def _rows_gemm(x2, w16, bias, bias16):
    """``x2 @ w16^T + bias`` in bf16 for a row range of a weight's shadow; a few
    output tiles go to the library GEMM, as in :func:`linear`."""
    T, K = x2.shape
    N = w16.shape[0]
    if _few_tiles(T, N):
        return F.linear(x2, w16, bias16)
    out = torch.empty((T, N), device=x2.device, dtype=torch.bfloat16)
    C().gemm(x2, w16, out, T, N, K, False, False, bias=bias)
    return out


def _rows_dgrad(dy2, w16, x):
    T, N = dy2.shape
    K = w16.shape[1]
    if _few_tiles(T, K):
        return torch.mm(dy2, w16).reshape(x[0]).to(x[1])
    dx = torch.empty((T, K), device=dy2.device,
                     dtype=torch.float32 if x[1] == torch.float32 else torch.bfloat16)
    C().gemm(dy2, w16, dx, T, K, N, False, True)
    return dx.reshape(x[0])


class _CrossProjFn(torch.autograd.Function):
    """Query projection of ``x`` and key/value projection of ``memory`` by row
    ranges of one packed weight; the weight's gradients accumulate into their
    ranges of ``.grad`` and its listeners are notified once."""

    @staticmethod
    def forward(ctx, x, memory, weight, bias):
        n = weight.shape[0] // 3
        x2, m2, w16 = as_bf16_2d(x), as_bf16_2d(memory), bf16_shadow(weight)
        b = bias.detach() if bias is not None else None
        b16 = bf16_shadow(bias) if bias is not None else None
        part = (lambda t, lo, hi: t[lo:hi] if t is not None else None)
        q = _rows_gemm(x2, w16[:n], part(b, 0, n), part(b16, 0, n))
        kv = _rows_gemm(m2, w16[n:], part(b, n, None), part(b16, n, None))
        ctx.save_for_backward(x2, m2, weight, bias)
        ctx.like = (x.shape, x.dtype), (memory.shape, memory.dtype)
        return q.reshape(*x.shape[:-1], n), kv.reshape(*memory.shape[:-1], 2 * n)

    @staticmethod
    def backward(ctx, dq, dkv):
        x2, m2, weight, bias = ctx.saved_tensors
        n, K = weight.shape[0] // 3, weight.shape[1]
        dq2, dkv2, w16 = as_bf16_2d(dq), as_bf16_2d(dkv), bf16_shadow(weight)
        dx = _rows_dgrad(dq2, w16[:n], ctx.like[0]) if ctx.needs_input_grad[0] else None
        dm = _rows_dgrad(dkv2, w16[n:], ctx.like[1]) if ctx.needs_input_grad[1] else None
        for dy2, in2, lo, hi in ((dq2, x2, 0, n), (dkv2, m2, n, 3 * n)):
            gw, gb = (grad_buffer(t)[lo:hi] if wants_grad(t) else None for t in (weight, bias))
            if in2.shape[0] == 0:  # an empty memory: zeros, where nothing was before
                continue
            if gw is not None:
                C().gemm(dy2, in2, gw, hi - lo, K, in2.shape[0], True, True,
                         flags=C().EPI_ACCUMULATE, k_splits=splitk_for(hi - lo, K, in2.shape[0]))
            if gb is not None:
                C().colsum(dy2, gb)
        for t in (weight, bias):
            if wants_grad(t):
                grad_ready(t)
        return dx, dm, None, None


def _check_projection(weight, bias, *inputs):
    if weight.dim() != 2 or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
        raise ValueError(f"the weight must be [rows, K] and the bias [rows] (got {tuple(weight.shape)}"
                         f"{'' if bias is None else f' and {tuple(bias.shape)}'})")
    for t in inputs:
        if t.dim() < 1 or t.shape[-1] != weight.shape[1]:
            raise ValueError(f"inputs must be [..., {weight.shape[1]}] (got {tuple(t.shape)})")
    for t in (*inputs[1:], weight, bias):
        if t is not None and t.device != inputs[0].device:
            raise ValueError(f"inputs, weight and bias must be on one device (got {inputs[0].device} and "
                             f"{t.device})")


def cross_projection(x: torch.Tensor, memory: torch.Tensor, weight: torch.Tensor,
                     bias: Optional[torch.Tensor] = None):
    """``(queries of x, keys and values of memory)`` by a packed ``[3N, K]``
    weight's rows: ``x [..., K] -> [..., N]``, ``memory [..., K] -> [..., 2N]``."""
    _check_projection(weight, bias, x, memory)
    if weight.shape[0] % 3:
        raise ValueError(f"the packed weight must be [3N, K] (got {tuple(weight.shape)})")
    n = weight.shape[0] // 3
    if (use_kernels(x) and n % 8 == 0 and weight.shape[1] % 8 == 0 and weight.is_leaf
            and (bias is None or bias.is_leaf)):  # computed ones get theirs through autograd
        return _CrossProjFn.apply(x, memory, weight, bias)
    if use_kernels(x):
        x, memory, weight = x.bfloat16(), memory.bfloat16(), weight.bfloat16()
        bias = bias.bfloat16() if bias is not None else None
    part = (lambda lo, hi: bias[lo:hi] if bias is not None else None)
    return (F.linear(x, weight[:n], part(0, n)), F.linear(memory, weight[n:], part(n, None)))


@torch.no_grad()
def project_rows(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], lo: int,
                 hi: int) -> torch.Tensor:
    """``x @ weight[lo:hi]^T + bias[lo:hi]`` without gradients: one part of a
    packed projection, from the weight's cached bf16 shadow on CUDA."""
    _check_projection(weight, bias, x)
    if not 0 <= lo <= hi <= weight.shape[0]:
        raise ValueError(f"rows {lo} to {hi} of {weight.shape[0]}")
    part = (lambda t: t[lo:hi] if t is not None else None)
    if not use_kernels(x):
        return F.linear(x, weight[lo:hi], part(bias))
    if has_tangent(x, weight, bias):
        b = part(bias)
        return F.linear(x.bfloat16(), weight[lo:hi].bfloat16(), b.bfloat16() if b is not None else None)
    b16 = bf16_shadow(bias) if bias is not None else None
    w16 = bf16_shadow(weight)[lo:hi]
    x2 = as_bf16_2d(x)
    if (hi - lo) % 8 or weight.shape[1] % 8 or lo * weight.shape[1] % 8:
        y = F.linear(x2, w16, part(b16))
    else:
        y = _rows_gemm(x2, w16, part(bias.detach() if bias is not None else None), part(b16))
    return y.reshape(*x.shape[:-1], hi - lo)
