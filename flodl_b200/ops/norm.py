"""Fused LayerNorm on CUDA (one kernel forward, one kernel backward).

Reference: ``autograd::layer_norm`` -> ``at::native_layer_norm``
(flodl/src/autograd/ops.rs:629, flodl-sys/ops_tensor.cpp:580-600).
The backward accumulates ``weight.grad``/``bias.grad`` in the same pass as the
input gradient and notifies the gradient-ready listeners.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from ._common import C, grad_buffer, grad_ready, use_kernels, wants_grad


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_bf16):
        xc = x.contiguous()
        Cdim = xc.shape[-1]
        rows = xc.numel() // Cdim
        mean = torch.empty(rows, device=x.device, dtype=torch.float32)
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        if out_bf16 or x.dtype == torch.bfloat16:
            y = torch.empty(xc.shape, device=x.device, dtype=torch.bfloat16)
            C().ln_fwd(xc, weight.detach() if weight is not None else None,
                       bias.detach() if bias is not None else None, y, None, mean, rstd, eps)
        else:
            y = torch.empty(xc.shape, device=x.device, dtype=torch.float32)
            C().ln_fwd(xc, weight.detach() if weight is not None else None,
                       bias.detach() if bias is not None else None, None, y, mean, rstd, eps)
        ctx.save_for_backward(xc, weight, bias, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, weight, bias, mean, rstd = ctx.saved_tensors
        dy16 = dy.contiguous()
        if dy16.dtype != torch.bfloat16:
            t = torch.empty(dy16.shape, device=dy.device, dtype=torch.bfloat16)
            C().cast_f32_bf16(dy16.float(), t)
            dy16 = t
        dx_f32 = dx_bf16 = None
        if xc.dtype == torch.bfloat16:
            dx_bf16 = torch.empty_like(xc)
            dx = dx_bf16
        else:
            dx_f32 = torch.empty(xc.shape, device=xc.device, dtype=torch.float32)
            dx = dx_f32
        dg = grad_buffer(weight) if wants_grad(weight) else None
        db = grad_buffer(bias) if wants_grad(bias) else None
        C().ln_bwd(dy16, xc, mean, rstd, weight.detach() if weight is not None else None, None,
                   dx_f32, dx_bf16, dg, db, None)
        if dg is not None:
            grad_ready(weight)
        if db is not None:
            grad_ready(bias)
        return dx, None, None, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               eps: float = 1e-5, out_bf16: bool = False) -> torch.Tensor:
    """LayerNorm over the last dimension.

    On CUDA, ``out_bf16=True`` writes the normalised output in bf16 (the operand
    format of the tcgen05 GEMMs) while statistics stay in f32.
    """
    if not use_kernels(x) or x.shape[-1] % 4 != 0 or x.shape[-1] > 2048 or x.dtype not in (
            torch.float32, torch.bfloat16):
        if x.is_cuda:
            raise RuntimeError(
                f"flodl_b200 layer_norm kernel supports f32/bf16 with C%4==0 and C<=2048 "
                f"(got {x.dtype}, C={x.shape[-1]})")
        return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)
    return _LayerNormFn.apply(x, weight, bias, float(eps), bool(out_bf16))


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        xc = x.contiguous()
        rows = xc.numel() // xc.shape[-1]
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        y = torch.empty_like(xc)
        C().rms_fwd(xc, weight.detach() if weight is not None else None, y, rstd, eps)
        ctx.save_for_backward(xc, weight, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, weight, rstd = ctx.saved_tensors
        dyc = dy.contiguous().to(xc.dtype)
        dx = torch.empty_like(xc)
        dw = grad_buffer(weight) if wants_grad(weight) else None
        C().rms_bwd(dyc, xc, weight.detach() if weight is not None else None, rstd, dx, dw)
        if dw is not None:
            grad_ready(weight)
        return dx, None, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-5) -> torch.Tensor:
    """RMSNorm over the last dimension, ``x / sqrt(mean(x^2) + eps) * weight``
    (flodl/src/nn/rmsnorm.rs:54-62). On CUDA one kernel forward and one
    backward (which also accumulates ``weight.grad``); f32 and bf16 inputs keep
    their dtype, statistics are f32."""
    if not use_kernels(x) or x.dtype not in (torch.float32, torch.bfloat16) or x.numel() == 0 or (
            x.shape[-1] > 8192 and wants_grad(weight)):
        xf = x.float() if x.dtype in (torch.float16, torch.bfloat16) else x  # at least f32
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
        y = y * weight if weight is not None else y
        return y.to(x.dtype) if x.dtype in (torch.float16, torch.bfloat16) else y
    return _RMSNormFn.apply(x, weight, float(eps))


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps):
        xc = x.contiguous()
        n = xc.shape[0] * groups
        mean = torch.empty(n, device=x.device, dtype=torch.float32)
        rstd = torch.empty(n, device=x.device, dtype=torch.float32)
        y = torch.empty_like(xc)
        C().gn_fwd(xc, weight.detach() if weight is not None else None,
                   bias.detach() if bias is not None else None, y, mean, rstd, groups, eps)
        ctx.groups = groups
        ctx.save_for_backward(xc, weight, bias, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, weight, bias, mean, rstd = ctx.saved_tensors
        dx = torch.empty_like(xc)
        dg = grad_buffer(weight) if wants_grad(weight) else None
        db = grad_buffer(bias) if wants_grad(bias) else None
        C().gn_bwd(dy.contiguous().to(xc.dtype), xc, weight.detach() if weight is not None else None,
                   mean, rstd, dx, dg, db, ctx.groups)
        if dg is not None:
            grad_ready(weight)
        if db is not None:
            grad_ready(bias)
        return dx, None, None, None, None


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """GroupNorm over ``x [N, C, *]`` (flodl/src/nn/groupnorm.rs:62-70): one
    kernel forward, one backward that also accumulates the affine gradients,
    on CUDA for f32 and bf16; elsewhere PyTorch's."""
    if (not use_kernels(x) or x.dtype not in (torch.float32, torch.bfloat16) or x.dim() < 2
            or x.shape[1] % groups):
        return F.group_norm(x, groups, weight, bias, eps)
    return _GroupNormFn.apply(x, int(groups), weight, bias, float(eps))


def check_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, offset):
    """Raises ValueError for arguments that :func:`qk_norm_rope` does not take."""
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"qk_norm_rope takes [B, S, heads, D] queries and keys (got {tuple(q.shape)}"
                         f" and {tuple(k.shape)})")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"queries {tuple(q.shape)} and keys {tuple(k.shape)} differ in batch, "
                         "positions or head size")
    if q.dtype != k.dtype or q.device != k.device or not q.is_floating_point():
        raise ValueError("queries and keys must be floating-point tensors of one dtype and device")
    if q.shape[3] == 0:
        raise ValueError("the head size must be positive")
    D = q.shape[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.device != q.device):
            raise ValueError(f"{name} must be [{D}] on {q.device} (got {tuple(w.shape)} on {w.device})")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is None:
        if use_kernels(q) and any(t is not None and t.dtype != torch.float32
                                  for t in (q_weight, k_weight)):
            raise ValueError("on CUDA the weights must be f32")
        if positions is not None:
            raise ValueError("positions need the cos and sin tables")
        return
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise ValueError(f"cos and sin must be [positions, R / 2] with R <= {D} (got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)})")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError("the tables must be on the inputs' device")
    if use_kernels(q) and any(t is not None and t.dtype != torch.float32
                              for t in (q_weight, k_weight, cos, sin)):
        raise ValueError("on CUDA the weights and tables must be f32")
    if positions is not None:
        if offset != 0:
            raise ValueError("give positions or an offset, not both")
        if positions.dtype != torch.int64 or positions.device != q.device or \
                tuple(positions.shape) != tuple(q.shape[:2]):
            raise ValueError(f"positions must be int64 {list(q.shape[:2])} on {q.device}")
    elif offset < 0 or offset + q.shape[1] > cos.shape[0]:
        raise ValueError(f"positions {offset} to {offset + q.shape[1] - 1} are outside the tables' "
                         f"{cos.shape[0]} rows")


def rotary_rows(cos, sin, positions):
    """The tables' rows of ``positions``. One outside the tables raises on the CPU;
    on CUDA, where the check would wait for the device, its row is NaN."""
    rows = cos.shape[0]
    if not positions.is_cuda:
        if positions.numel() and (int(positions.min()) < 0 or int(positions.max()) >= rows):
            raise IndexError(f"a position is outside the tables' {rows} rows")
        return cos[positions], sin[positions]
    if rows == 0:
        return tuple(t.new_full((*positions.shape, t.shape[1]), float("nan")) for t in (cos, sin))
    bad = ((positions < 0) | (positions >= rows))[..., None]
    at = positions.clamp(0, rows - 1)
    return tuple(t[at].masked_fill(bad, float("nan")) for t in (cos, sin))


def _qk_norm_rope_composed(x, w, cos, sin, eps):
    at_least = torch.float64 if x.dtype == torch.float64 else torch.float32
    y = x.to(at_least)
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps)
    y = y * w if w is not None else y
    if cos is not None:
        R = 2 * cos.shape[-1]
        c, s = cos.to(at_least).unsqueeze(-2), sin.to(at_least).unsqueeze(-2)
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        y = torch.cat((torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), y[..., R:]), -1)
    return y.to(x.dtype)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, offset: int = 0,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """RMSNorm over each query and key head, then the rotary embedding.

    ``q [B, S, H, D]`` and ``k [B, S, Hk, D]`` (H and Hk may differ; views of a
    packed projection are read in place) are normed over D as
    :func:`rms_norm` does, scaled by the f32 ``[D]`` weights, and the pairs
    ``(2i, 2i + 1)`` of their first ``R = 2 * cos.shape[1]`` values are turned
    by the angles of the tables' rows (``nn.RotaryEmbedding``'s ``cos`` and
    ``sin``): row ``offset + s``, or ``positions[b, s]`` (int64) for sequences
    that start at positions of their own. Without tables only the norm runs.
    Returns new contiguous tensors in the inputs' dtype; the arithmetic between
    is f32 and rounded once.

    CUDA f32, bf16 and f16 inputs with 2 <= D <= 256 run one kernel forward and one
    backward (plus a reduction of the weight gradients); other inputs, those with
    forward-mode tangents and tables that want gradients run the composed form. A
    position outside the tables gives NaN in the rotated values of its heads on
    CUDA (the kernel records code 5 in the error word, too); on the CPU it raises.
    """
    if use_kernels(q):
        y = C().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, offset, eps)
        if y is not None:
            return y
    check_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, offset)
    if cos is not None and cos.shape[1] == 0:
        cos = sin = positions = None
    c = s = None
    if cos is not None and positions is None:
        c, s = cos[offset:offset + q.shape[1]], sin[offset:offset + q.shape[1]]
    elif cos is not None:
        c, s = rotary_rows(cos, sin, positions)
    return (_qk_norm_rope_composed(q, q_weight, c, s, eps),
            _qk_norm_rope_composed(k, k_weight, c, s, eps))
