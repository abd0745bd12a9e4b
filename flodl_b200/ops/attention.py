"""Scaled dot-product attention on packed QKV.

Reference: ``at::scaled_dot_product_attention`` (flodl-sys/ops_nn.cpp:407-431,
flodl/src/nn/attention.rs:136-230). The CUDA path runs the sm_100a flash
attention kernels (``_C.flash_attn_fwd`` / ``_C.flash_attn_bwd``): S = QK^T and
O += PV on tcgen05 with the accumulators in TMEM, online softmax, causal tile
skipping. Q/K/V are read straight out of the packed ``[T, 3C]`` projection
output and O is written as ``[T, C]`` (token-major), so no transposes run
around the kernel.

:func:`cross_attention` takes queries, keys and values in tensors of their own
(another sequence's states, shared memory heads, single tokens of serving) and
:func:`attention_qk_norm` norms and rotates the heads of a packed projection
before either form.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ._common import C, has_tangent, use_kernels
from .norm import qk_norm_rope


def attn_fwd_packed(qkv: torch.Tensor, B: int, S: int, H: int, causal: bool,
                    key_padding: Optional[torch.Tensor] = None):
    """qkv [B*S, 3*H*D] bf16 -> (out [B*S, H*D] bf16, lse [B, H, S] f32)."""
    D = qkv.shape[1] // (3 * H)
    out = torch.empty((B * S, H * D), device=qkv.device, dtype=torch.bfloat16)
    lse = torch.empty((B, H, S), device=qkv.device, dtype=torch.float32)
    C().flash_attn_fwd(qkv, out, lse, B, S, H, D, bool(causal), 1.0 / math.sqrt(D), key_padding)
    return out, lse


def attn_bwd_packed(dout: torch.Tensor, qkv: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                    B: int, S: int, H: int, causal: bool,
                    key_padding: Optional[torch.Tensor] = None,
                    bias_grad: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the packed QKV: dqkv [B*S, 3*H*D] bf16. With ``bias_grad``
    (f32 [3*H*D]) the column sums of dqkv - the gradient of the packed
    projection's bias - are accumulated into it in the same pass."""
    D = qkv.shape[1] // (3 * H)
    dqkv = torch.empty_like(qkv)
    C().flash_attn_bwd(dout.contiguous(), qkv, out, lse, dqkv, B, S, H, D, bool(causal),
                       1.0 / math.sqrt(D), key_padding, bias_grad)
    return dqkv


class _PackedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, B, S, H, causal, key_padding):
        out, lse = attn_fwd_packed(qkv, B, S, H, causal, key_padding)
        ctx.save_for_backward(qkv, out, lse, key_padding)
        ctx.dims = (B, S, H, causal)
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, out, lse, key_padding = ctx.saved_tensors
        B, S, H, causal = ctx.dims
        d16 = dout if dout.dtype == torch.bfloat16 else dout.to(torch.bfloat16)
        return attn_bwd_packed(d16, qkv, out, lse, B, S, H, causal, key_padding), None, None, None, None, None


def attention_packed(qkv: torch.Tensor, B: int, S: int, H: int, causal: bool = False,
                     key_padding: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Self-attention over packed ``qkv [B*S, 3C]``; returns ``[B*S, C]``.

    ``key_padding`` (bool ``[B, S]``, True = masked key) implements the padding
    mask used by BERT-style encoders; with ``causal`` both apply. On CUDA the
    flash kernel takes head size 64, :func:`cross_attention` the others and empty
    inputs; the result is bf16.
    """
    if not use_kernels(qkv):
        D = qkv.shape[1] // (3 * H)
        q, k, v = qkv.view(B, S, 3, H, D).permute(2, 0, 3, 1, 4).unbind(0)
        mask = None
        if key_padding is not None:
            mask = ~key_padding[:, None, None, :]
            if causal:
                mask = mask & torch.ones(S, S, dtype=torch.bool, device=qkv.device).tril()
        o = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=causal and mask is None)
        return o.permute(0, 2, 1, 3).reshape(B * S, H * D)
    q16 = qkv if qkv.dtype == torch.bfloat16 else qkv.to(torch.bfloat16)
    if qkv.shape[1] != 3 * H * 64 or q16.numel() == 0:
        q, k, v = q16.reshape(B, S, 3, H, qkv.shape[1] // (3 * H)).unbind(2)
        return cross_attention(q, k, v, key_padding, causal).view(B * S, qkv.shape[1] // 3)
    return _PackedAttnFn.apply(q16.contiguous(), B, S, H, causal, key_padding)


def scaled_dot_product_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                 attn_mask: Optional[torch.Tensor] = None, is_causal: bool = False,
                                 dropout_p: float = 0.0) -> torch.Tensor:
    """Functional SDPA on ``[B, H, S, D]`` tensors (floDl's functional API).

    Self-attention with head size 64 (the flash kernel's) runs the kernel
    through the packed layout when there is no mask or the mask only hides
    keys (boolean, broadcast over heads and queries: ``[B, 1, 1, S]`` with
    True = attend, the padding mask of encoder batches); anything else uses
    the composed (explicit softmax) form, which is also the CPU path.
    """
    B, H, S, D = q.shape
    key_padding = None
    if (attn_mask is not None and attn_mask.dtype == torch.bool and attn_mask.dim() == 4
            and attn_mask.shape[1] == 1 and attn_mask.shape[2] == 1
            and attn_mask.shape[0] in (1, B) and attn_mask.shape[3] == S and not is_causal):
        key_padding = (~attn_mask[:, 0, 0, :]).expand(B, S).contiguous()
    if (q.is_cuda and (attn_mask is None or key_padding is not None) and dropout_p == 0.0
            and k.shape == q.shape and v.shape == q.shape and D == 64):
        qkv = torch.stack([q, k, v], dim=0).permute(1, 3, 0, 2, 4).reshape(B * S, 3 * H * D)
        o = attention_packed(qkv.to(torch.bfloat16), B, S, H, is_causal, key_padding)
        return o.view(B, S, H, D).permute(0, 2, 1, 3).to(q.dtype)
    scale = 1.0 / math.sqrt(D)
    s = torch.matmul(q, k.transpose(-2, -1)) * scale
    if is_causal:
        m = torch.ones(S, k.shape[-2], dtype=torch.bool, device=q.device).tril()
        s = s.masked_fill(~m, float("-inf"))
    if attn_mask is not None:
        if attn_mask.dtype == torch.bool:
            s = s.masked_fill(~attn_mask, float("-inf"))
        else:
            s = s + attn_mask
    p = torch.softmax(s.float(), dim=-1).to(q.dtype)
    if dropout_p > 0:
        p = F.dropout(p, dropout_p)
    return torch.matmul(p, v)


# ----------------------------------------------------------------- separate q, k, v
def _cross_composed(q, k, v, key_padding, causal, scale):
    """The explicit form in the inputs' precision, at least f32."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    work = torch.float64 if q.dtype == torch.float64 else torch.float32
    qh, kh, vh = (t.to(work).transpose(1, 2) for t in (q, k, v))
    if key_padding is not None:  # what a hidden position holds has no effect
        hidden = key_padding[:, None, :, None]
        kh, vh = kh.masked_fill(hidden, 0.0), vh.masked_fill(hidden, 0.0)
    if Hk != H:
        kh, vh = kh.repeat_interleave(H // Hk, 1), vh.repeat_interleave(H // Hk, 1)
    s = torch.matmul(qh, kh.transpose(-1, -2)) * scale
    if key_padding is not None:
        s = s.masked_fill(key_padding[:, None, None, :], float("-inf"))
    if causal:
        i = torch.arange(Sq, device=q.device)
        s = s.masked_fill(i[None, :] > i[:, None], float("-inf"))
    if Sk:
        m = s.detach().amax(-1, keepdim=True)
        s = s - m.masked_fill(m == float("-inf"), 0.0)
    e = torch.exp(s)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, vh) / total.masked_fill(total == 0, 1.0)
    return o.transpose(1, 2).to(q.dtype).contiguous()


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    key_padding: Optional[torch.Tensor] = None, causal: bool = False,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of ``q [B, Sq, H, D]`` over a memory ``k, v [B, Sk, Hk, D]`` of
    another length: ``softmax(scale * q k^T) v``, token-major like
    :func:`attention_packed`, returned contiguous as ``[B, Sq, H, D]``.

    * H is a multiple of Hk; query head h reads memory head ``h // (H // Hk)``.
    * ``key_padding`` (bool ``[B, Sk]``, True = hidden key) hides positions of
      the memory; what they hold, NaN included, has no effect. A query that
      sees no key gives zeros, and no gradient.
    * ``causal`` (equal lengths only) lets query i see keys 0..i.
    * ``scale`` is positive, ``1 / sqrt(D)`` by default.

    CUDA bf16 and f16 inputs with D a multiple of 8 up to 128 run the sm_100a
    kernels: views with 16-byte strides (a packed key/value projection's halves,
    head-major tensors transposed to this layout) are read in place, others are
    copied. Up to 16 query rows per memory head (``Sq * H / Hk``; the single
    tokens of serving) take a form that streams the memory once. Scores and
    sums are f32; probabilities are rounded to the inputs' type for the products,
    and score gradients in the backward (in f16 at a power of two that the data
    gives, so that small ones do not vanish nor large ones overflow; the gradients
    returned have f16's own range). With gradients, outputs are divided by the sum
    of the rounded probabilities and may differ by a rounding from those without.
    Gradients are the same from run to run. Other inputs, scales below 1e-18 or
    beyond 1e18, and inputs with forward-mode tangents run the composed form in f32
    or f64.
    """
    if use_kernels(q):
        out = C().cross_attention(q, k, v, key_padding, causal, scale)
        if out is not None:
            return out
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"cross_attention takes [B, S, heads, D] tensors (got {tuple(q.shape)} and "
                         f"{tuple(k.shape)})")
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    if k.shape != v.shape:
        raise ValueError(f"keys {tuple(k.shape)} and values {tuple(v.shape)} differ")
    if k.shape[0] != B or k.shape[3] != D or D == 0:
        raise ValueError(f"queries {tuple(q.shape)} and keys {tuple(k.shape)} differ in batch or "
                         "head size")
    if H == 0 or Hk == 0 or H % Hk:
        raise ValueError(f"{H} query heads are not a multiple of {Hk} memory heads")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device
            and q.dtype.is_floating_point):
        raise ValueError("queries, keys and values must be floating-point tensors of one dtype and "
                         "device")
    if key_padding is not None and (key_padding.dtype != torch.bool or key_padding.shape != (B, Sk)
                                    or key_padding.device != q.device):
        raise ValueError(f"key_padding must be bool [{B}, {Sk}] on {q.device}")
    if causal and Sq != Sk:
        raise ValueError(f"causal attention needs equal lengths (got {Sq} and {Sk})")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite (got {scale})")
    return _cross_composed(q, k, v, key_padding, causal, scale)


def _fresh(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _CrossPackedFn(torch.autograd.Function):
    """cross_attention on a packed key/value projection: the gradient comes as
    one packed tensor, without copies of its halves."""

    @staticmethod
    def forward(ctx, q, kv, key_padding, causal, scale):
        q, kv = _fresh(q), _fresh(kv)
        out, res, lse, bits = C().cross_attn_fwd(q, kv[:, :, 0], kv[:, :, 1], key_padding, causal, scale,
                                                 True)
        ctx.save_for_backward(q, kv, out, res, lse, key_padding, bits)
        ctx.consts = (causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, kv, out, res, lse, key_padding, bits = ctx.saved_tensors
        dq = torch.empty_like(q) if ctx.needs_input_grad[0] else None
        dkv = torch.empty_like(kv) if ctx.needs_input_grad[1] else None
        C().cross_attn_bwd(_fresh(dout.to(q.dtype)), q, kv[:, :, 0], kv[:, :, 1], out, res, lse,
                           key_padding, bits, *ctx.consts, dq,
                           *((dkv[:, :, 0], dkv[:, :, 1]) if dkv is not None else (None, None)))
        return dq, dkv, None, None, None


def _kernels_take(t: torch.Tensor) -> bool:
    D = t.shape[-1]
    return (use_kernels(t) and t.dtype in (torch.bfloat16, torch.float16) and D % 8 == 0 and D <= 128
            and t.numel() > 0)


def cross_attention_packed(q: torch.Tensor, kv: torch.Tensor,
                           key_padding: Optional[torch.Tensor] = None, causal: bool = False,
                           scale: Optional[float] = None) -> torch.Tensor:
    """:func:`cross_attention` with the memory's keys and values in one packed
    projection ``kv [B, Sk, 2, Hk, D]``; its gradient is packed likewise."""
    if kv.dim() != 5 or kv.shape[2] != 2:
        raise ValueError(f"packed keys and values are [B, Sk, 2, Hk, D] (got {tuple(kv.shape)})")
    if (torch.is_grad_enabled() and (q.requires_grad or kv.requires_grad) and q.dim() == 4
            and _kernels_take(q) and kv.numel() > 0 and kv.dtype == q.dtype and kv.device == q.device
            and kv.shape[0] == q.shape[0] and kv.shape[4] == q.shape[3]
            and q.shape[2] % kv.shape[3] == 0 and not (causal and q.shape[1] != kv.shape[1])
            and not has_tangent(q, kv)):
        pad = key_padding
        ok = pad is None or (pad.dtype == torch.bool and pad.shape == kv.shape[:2]
                             and pad.device == q.device)
        c = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
        if ok and C().CROSS_ATTN_LEAST_SCALE <= c <= 1 / C().CROSS_ATTN_LEAST_SCALE:
            return _CrossPackedFn.apply(q, kv, pad.contiguous() if pad is not None else None,
                                        bool(causal), c)
    return cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_padding, causal, scale)


class _QkNormAttnFn(torch.autograd.Function):
    """Norm and rotation of a packed projection's queries and keys, then
    attention with its values in place; the packed gradient is written once."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, positions, eps, causal, key_padding, scale):
        qkv = _fresh(qkv)
        q, k, v = qkv.unbind(2)
        det = (lambda w: w.detach() if w is not None else None)
        yq, yk = C().qk_norm_rope(q, k, det(q_weight), det(k_weight), cos, sin, positions, 0, eps)
        out, res, lse, bits = C().cross_attn_fwd(yq, yk, v, key_padding, causal, scale, True)
        ctx.save_for_backward(qkv, yq, yk, q_weight, k_weight, cos, sin, positions, out, res, lse,
                              key_padding, bits)
        ctx.consts = (eps, causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (qkv, yq, yk, q_weight, k_weight, cos, sin, positions, out, res, lse, key_padding,
         bits) = ctx.saved_tensors
        eps, causal, scale = ctx.consts
        dqkv = torch.empty_like(qkv)
        q, k, v = qkv.unbind(2)
        dq, dk, dv = dqkv.unbind(2)
        dyq, dyk = torch.empty_like(yq), torch.empty_like(yk)
        C().cross_attn_bwd(_fresh(dout.to(qkv.dtype)), yq, yk, v, out, res, lse, key_padding, bits,
                           causal, scale, dyq, dyk, dv)
        dwq, dwk = C().qk_norm_rope_backward(dyq, dyk, q, k, q_weight, k_weight, cos, sin, positions,
                                             0, eps, dq, dk)
        return dqkv, dwq, dwk, None, None, None, None, None, None, None


def attention_qk_norm(qkv: torch.Tensor, B: int, S: int, H: int, q_weight: Optional[torch.Tensor] = None,
                      k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                      sin: Optional[torch.Tensor] = None, causal: bool = False,
                      key_padding: Optional[torch.Tensor] = None,
                      positions: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """Self-attention over packed ``qkv [B*S, 3C]`` whose queries and keys are
    normed per head and rotated first (:func:`qk_norm_rope`, then
    :func:`cross_attention` over the same positions); returns ``[B*S, C]``. On CUDA
    other types than bf16 and f16 are cast to bf16, as :func:`attention_packed` does."""
    if qkv.dim() != 2 or qkv.shape[0] != B * S or qkv.shape[1] % (3 * H):
        raise ValueError(f"qkv must be [{B * S}, 3 * {H} * D] (got {tuple(qkv.shape)})")
    if use_kernels(qkv) and qkv.dtype not in (torch.bfloat16, torch.float16):
        qkv = qkv.to(torch.bfloat16)
    D = qkv.shape[1] // (3 * H)
    packed = qkv.view(B, S, 3, H, D) if qkv.is_contiguous() else qkv.reshape(B, S, 3, H, D)
    needs = any(t is not None and t.requires_grad for t in (qkv, q_weight, k_weight))
    if (torch.is_grad_enabled() and needs and _kernels_take(packed)
            and not any(t is not None and t.requires_grad for t in (cos, sin))
            and not has_tangent(packed, q_weight, k_weight, cos, sin)):
        # the checks of both operators, on views (nothing is launched for them)
        from .norm import check_qk_norm_rope
        check_qk_norm_rope(packed[:, :, 0], packed[:, :, 1], q_weight, k_weight, cos, sin, positions, 0)
        if key_padding is not None and (key_padding.dtype != torch.bool
                                        or key_padding.shape != (B, S)
                                        or key_padding.device != qkv.device):
            raise ValueError(f"key_padding must be bool [{B}, {S}] on {qkv.device}")
        if cos is not None and cos.shape[1] == 0:
            cos = sin = positions = None
        c = (lambda t: t.contiguous() if t is not None else None)
        out = _QkNormAttnFn.apply(packed, c(q_weight), c(k_weight), c(cos), c(sin), c(positions),
                                  float(eps), bool(causal), c(key_padding), 1.0 / math.sqrt(D))
    else:
        q, k, v = packed.unbind(2)
        q, k = qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=positions, eps=eps)
        out = cross_attention(q, k, v, key_padding, causal)
    return out.reshape(B * S, H * D)
