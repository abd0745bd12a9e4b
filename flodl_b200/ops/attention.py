"""Scaled dot-product attention on packed QKV.

Reference: ``at::scaled_dot_product_attention`` (flodl-sys/ops_nn.cpp:407-431,
flodl/src/nn/attention.rs:136-230). The CUDA path runs the sm_100a flash
attention kernels (``_C.flash_attn_fwd`` / ``_C.flash_attn_bwd``): S = QK^T and
O += PV on tcgen05 with the accumulators in TMEM, online softmax, causal tile
skipping. Q/K/V are read straight out of the packed ``[T, 3C]`` projection
output and O is written as ``[T, C]`` (token-major), so no transposes run
around the kernel.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F

from ._common import C, use_kernels


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
    mask used by BERT-style encoders.
    """
    if not use_kernels(qkv):
        D = qkv.shape[1] // (3 * H)
        q, k, v = qkv.view(B, S, 3, H, D).permute(2, 0, 3, 1, 4).unbind(0)
        mask = None
        if key_padding is not None:
            mask = ~key_padding[:, None, None, :]
        o = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=causal and mask is None)
        return o.permute(0, 2, 1, 3).reshape(B * S, H * D)
    q16 = qkv if qkv.dtype == torch.bfloat16 else qkv.to(torch.bfloat16)
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
    sums are f32, probabilities are rounded to the inputs' type for the
    products. Gradients are the same from run to run. Other inputs run the
    composed form in f32 or f64.
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
