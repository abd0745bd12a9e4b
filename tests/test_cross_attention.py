"""Attention over a memory of another length: values and gradients against the
formulas in 64 bits, masks, layouts, and refusals.

Tolerances. u = 2^-24 and t are half a step of f32 and of the tensors' type
(`finfo.eps / 2`). Products of 16-bit values are exact in f32; a sum of n of
them is off by at most 2 n u times the sum of magnitudes (the tensor cores may
truncate). With c the scale, a score's exponent is off by
c 2 D u sum|q||k| + 2 u |c s| and its exponential by that and 2^-22, so a
probability by a relative e, the largest of these over the row plus the row
sum's e + 2 Sk u and the stored lse's rounding u |lse|. For the kernels
probabilities and dS are rounded to the tensors' type (t each), and
delta = sum dO * O uses O to t^2 (its rounding's remainder is kept, rounded)
with the error of its probabilities. The bounds below add these parts; the
composed form (f32 throughout, one rounding at the end) lies within them too.
f16 has no normal numbers below 2^-14: a rounding there is off by up to 2^-25
whatever the value (P is kept relative to a row's maximum or, for dV, at 2^7
times its value).
"""
import itertools
import math

import pytest
import torch

from flodl_b200 import ops

U = 2.0 ** -24


def reference(q, k, v, pad, causal, scale, dout=None):
    """out[, dq, dk, dv], each with its bound, in 64 bits."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    c = scale if scale is not None else 1.0 / math.sqrt(D)
    t = torch.finfo(q.dtype).eps / 2
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    Q = q.double().transpose(1, 2)
    K, V = (x.double().transpose(1, 2) for x in (k, v))
    if pad is not None:
        K, V = (x.masked_fill(pad[:, None, :, None], 0.0) for x in (K, V))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    vis = torch.ones(B, 1, Sq, Sk, dtype=torch.bool, device=q.device)
    if causal:
        vis = vis.tril()
    if pad is not None:
        vis = vis & ~pad[:, None, None, :]
    s = c * (Q @ K.transpose(-1, -2))
    mag = c * (Q.abs() @ K.abs().transpose(-1, -2))
    e = ((2 * D * U * mag + 2 * U * s.abs()) * vis).amax(-1, keepdim=True) + 2.0 ** -22
    s = s.masked_fill(~vis, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = m.masked_fill(m == float("-inf"), 0.0)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    lse = (m + l.clamp(min=1e-300).log()).abs().clamp(max=1e4) * (l > 0)
    l = l.masked_fill(l == 0, 1.0)
    P = p / l
    e = 3 * e + 4 * Sk * U + 4 * U * lse + 32 * U
    O = P @ V
    bO = t * O.abs() + (t + e) * (P @ V.abs()) + sub * V.abs().sum(-2, keepdim=True) + sub
    back = lambda x: x.transpose(1, 2)
    fold = lambda x: x.unflatten(1, (Hk, G)).sum(2).transpose(1, 2)
    res = [back(O), back(bO)]
    if dout is None:
        return res
    dO = dout.double().transpose(1, 2)
    dP = dO @ V.transpose(-1, -2)
    delta = (dO * O).sum(-1, keepdim=True)
    err_O = bO - (t - 2 * t * t) * O.abs()  # of O before its rounding, and of the remainder's
    b_dP = 2 * D * U * (dO.abs() @ V.abs().transpose(-1, -2)) + (dO.abs() * err_O).sum(-1, keepdim=True) \
        + 2 * D * U * (dO * O).abs().sum(-1, keepdim=True)
    dS = P * (dP - delta)
    b_dS = (P * b_dP + (t + e) * dS.abs() + sub) * vis
    dQ = c * (dS @ K)
    bQ = t * dQ.abs() + c * (b_dS @ K.abs()) + 4 * Sk * U * c * (dS.abs() @ K.abs()) + sub
    T = lambda x: x.transpose(-1, -2)
    N = 4 * Sq * G * U
    dK, dV = fold(c * (T(dS) @ Q)), fold(T(P) @ dO)
    bK = t * dK.abs() + fold(c * (T(b_dS) @ Q.abs()) + N * c * (T(dS.abs()) @ Q.abs())) + sub
    bV = t * dV.abs() + fold(T((t + e + N) * P + sub * 2.0 ** -7 * vis) @ dO.abs()) + sub
    return res + [back(dQ), back(bQ), dK, bK, dV, bV]


def within(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    err = (got.double() - want).abs()
    over = (err - bound).max().item() if err.numel() else -1.0
    assert over <= 0, f"{what}: off by {err.max().item():.3g}, beyond its bound by {over:.3g}"


def make(B, Sq, H, Hk, Sk, D, dtype, device, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)
    return (rnd(B, Sq, H, D) * gain, rnd(B, Sk, Hk, D), rnd(B, Sk, Hk, D), rnd(B, Sq, H, D))


def mask_of(kind, B, Sk, device, seed=3):
    if kind is None:
        return None
    g = torch.Generator().manual_seed(seed)
    pad = torch.zeros(B, Sk, dtype=torch.bool)
    if kind == "right":
        for b in range(B):
            pad[b, max(1, Sk - (b + 1) * Sk // (B + 1)):] = True
    elif kind == "left":
        for b in range(B):
            pad[b, :b * Sk // (B + 1)] = True
    elif kind == "scattered":
        pad = torch.rand(B, Sk, generator=g) < 0.4
    elif kind == "empty":
        pad[-1] = True
        pad[0, Sk // 2:] = True
    elif kind == "one":
        pad[:] = True
        pad[:, Sk // 2] = False
    return pad.to(device)


def check(device, dtype, B, Sq, H, Hk, Sk, D, mask=None, causal=False, scale=None, gain=1.0, grad=True):
    q, k, v, do = make(B, Sq, H, Hk, Sk, D, dtype, device, gain=gain)
    pad = mask_of(mask, B, Sk, device)
    leaves = [x.clone().requires_grad_(grad) for x in (q, k, v)]
    out = ops.cross_attention(*leaves, key_padding=pad, causal=causal, scale=scale)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    want = reference(q, k, v, pad, causal, scale, do if grad else None)
    within(out.detach(), want[0], want[1], "out")
    if grad:
        out.backward(do)
        for i, (x, n) in enumerate(zip(leaves, ("dq", "dk", "dv"))):
            within(x.grad, want[2 + 2 * i], want[3 + 2 * i], n)
        if pad is not None:
            assert (leaves[1].grad[pad] == 0).all() and (leaves[2].grad[pad] == 0).all()
    return out


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("mask", [None, "right", "left", "scattered", "empty"])
@pytest.mark.parametrize("shape", [(2, 3, 4, 2, 7, 8), (1, 1, 2, 1, 1, 5), (3, 6, 2, 2, 5, 16)])
def test_cpu_values_and_gradients(shape, mask):
    for dtype in (torch.float32, torch.bfloat16):
        check("cpu", dtype, *shape, mask=mask)
    check("cpu", torch.float32, *shape, mask=mask, scale=0.7)


def test_cpu_causal_gradcheck_and_zero_keys():
    check("cpu", torch.float32, 2, 5, 2, 1, 5, 8, mask="left", causal=True)
    q, k, v, _ = make(1, 3, 2, 1, 4, 4, torch.float64, "cpu")
    pad = torch.tensor([[False, True, False, False]])
    f = lambda a, b, c: ops.cross_attention(a, b, c, key_padding=pad)
    assert torch.autograd.gradcheck(f, [x.requires_grad_() for x in (q, k, v)])
    out = ops.cross_attention(torch.randn(2, 3, 2, 4), torch.randn(2, 0, 1, 4), torch.randn(2, 0, 1, 4))
    assert out.shape == (2, 3, 2, 4) and (out == 0).all()
    assert ops.cross_attention(torch.randn(0, 3, 2, 4), torch.randn(0, 5, 1, 4),
                               torch.randn(0, 5, 1, 4)).shape == (0, 3, 2, 4)


def hidden_garbage(device, dtype, *shape):
    q, k, v, do = make(*shape, dtype, device)
    B, Sk = shape[0], shape[4]
    for kind in ("right", "scattered", "empty", "one"):
        pad = mask_of(kind, B, Sk, device)
        res = []
        for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
            a = [q.clone().requires_grad_()] + [x.masked_fill(pad[..., None, None], fill).requires_grad_()
                                                for x in (k, v)]
            o = ops.cross_attention(*a, key_padding=pad)
            o.backward(do)
            res.append([o.detach()] + [x.grad for x in a])
        for other in res[1:]:
            for x, y in zip(res[0], other):
                assert torch.equal(x, y)


def test_cpu_hidden_positions_have_no_effect():
    hidden_garbage("cpu", torch.float32, 3, 4, 2, 1, 9, 8)


def refusals(device):
    q, k, v, _ = make(2, 5, 4, 2, 5, 16, torch.bfloat16, device)
    pad = torch.zeros(2, 5, dtype=torch.bool, device=device)
    good = dict(q=q, k=k, v=v, key_padding=pad)
    ops.cross_attention(**good, causal=True)
    for change in (dict(q=q[0]), dict(k=k[:, :4]), dict(k=k[:1], v=v[:1]), dict(k=k[..., :8], v=v[..., :8]),
                   dict(q=q[:, :, :3]), dict(q=q.float()), dict(q=q.long(), k=k.long(), v=v.long()),
                   dict(key_padding=pad[:, :4]), dict(key_padding=pad.int()), dict(key_padding=pad[:1]),
                   dict(q=q[:, :3], causal=True), dict(scale=0.0), dict(scale=-1.0),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(k=k[:, :, :0], v=v[:, :, :0])):
        with pytest.raises(ValueError):
            ops.cross_attention(**{**good, **change})


def test_cpu_refusals():
    refusals("cpu")


# ------------------------------------------------------------------ GPU
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 128])
def test_gpu_few_rows(D, dtype):
    """The form for few query rows, around its step and split borders."""
    for Sk, (Sq, H, Hk) in itertools.product((1, 15, 16, 17, 32, 33, 100, 1025),
                                             ((1, 2, 2), (1, 16, 1), (3, 10, 2), (16, 1, 1))):
        check("cuda", dtype, 2, Sq, H, Hk, Sk, D, grad=False)
    check("cuda", dtype, 1, 1, 4, 1, 20001, D, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["right", "left", "scattered", "empty", "one"])
def test_gpu_few_rows_masks(mask, dtype):
    for Sk, D in ((1, 64), (40, 64), (40, 128), (700, 64), (700, 128), (6000, 64), (6000, 96)):
        check("cuda", dtype, 3, 2, 4, 2, Sk, D, mask=mask, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gpu_few_rows_with_gradient(D):
    check("cuda", torch.bfloat16, 2, 1, 4, 1, 300, D, mask="right")
    check("cuda", torch.float16, 2, 7, 4, 2, 7, D, causal=True)
    check("cuda", torch.bfloat16, 2, 7, 4, 2, 7, D, causal=True, mask="left")


TILES = [  # B, Sq, H, Hk, Sk, D
    (1, 17, 1, 1, 1, 64), (2, 128, 2, 2, 128, 64), (1, 129, 3, 1, 127, 64), (2, 100, 2, 1, 300, 40),
    (1, 200, 4, 4, 65, 8), (2, 128, 2, 2, 128, 128), (1, 257, 2, 1, 193, 128), (2, 64, 4, 2, 500, 96),
    (1, 300, 2, 2, 64, 72), (1, 20, 8, 2, 2000, 64), (1, 20, 8, 2, 2000, 128), (2, 513, 2, 2, 640, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TILES)
def test_gpu_tiles(shape, dtype):
    check("cuda", dtype, *shape)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 72, 128])
def test_gpu_many_items_of_one_tile(D):
    # several items per CTA in every kernel, each with a single streamed tile
    check("cuda", torch.bfloat16, 40, 17, 8, 8, 130, D)
    check("cuda", torch.bfloat16, 40, 130, 8, 8, 17, D, mask="right")
    check("cuda", torch.bfloat16, 50, 150, 8, 8, 150, D, causal=True)
    check("cuda", torch.bfloat16, 100, 40, 8, 4, 50, D, mask="empty")
    check("cuda", torch.bfloat16, 40, 130, 8, 8, 1100, D, mask="one")


@pytest.mark.gpu
@pytest.mark.parametrize("gains", [  # of queries and keys, values, output gradients
    (1.0, 1.0, 1.0), (1.0, 1.0, 1e-2), (1.0, 1.0, 1e-3), (1.0, 1.0, 1e-4), (1.0, 1e-2, 1e-2),
    (0.01, 300.0, 1e3)])
@pytest.mark.parametrize("shape,mask,causal", [
    ((1, 130, 2, 1, 8192, 64), None, False), ((2, 70, 4, 2, 9000, 128), "scattered", False),
    ((2, 3, 4, 2, 9001, 64), "right", False), ((2, 200, 2, 2, 200, 96), None, True),
    ((3, 40, 2, 1, 60, 64), "empty", False), ((40, 150, 8, 4, 700, 64), "right", False)])
def test_gpu_f16_gradients_keep_their_range(shape, mask, causal, gains):
    """Long rows and small or large output gradients in f16. Two roundings to f16 are
    behind a gradient, of P or dS and of the result. Each is a relative error of the
    same distribution, independent from term to term, so that in the norm of a sum of
    many terms of either sign each counts as the rounding of the exact gradient does:
    sqrt(2) of it together. 2 leaves room for f32's errors and O's rounding in delta."""
    q, k, v, do = make(*shape, torch.float16, "cuda")
    q, k, v, do = q * gains[0], k * gains[0], v * gains[1], do * gains[2]
    pad = mask_of(mask, shape[0], shape[4], "cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    ops.cross_attention(*leaves, key_padding=pad, causal=causal).backward(do)
    want = reference(q, k, v, pad, causal, None, do)
    for x, i, n in zip(leaves, (2, 4, 6), ("dq", "dk", "dv")):
        once = (want[i].half().double() - want[i]).norm().item()
        err = (x.grad.double() - want[i]).norm().item()
        assert err <= 2 * once, f"{n}: {err / want[i].norm():.3g}, rounding once {once / want[i].norm():.3g}"


@pytest.mark.gpu
def test_gpu_f16_gradients_of_unlike_heads_and_rows():
    """Output gradients of very different sizes by sample, head and row, values by head,
    rows without any gradient; a sample whose gradient is infinite stays to itself."""
    shape = (3, 150, 4, 2, 600, 64)
    q, k, v, do = make(*shape, torch.float16, "cuda")
    do[0] *= 1e-4
    do[1, :, 1] *= 1e-3
    do[1, ::3] = 0
    do[1, 1::3, 2:] *= 1e-2
    v[1, :, 1] *= 100
    want = reference(q, k, v, None, False, None, do)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = ops.cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, do, retain_graph=True)
    for g, i, n in zip(grads, (2, 4, 6), ("dq", "dk", "dv")):
        for b in range(3):
            for h in range(g.shape[2]):
                w = want[i][b, :, h]
                once = (w.half().double() - w).norm().item()
                assert (g[b, :, h].double() - w).norm().item() <= 2 * once, (n, b, h)
    assert (grads[0][1, ::3] == 0).all()
    do[2, 5] = float("inf")
    again = torch.autograd.grad(out, leaves, do)
    for a, b in zip(grads, again):
        assert torch.equal(a[:2], b[:2]) and not torch.isfinite(b[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_gpu_gradients_of_one_side(packed):
    # frozen memories, frozen queries: the wanted side's gradient is the same
    q, k, v, do = make(2, 70, 4, 2, 90, 64, torch.bfloat16, "cuda")
    kv = torch.stack((k, v), 2)

    def grads(wants_q, wants_kv):
        a, b = q.clone().requires_grad_(wants_q), kv.clone().requires_grad_(wants_kv)
        out = (ops.cross_attention_packed(a, b) if packed
               else ops.cross_attention(a, b[:, :, 0], b[:, :, 1]))
        out.backward(do)
        return a.grad, b.grad

    both = grads(True, True)
    only_q, none = grads(True, False)
    assert none is None and torch.equal(only_q, both[0])
    none, only_kv = grads(False, True)
    assert none is None and torch.equal(only_kv, both[1])
    x = v.clone().requires_grad_()
    ops.cross_attention(q, k, x).backward(do)
    assert torch.equal(x.grad, both[1][:, :, 1])


SPLIT = [  # long key axes of few heads: 2 to 8 pieces, and more than that
    (1, 128, 1, 1, 512, 128), (1, 128, 1, 1, 2048, 128), (1, 140, 1, 1, 2100, 64),
    (2, 1, 1, 1, 2500, 64), (5, 3, 2, 1, 1300, 128), (1, 40, 2, 1, 9000, 72),
    (1, 100, 1, 1, 16000, 64), (1, 2, 4, 2, 16000, 128),
    (1, 9000, 1, 1, 100, 128), (2, 700, 1, 1, 90, 64),
    (60, 1, 8, 8, 1600, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [None, "scattered", "empty", "one"])
@pytest.mark.parametrize("shape", SPLIT)
def test_gpu_split_keys(shape, mask):
    check("cuda", torch.bfloat16, *shape, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 96])
@pytest.mark.parametrize("rows", [17, 45, 100, 129])
def test_gpu_row_tiles_that_end_inside_a_warp(rows, D):
    # pieces of long axes that a second kernel joins (their rows are stored lane by
    # lane), and hidden keys in tiles of every kernel
    check("cuda", torch.bfloat16, 1, rows, 1, 1, 16000, D, mask="scattered")
    check("cuda", torch.bfloat16, 1, 9000, 1, 1, rows, D, mask="scattered")
    check("cuda", torch.float16, 3, rows, 2, 1, 200, D, mask="scattered")


@pytest.mark.gpu
@pytest.mark.parametrize("Sk", [65536, 65600, 140001, 1_100_000])
def test_gpu_few_rows_masks_of_long_memories(Sk):
    """More mask words than one CTA holds: pieces by that limit, joined by a cluster
    and, above sixteen, by a second kernel."""
    for D, mask in ((64, "scattered"), (8, "right"), (128, "one")):
        check("cuda", torch.bfloat16, 2, 1, 2, 1, Sk, D, mask=mask, grad=False)
    check("cuda", torch.float16, 1, 3, 4, 1, Sk, 8, mask="empty", grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gpu_many_heads_of_one_memory_head(dtype):
    for Sq, H, Hk, Sk in ((1, 17, 1, 300), (1, 40, 1, 1000), (5, 64, 2, 70), (1, 33, 3, 5), (130, 24, 1, 90)):
        check("cuda", dtype, 2, Sq, H, Hk, Sk, 64)
        check("cuda", dtype, 2, Sq, H, Hk, Sk, 96, mask="right")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["right", "left", "scattered", "empty", "one"])
def test_gpu_tiles_masks(mask, dtype):
    for D in (64, 128):
        check("cuda", dtype, 3, 150, 2, 1, 333, D, mask=mask)
        check("cuda", dtype, 3, 33, 4, 2, 1500, D, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("mask", [None, "right", "left", "empty"])
def test_gpu_tiles_causal(mask, D):
    for S in (65, 128, 300):
        check("cuda", torch.bfloat16, 2, S, 4, 2, S, D, mask=mask, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gpu_many_items_per_cta(D):
    """Hundreds of items: every CTA of the persistent kernels walks several."""
    check("cuda", torch.bfloat16, 20, 200, 16, 16, 150, D, mask="right")
    check("cuda", torch.bfloat16, 25, 130, 16, 8, 260, D)
    check("cuda", torch.bfloat16, 20, 256, 12, 12, 256, D, causal=True)


@pytest.mark.gpu
def test_gpu_peaked_scores_and_scale():
    for D in (64, 128):
        check("cuda", torch.bfloat16, 2, 140, 2, 1, 400, D, gain=6.0)
        check("cuda", torch.float16, 2, 140, 2, 1, 400, D, gain=6.0, mask="scattered")
        check("cuda", torch.bfloat16, 2, 140, 2, 1, 400, D, scale=1.0, grad=False)
        check("cuda", torch.bfloat16, 2, 2, 2, 1, 400, D, gain=6.0, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 2, 4, 2, 700, 64), (3, 2, 4, 2, 700, 128), (3, 150, 2, 1, 333, 64),
                                   (3, 150, 2, 1, 333, 128), (3, 20, 2, 2, 1400, 96)])
def test_gpu_hidden_positions_have_no_effect(shape):
    hidden_garbage("cuda", torch.bfloat16, *shape)
    hidden_garbage("cuda", torch.float16, *shape)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 150])
def test_gpu_layouts(Sq):
    """Views give what their contiguous copies give."""
    B, H, Hk, Sk, D = 2, 4, 2, 260, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    kv = rnd(B, Sk, 2, Hk, D)
    flat = rnd(B * Sq * H * D + 8)
    cases = [
        (rnd(B, H, Sq, D).transpose(1, 2), kv[:, :, 0], kv[:, :, 1]),          # head-major, packed halves
        (flat[1:-7].view(B, Sq, H, D), kv[:, :, 0], kv[:, :, 1]),              # 2-byte alignment
        (rnd(B, Sq, H, D + 4)[..., :D], rnd(B, Sk, Hk, D), rnd(B, Sk, Hk, D)),  # 8-byte row stride
        (rnd(B, Sq, H, D), rnd(1, Sk, Hk, D).expand(B, -1, -1, -1), rnd(B, Sk, 1, D).expand(-1, -1, Hk, -1)),
        (rnd(B, Sq, D, H).transpose(2, 3), rnd(Sk, B, Hk, D).transpose(0, 1), kv[:, :, 1]),
    ]
    for q, k, v in cases:
        do = rnd(B, H, Sq, D).transpose(1, 2)
        res = []
        for f in (lambda x: x, lambda x: x.contiguous()):
            leaves = [f(x).detach().requires_grad_() for x in (q, k, v)]
            o = ops.cross_attention(*leaves)
            o.backward(f(do))
            res.append([o.detach()] + [x.grad for x in leaves])
        for x, y in zip(*res):
            assert torch.equal(x, y)
    # a summed output's gradient has no strides at all
    leaves = [x.detach().requires_grad_() for x in cases[0]]
    ops.cross_attention(*leaves).sum().backward()
    other = [x.detach().requires_grad_() for x in cases[0]]
    o = ops.cross_attention(*other)
    o.backward(torch.ones_like(o))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, other))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 40])
def test_gpu_offsets_beyond_32_bits(Sq):
    """The second sample's memory starts past 2^31 elements."""
    H, Sk, D = 2, 300, 64
    far = 2 ** 31 + 64
    buf = torch.empty(far + Sk * H * D, device="cuda", dtype=torch.bfloat16)
    k = buf.as_strided((2, Sk, H, D), (far, H * D, D, 1))
    q, kk, _, _ = make(2, Sq, H, H, Sk, D, torch.bfloat16, "cuda")
    k.copy_(kk)
    a = ops.cross_attention(q, k, k)
    assert torch.equal(a, ops.cross_attention(q, kk, kk))
    del buf, k


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 4, 4, 5000, 64), (2, 150, 4, 2, 333, 64), (1, 40, 2, 2, 3000, 128)])
def test_gpu_repeats_graphs_and_streams(shape):
    """Eager repeats, a captured pass (forward and backward) replayed on new
    inputs, and a side stream give the same bits."""
    q, k, v, do = make(*shape, torch.bfloat16, "cuda")
    pad = mask_of("right", shape[0], shape[4], "cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]

    def once():
        o = ops.cross_attention(*leaves, key_padding=pad)
        return (o,) + torch.autograd.grad(o, leaves, do)

    eager = [x.detach().clone() for x in once()]
    assert all(torch.equal(a, b) for a, b in zip(eager, once()))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = once()
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1, stream=st):
            out1 = once()
        with torch.cuda.graph(g2, stream=st):
            out2 = once()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(eager, side))
    with torch.no_grad():
        for x in leaves:
            x.mul_(0.5)
    g1.replay()
    g2.replay()
    g1.replay()
    fresh = once()
    torch.cuda.synchronize()
    for a, b, c in zip(fresh, out1, out2):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_gpu_f16_passes_at_once():
    """Training passes of several shapes on streams, in threads and as graphs replayed
    side by side give the bits of one after another."""
    import threading
    shapes = [(2, 130, 4, 2, 700, 64), (1, 40, 2, 2, 3000, 128), (3, 3, 4, 1, 500, 96), (8, 200, 8, 8, 200, 64)]
    data = []
    for i, shape in enumerate(shapes):
        q, k, v, do = make(*shape, torch.float16, "cuda", seed=i)
        data.append(([x.requires_grad_() for x in (q, k, v)], do * 10.0 ** (1 - i),
                     mask_of("right", shape[0], shape[4], "cuda")))

    def once(i):
        leaves, do, pad = data[i]
        out = ops.cross_attention(*leaves, key_padding=pad)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    want = [once(i) for i in range(4)]
    torch.cuda.synchronize()
    same = lambda got: all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    streams = [torch.cuda.Stream() for _ in range(4)]
    for turn in range(4):
        got = [None] * 4
        for i in range(4):
            with torch.cuda.stream(streams[(i + turn) % 4]):
                got[i] = once(i)
        torch.cuda.synchronize()
        assert same(got)

    got = [None] * 4

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = once(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert same(got)
    graphs = []
    for i in range(4):
        with torch.cuda.stream(streams[i]):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i], stream=streams[i]):
                got[i] = once(i)
    for _ in range(3):
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert same(got)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-50, 1e-40, 1e-18, 1e-10])
def test_gpu_tiny_scales(scale):
    """Scores vanish: a query's output is the mean of the values (a sum of 70 rounded
    weights and the output's rounding), however far below f32's range the scale is."""
    for Sq in (1, 40):
        q, k, v, do = make(2, Sq, 2, 1, 70, 64, torch.bfloat16, "cuda")
        t = torch.finfo(torch.bfloat16).eps / 2
        want = v.double().mean(1, keepdim=True).expand(2, Sq, 2, 64)
        bound = 2 * t * v.double().abs().mean(1, keepdim=True).expand(2, Sq, 2, 64)
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        a = ops.cross_attention(*leaves, scale=scale)
        b = ops.cross_attention_packed(leaves[0], torch.stack(leaves[1:], 2), scale=scale)
        for y in (a, b):
            within(y.detach(), want, bound, "out")
            grads = torch.autograd.grad(y, leaves, do, retain_graph=True)
            assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.gpu
def test_gpu_refusals_and_other_forms():
    from flodl_b200._ext import cuda_ext
    refusals("cuda")
    q, k, v, _ = make(1, 4, 2, 2, 6, 64, torch.float32, "cuda")
    check("cuda", torch.float32, 2, 5, 2, 1, 9, 24, mask="empty")        # composed, f32
    check("cuda", torch.bfloat16, 2, 5, 2, 1, 9, 20, mask="right")       # D not a multiple of 8
    check("cuda", torch.bfloat16, 1, 5, 2, 1, 9, 160)                    # D above 128
    C = cuda_ext()
    b = lambda x: x.bfloat16()
    with pytest.raises(RuntimeError):
        C.cross_attn_fwd(q, k, v, None, False, 1.0, False)               # f32
    with pytest.raises(RuntimeError):
        C.cross_attn_fwd(b(q), b(k)[..., :32], b(v), None, False, 1.0, False)
    with pytest.raises(RuntimeError):
        C.cross_attn_fwd(b(q).transpose(2, 3), b(k), b(v), None, False, 1.0, False)
    with pytest.raises(RuntimeError):
        C.cross_attn_fwd(b(q), b(k), b(v), None, True, 1.0, False)
    with pytest.raises(RuntimeError):
        C.cross_attn_fwd(b(q), b(k), b(v), None, False, -1.0, False)
    assert cuda_ext().kernel_error() == 0


@pytest.mark.gpu
def test_gpu_differentiable_once_and_partial_gradients():
    q, k, v, do = make(2, 40, 2, 1, 70, 64, torch.bfloat16, "cuda")
    want = None
    for need in itertools.product((False, True), repeat=3):
        if not any(need):
            continue
        leaves = [x.clone().requires_grad_(n) for x, n in zip((q, k, v), need)]
        ops.cross_attention(*leaves).backward(do)
        grads = [x.grad for x in leaves]
        if all(need):
            want = grads
        assert all((g is not None) == n for g, n in zip(grads, need))
    g, = torch.autograd.grad(ops.cross_attention(*leaves), leaves[0], do, create_graph=True)
    assert torch.equal(g.detach(), want[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaves[0])
