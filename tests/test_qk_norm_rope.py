"""Per-head query/key RMS norm with the rotary embedding: values and gradients
against the formulas in 64 bits, layouts, and refusals.

Tolerances. With u = 2^-24 (half a step of f32) and t = half a step of the
output type (`finfo.eps / 2`), a rotated value a c - d s of normed values a, d
carries the output rounding t |y| and the f32 errors of the row's root mean
square (a sum of D squares by at most 8 + 5 additions, halved by the root, two
roundings for the root and the reciprocal), two products and the rotation:
below 16 u (|a c| + |d s|). An input gradient r (g w - xh mean(g w xh)) sums
its two parts' magnitudes with at most 32 roundings each. A weight gradient is
a sum over N rows: at most (N + 32) u times the sum of magnitudes, in whatever
order.
"""
import math

import pytest
import torch

from flodl_b200 import nn, ops

U = 2.0 ** -24


def tables(rows, R, device="cpu"):
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().to(device), ang.sin().float().to(device)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turn(y, c, s, back=False):
    """Rotation of the pairs in 64 bits; c, s broadcast over the heads."""
    R = 2 * c.shape[-1]
    a, d = y[..., 0:R:2], y[..., 1:R:2]
    if back:
        s = -s
    return torch.cat((torch.stack((a * c - d * s, a * s + d * c), -1).flatten(-2), y[..., R:]), -1)


def reference(x, w, c, s, eps, dy=None):
    """(y, bound of y[, dx, bound of dx, dw, bound of dw]) in 64 bits."""
    D = x.shape[-1]
    x64, w64 = x.double(), (w.double() if w is not None else torch.ones(D, device=x.device).double())
    c, s = c.double().unsqueeze(-2), s.double().unsqueeze(-2)
    r = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x64 * r
    y = turn(xh * w64, c, s)
    R = 2 * c.shape[-1]
    absturn = lambda v: torch.cat((torch.stack((v[..., 0:R:2] * c.abs() + v[..., 1:R:2] * s.abs(),
                                                v[..., 0:R:2] * s.abs() + v[..., 1:R:2] * c.abs()),
                                               -1).flatten(-2), v[..., R:]), -1)
    t = half_step(x.dtype)
    out = [y, t * y.abs() + 16 * U * absturn((xh * w64).abs()) + 1e-30]
    if dy is not None:
        g, ga = turn(dy.double(), c, s, back=True), absturn(dy.double().abs())
        dx = r * (g * w64 - xh * (g * w64 * xh).mean(-1, keepdim=True))
        mag = r * (ga * w64.abs() + xh.abs() * (ga * w64.abs() * xh.abs()).mean(-1, keepdim=True))
        rows = x64.numel() // D
        out += [dx, t * dx.abs() + 32 * U * mag + 1e-30, (g * xh).sum((0, 1, 2)),
                (rows + 32) * U * (ga * xh.abs()).sum((0, 1, 2)) + 1e-30]
    return out


def within(got, want, bound, tiny=0.0):
    err = (got.double() - want).abs()
    worst = (err - bound).max().item() if err.numel() else -1.0
    assert torch.isfinite(got).all()
    assert worst <= tiny, f"off by {err.max().item():.3g}, beyond its bound by {worst:.3g}"


def inputs(B, S, H, Hk, D, dtype, device, seed=0, packed=True):
    g = torch.Generator().manual_seed(seed)
    if packed:
        qkv = torch.randn(B, S, (H + 2 * Hk) * D, generator=g).to(dtype).to(device)
        q = qkv[..., :H * D].unflatten(-1, (H, D))
        k = qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
    else:
        q = torch.randn(B, S, H, D, generator=g).to(dtype).to(device)
        k = torch.randn(B, S, Hk, D, generator=g).to(dtype).to(device)
    qw = (1 + 0.3 * torch.randn(D, generator=g)).to(device)
    kw = (1 + 0.3 * torch.randn(D, generator=g)).to(device)
    dq = torch.randn(B, S, H, D, generator=g).to(dtype).to(device)
    dk = torch.randn(B, S, Hk, D, generator=g).to(dtype).to(device)
    return q, k, qw, kw, dq, dk


def check(device, dtype, B, S, H, Hk, D, R, positions=False, offset=0, weights=True, packed=True):
    q, k, qw, kw, dq, dk = inputs(B, S, H, Hk, D, dtype, device, packed=packed)
    eps = 1e-5
    cos, sin = tables(S + offset + 40, R, device)
    pos = None
    if positions:
        g = torch.Generator().manual_seed(5)
        pos = torch.randint(0, S + 40, (B, S), generator=g).to(device)
    c, s = (cos[pos], sin[pos]) if positions else (cos[offset:offset + S], sin[offset:offset + S])
    qr, kr = q.detach().requires_grad_(), k.detach().requires_grad_()
    qwr = qw.clone().requires_grad_() if weights else None
    kwr = kw.clone().requires_grad_() if weights else None
    yq, yk = ops.qk_norm_rope(qr, kr, qwr, kwr, cos if R else None, sin if R else None,
                              offset=0 if positions else offset, positions=pos if R else None, eps=eps)
    assert yq.dtype == dtype and yk.dtype == dtype
    torch.autograd.backward((yq, yk), (dq, dk))
    # a subnormal f16 result is off by up to half of its fixed step
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for x, w, y, dy, leaf, wl in ((q, qw, yq, dq, qr, qwr), (k, kw, yk, dk, kr, kwr)):
        want = reference(x, w if weights else None, c, s, eps, dy)
        within(y.detach(), want[0], want[1], tiny)
        within(leaf.grad, want[2], want[3], tiny)
        if weights:
            within(wl.grad, want[4], want[5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 5, 4, 2, 16, 16), (1, 1, 1, 1, 2, 2), (2, 3, 3, 1, 7, 6), (1, 4, 2, 2, 24, 8)])
def test_cpu_values_and_gradients(shape, dtype):
    check("cpu", dtype, *shape)
    check("cpu", dtype, *shape, positions=True)
    check("cpu", dtype, *shape, offset=9, weights=False)


def test_cpu_norm_only_and_gradcheck():
    check("cpu", torch.float32, 2, 3, 2, 1, 8, 0)
    cos, sin = tables(6, 4)
    q, k = torch.randn(1, 3, 2, 6).double().requires_grad_(), torch.randn(1, 3, 1, 6).double().requires_grad_()
    w = torch.randn(6).double().requires_grad_()
    assert torch.autograd.gradcheck(
        lambda a, b, v: ops.qk_norm_rope(a, b, v, v, cos, sin, offset=2), (q, k, w))


def test_agrees_with_rms_norm_then_rotary_module():
    q, k, qw, kw, _, _ = inputs(2, 6, 3, 3, 16, torch.float32, "cpu")
    rope = nn.RotaryEmbedding(16, 32)
    yq, yk = ops.qk_norm_rope(q, k, qw, kw, rope.cos, rope.sin, offset=4)
    for x, w, y in ((q, qw, yq), (k, kw, yk)):
        want = rope(ops.rms_norm(x, w).transpose(1, 2), offset=4).transpose(1, 2)
        torch.testing.assert_close(y, want, rtol=0, atol=32 * U * float(want.abs().max()))


def refusals(device):
    q, k, qw, kw, _, _ = inputs(2, 6, 4, 2, 16, torch.float32, device)
    cos, sin = tables(8, 16, device)
    bad = [
        dict(q=q[0]), dict(k=k[:, :5]), dict(k=k[..., :8]), dict(k=k.to(torch.bfloat16)),
        dict(q_weight=qw[:8]), dict(k_weight=kw[None]), dict(sin=None), dict(cos=cos[:, :4]),
        dict(cos=torch.zeros(8, 9, device=device), sin=torch.zeros(8, 9, device=device)),
        dict(offset=3), dict(offset=-1),
        dict(positions=torch.zeros(2, 5, dtype=torch.int64, device=device)),
        dict(positions=torch.zeros(2, 6, dtype=torch.int32, device=device)),
        dict(positions=torch.zeros(2, 6, dtype=torch.int64, device=device), offset=1),
        dict(cos=None, sin=None, positions=torch.zeros(2, 6, dtype=torch.int64, device=device)),
        dict(q=q.long(), k=k.long()),
    ]
    good = dict(q=q, k=k, q_weight=qw, k_weight=kw, cos=cos, sin=sin)
    ops.qk_norm_rope(**good, offset=2)
    for change in bad:
        with pytest.raises(ValueError):
            ops.qk_norm_rope(**{**good, **change})


def test_cpu_refusals():
    refusals("cpu")
    q, k, *_ = inputs(1, 2, 1, 1, 4, torch.float32, "cpu")
    cos, sin = tables(3, 4)
    for at in (-1, 3):
        with pytest.raises(IndexError):
            ops.qk_norm_rope(q, k, None, None, cos, sin, positions=torch.tensor([[0, at]]))


def test_empty_batch():
    q, k, qw, kw, _, _ = inputs(0, 3, 2, 1, 8, torch.float32, "cpu")
    yq, yk = ops.qk_norm_rope(q, k, qw, kw)
    assert yq.shape == (0, 3, 2, 8) and yk.shape == (0, 3, 1, 8)


# ------------------------------------------------------------------ GPU
SHAPES = [  # B, S, H, Hk, D, R
    (1, 1, 1, 1, 64, 64), (2, 7, 8, 8, 64, 64), (3, 5, 12, 4, 128, 64), (2, 9, 6, 3, 40, 40),
    (2, 33, 5, 1, 96, 90), (1, 6, 3, 2, 36, 36), (2, 3, 4, 4, 33, 32), (1, 17, 16, 2, 256, 256),
    (2, 4, 2, 1, 8, 4), (1, 2, 3, 1, 2, 2), (2, 700, 8, 8, 64, 64), (2, 5, 4, 4, 72, 20),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gpu_values_and_gradients(shape, dtype):
    check("cuda", dtype, *shape)
    check("cuda", dtype, *shape, positions=True, packed=False)


@pytest.mark.gpu
def test_gpu_variants():
    check("cuda", torch.bfloat16, 2, 5, 4, 2, 64, 0)
    check("cuda", torch.bfloat16, 2, 5, 4, 2, 64, 64, offset=31, weights=False)
    check("cuda", torch.float32, 1, 3, 2, 2, 320, 64)  # beyond the kernel: composed


@pytest.mark.gpu
def test_gpu_views_and_alignment():
    """Transposed, offset, broadcast and reversed-order views give what their
    contiguous copies give."""
    g = torch.Generator(device="cuda").manual_seed(1)
    B, S, H, D = 2, 9, 4, 64
    cos, sin = tables(S, D, "cuda")
    w = torch.rand(D, device="cuda", generator=g)
    base = torch.randn(B, H, S, D, device="cuda", generator=g).bfloat16()
    flat = torch.randn(B * S * H * D + 3, device="cuda", generator=g).bfloat16()
    views = [base.transpose(1, 2), flat[3:].view(B, S, H, D), base[:1].transpose(1, 2).expand(B, S, H, D),
             base.transpose(1, 2).transpose(2, 3).contiguous().transpose(2, 3)]
    for v in views:
        a = ops.qk_norm_rope(v, v, w, w, cos, sin)
        b = ops.qk_norm_rope(v.contiguous(), v.contiguous(), w, w, cos, sin)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[0], a[1])


@pytest.mark.gpu
def test_gpu_weight_gradient_routes():
    """A leaf weight accumulates into .grad (twice over two steps, and when one
    weight serves both), a computed one through autograd; results repeat."""
    q, k, qw, kw, dq, dk = inputs(3, 50, 4, 2, 64, torch.bfloat16, "cuda")
    cos, sin = tables(50, 64, "cuda")

    def grads(wq, wk):
        y = ops.qk_norm_rope(q, k, wq, wk, cos, sin)
        torch.autograd.backward(y, (dq, dk))

    a, b = qw.clone().requires_grad_(), kw.clone().requires_grad_()
    grads(a, b)
    one = a.grad.clone(), b.grad.clone()
    grads(a, b)
    assert torch.equal(a.grad, one[0] + one[0]) and torch.equal(b.grad, one[1] + one[1])
    s = qw.clone().requires_grad_()
    grads(s, s)
    d = qw.clone().requires_grad_()
    grads(d * 1.0, d * 1.0)
    torch.testing.assert_close(d.grad, s.grad, rtol=4 * U, atol=0)
    fired = []
    from flodl_b200.ops._common import add_grad_ready_listener
    e = qw.clone().requires_grad_()
    add_grad_ready_listener(e, lambda p: fired.append(p))
    grads(e, e)
    assert len(fired) == 1 and fired[0] is e and torch.equal(e.grad, s.grad)


@pytest.mark.gpu
def test_gpu_refusals_and_bad_positions():
    from flodl_b200._ext import cuda_ext
    refusals("cuda")
    q, k, qw, kw, _, _ = inputs(1, 3, 2, 1, 16, torch.float32, "cuda")
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw.double(), kw)
    cos, sin = tables(4, 8, "cuda")
    cuda_ext().clear_kernel_error()
    for at in (-1, 4, 2 ** 40):
        pos = torch.tensor([[0, at, 3]], device="cuda")
        yq, yk = ops.qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos)
        torch.cuda.synchronize()
        assert cuda_ext().kernel_error() == 5
        cuda_ext().clear_kernel_error()
        assert torch.isnan(yq[0, 1, :, :8]).all() and torch.isfinite(yq[0, 1, :, 8:]).all()
        assert torch.isfinite(yq[0, [0, 2]]).all() and torch.isfinite(yk[0, [0, 2]]).all()


@pytest.mark.gpu
def test_gpu_graph_replay_and_side_stream():
    q, k, qw, kw, dq, dk = inputs(2, 20, 4, 4, 64, torch.bfloat16, "cuda")
    q, k = q.contiguous(), k.contiguous()
    cos, sin = tables(20, 64, "cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        eager = ops.qk_norm_rope(q, k, qw, kw, cos, sin)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = ops.qk_norm_rope(q, k, qw, kw, cos, sin)
        g.replay()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(out, eager))
    q.copy_(dq)
    want = ops.qk_norm_rope(q, k, qw, kw, cos, sin)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_gpu_extreme_rows():
    """All-zero rows (only eps under the root) and rows of large values."""
    x = torch.zeros(1, 2, 2, 64, device="cuda")
    x[0, 1] = 1e18
    y, _ = ops.qk_norm_rope(x, x, None, None)
    assert (y[0, 0] == 0).all()
    torch.testing.assert_close(y[0, 1], torch.ones_like(y[0, 1]), rtol=16 * U, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
def test_gpu_spans_beyond_32_bits(dim):
    """A sample (or a position) more than 2^31 elements from the first."""
    B, S, H, D = (3, 4, 2, 64) if dim == 0 else (1, 3, 2, 64)
    far = 2 ** 30 + 64
    strides = (far, H * D, D, 1) if dim == 0 else (far, far, D, 1)
    buf = torch.empty(2 * far + S * H * D, device="cuda", dtype=torch.bfloat16)
    x = buf.as_strided((B, S, H, D), strides)
    q, _, qw, kw, dq, _ = inputs(B, S, H, H, D, torch.bfloat16, "cuda", packed=False)
    x.copy_(q)
    cos, sin = tables(S + 9, D, "cuda")
    pos = torch.randint(0, S + 9, (B, S), device="cuda")
    for kw_pos in (dict(offset=5), dict(positions=pos)):
        res = []
        for v in (x, q):
            leaf = v.detach().requires_grad_()
            a, b = qw.clone().requires_grad_(), kw.clone().requires_grad_()
            y = ops.qk_norm_rope(leaf, leaf, a, b, cos, sin, **kw_pos)
            g = torch.autograd.grad(y, leaf, (dq, dq))[0]
            res.append((*[t.detach() for t in y], g, a.grad, b.grad))
        for i, (u, w) in enumerate(zip(*res)):
            if i < 3:
                assert torch.equal(u, w)
            else:  # other launches, other order of the rows' sum
                torch.testing.assert_close(u, w, rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
def test_gpu_differentiable_once_and_partial_use():
    q, k, qw, kw, dq, _ = inputs(1, 4, 2, 2, 64, torch.bfloat16, "cuda", packed=False)
    q, k = q.requires_grad_(), k.requires_grad_()
    y = ops.qk_norm_rope(q, k, qw, kw)[0]
    g, = torch.autograd.grad(y, q, dq, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)
    # only one of the two results used: the other has no gradient
    y = ops.qk_norm_rope(q, k, qw, kw)[1]
    a, b = torch.autograd.grad(y, (q, k), dq, allow_unused=True)
    assert (a is None or (a == 0).all()) and torch.isfinite(b).all() and b.abs().max() > 0
