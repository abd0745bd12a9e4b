"""MultiheadAttention over a memory, and with normed and rotated heads: the
layer against its own composition from plain operations, its gradients
(differences in 64 bits on the CPU; on CUDA against the same layer in f32), the
serving form, and a decoder block of both.

CUDA tolerances. Projections, attention and the output projection round to bf16
(half a step t = 2^-8): four roundings on the way to the output, of values whose
sizes are those of the output's row up to the softmax mean, and about twice as
many on the way back. Norm-wise an output is within 4 t of the f32 layer's and a
gradient within 12 t, each rounding taken at its largest.
"""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from flodl_b200 import nn, ops
from flodl_b200.graph import FlowBuilder
from flodl_b200.nn import MultiheadAttention, RotaryEmbedding

T = 2.0 ** -8


def plain(m, x, memory=None, pad=None, positions=None):
    """The layer's formula in the parameters' precision."""
    B, S, C = x.shape
    H = m.num_heads
    mem = x if memory is None else memory
    W, b = m.qkv.weight, m.qkv.bias
    heads = lambda t: t.view(B, t.shape[1], H, C // H).transpose(1, 2)
    q = heads(F.linear(x, W[:C], b[:C]))
    k, v = (heads(F.linear(mem, W[i * C:(i + 1) * C], b[i * C:(i + 1) * C])) for i in (1, 2))
    if m.q_norm is not None:
        norm = lambda t, w: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + m.q_norm.eps) * w
        q, k = norm(q, m.q_norm.weight), norm(k, m.k_norm.weight)
    if m.rotary is not None and memory is None:
        pos = positions if positions is not None else torch.arange(S, device=x.device).expand(B, S)
        c, s = m.rotary.cos[pos][:, None].to(x.dtype), m.rotary.sin[pos][:, None].to(x.dtype)
        R = 2 * c.shape[-1]

        def turn(t):
            a, d = t[..., 0:R:2], t[..., 1:R:2]
            return torch.cat((torch.stack((a * c - d * s, a * s + d * c), -1).flatten(-2), t[..., R:]), -1)
        q, k = turn(q), turn(k)
    z = q @ k.transpose(-1, -2) / math.sqrt(C // H)
    if pad is not None:
        z = z.masked_fill(pad[:, None, None, :], float("-inf"))
    if m.causal and mem.shape[1] == S:
        z = z.masked_fill(torch.ones(S, S, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
    o = torch.nan_to_num(torch.softmax(z, -1)) @ v
    return m.out_proj.weight.new_zeros(()) + F.linear(o.transpose(1, 2).reshape(B, S, C), m.out_proj.weight,
                                                      m.out_proj.bias)


def layer(kind, C=32, H=4, causal=False, device=None):
    torch.manual_seed(0)
    rope = RotaryEmbedding(C // H // (2 if kind == "half" else 1), 64, device=device) if kind in (
        "rotary", "both", "half") else None
    m = MultiheadAttention(C, H, causal=causal, device=device, qk_norm=kind in ("norm", "both", "half"),
                           rotary=rope)
    if m.q_norm is not None:
        with torch.no_grad():
            m.q_norm.weight.uniform_(0.5, 1.5)
            m.k_norm.weight.uniform_(0.5, 1.5)
    return m


KINDS = ["plain", "norm", "rotary", "both", "half"]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_cpu_self_attention(kind, causal):
    m = layer(kind, causal=causal)
    x = torch.randn(2, 7, 32)
    pos = torch.randint(0, 64, (2, 7)) if m.rotary is not None else None
    torch.testing.assert_close(m(x), plain(m, x), rtol=1e-5, atol=1e-5)
    if pos is not None:
        torch.testing.assert_close(m(x, positions=pos), plain(m, x, positions=pos), rtol=1e-5, atol=1e-5)
    if not causal:
        pad = torch.tensor([[False] * 5 + [True] * 2, [False] * 7])
        torch.testing.assert_close(m(x, key_padding_mask=pad), plain(m, x, pad=pad), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("kind", KINDS)
def test_cpu_causal_with_padding(kind):
    """Both masks at once: right padding, left padding (rows that see no key), all hidden."""
    m = layer(kind, causal=True)
    x = torch.randn(3, 7, 32)
    pad = torch.tensor([[False] * 5 + [True] * 2, [True] * 3 + [False] * 4, [True] * 7])
    y = m(x, key_padding_mask=pad)
    torch.testing.assert_close(y, plain(m, x, pad=pad), rtol=1e-5, atol=1e-5)
    later = x.clone()
    later[:, 4:] += 1.0  # what comes after a query has no effect on it
    torch.testing.assert_close(m(later, key_padding_mask=pad)[:, :4], y[:, :4], rtol=0, atol=0)


@pytest.mark.parametrize("kind", ["plain", "norm"])
def test_cpu_cross_attention_and_serving_form(kind):
    m = layer(kind)
    x, mem = torch.randn(2, 3, 32), torch.randn(2, 9, 32)
    pad = torch.tensor([[False] * 9, [True] * 9])
    want = plain(m, x, mem, pad)
    torch.testing.assert_close(m(x, mem, key_padding_mask=pad), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(m(x, {"memory": mem}), plain(m, x, mem), rtol=1e-5, atol=1e-5)
    kv = m.project_memory(mem)
    steps = [m.attend_memory(x[:, i:i + 1], kv, pad) for i in range(3)]
    torch.testing.assert_close(torch.cat(steps, 1), want, rtol=1e-5, atol=1e-5)
    assert not kv.requires_grad and not steps[0].requires_grad


def norms_once(device, monkeypatch):
    """A step over a projected memory norms the new queries only."""
    m = layer("norm", device=device)
    x, mem = torch.randn(2, 1, 32, device=device), torch.randn(2, 90, 32, device=device)
    with torch.no_grad():
        want = m(x, mem)
    sizes, rms_norm = [], ops.rms_norm
    monkeypatch.setattr(ops, "rms_norm", lambda t, *a: (sizes.append(t.numel()), rms_norm(t, *a))[1])
    kv = m.project_memory(mem)
    assert sizes == [mem.numel()]
    y = m.attend_memory(x, kv)
    assert sizes[1:] == [x.numel()]
    # the same values in the same kernels; only the library's small products may differ
    torch.testing.assert_close(y, want, rtol=0, atol=4 * T * float(want.abs().max()) if x.is_cuda else 1e-5)


def test_cpu_serving_norms_the_memory_once(monkeypatch):
    norms_once("cpu", monkeypatch)


@pytest.mark.gpu
def test_gpu_serving_norms_the_memory_once(monkeypatch):
    norms_once("cuda", monkeypatch)


def empty_sequences(device, dtype):
    """A memory without positions gives the output bias and no gradient but its own;
    a batch without samples gives an empty output."""
    for kind in KINDS:
        m = layer(kind, 128, 2, device=device)
        x = torch.randn(2, 3, 128, device=device).to(dtype).requires_grad_()
        mem = torch.randn(2, 0, 128, device=device).to(dtype)
        y = m(x, mem)
        bias = m.out_proj.bias.detach()
        t = T if x.is_cuda else 0.0  # the projection rounds
        assert ((y.detach().float() - bias).abs() <= t * bias.abs()).all()
        y.float().sum().backward()
        assert (x.grad == 0).all() and (m.qkv.weight.grad == 0).all() and (m.qkv.bias.grad == 0).all()
        serve = m.attend_memory(x.detach()[:, :1], m.project_memory(mem))
        assert torch.equal(serve, y.detach()[:, :1])
        with torch.no_grad():
            none = torch.randn(0, 3, 128, device=device).to(dtype)
            assert m(none).shape == (0, 3, 128) and m(none, none).shape == (0, 3, 128)


def test_cpu_empty_sequences():
    empty_sequences("cpu", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_empty_sequences(dtype):
    empty_sequences("cuda", dtype)


def shared_masks(device):
    """One mask for all samples, and one flag for all keys of a sample."""
    x, mem = torch.randn(2, 3, 32, device=device), torch.randn(2, 9, 32, device=device)
    for kind in KINDS:
        m = layer(kind, device=device)
        for y, keys in ((None, 3), (mem, 9)):
            one = torch.zeros(1, keys, dtype=torch.bool, device=device)
            one[0, 2] = True
            flags = torch.tensor([[False], [True]], device=device)
            for mask in (one, flags):
                full = mask.expand(2, keys).contiguous()
                assert torch.equal(m(x, y, key_padding_mask=mask), m(x, y, key_padding_mask=full))
                if y is not None:
                    kv = m.project_memory(y)
                    assert torch.equal(m.attend_memory(x[:, :1], kv, mask), m.attend_memory(x[:, :1], kv, full))
        with pytest.raises(ValueError):
            m(x, mem, key_padding_mask=torch.zeros(2, 4, dtype=torch.bool, device=device))


def test_cpu_masks_shared_by_the_batch():
    shared_masks("cpu")


@pytest.mark.gpu
def test_gpu_masks_shared_by_the_batch():
    shared_masks("cuda")


@pytest.mark.parametrize("kind", ["plain", "both"])
def test_cpu_gradients_by_differences(kind):
    m = layer(kind, C=8, H=2).double()
    x, mem = (torch.randn(1, n, 8, dtype=torch.float64, requires_grad=True) for n in (3, 4))
    assert torch.autograd.gradcheck(lambda a: m(a), (x,))
    assert torch.autograd.gradcheck(lambda a, b: m(a, b), (x, mem))
    m(x, mem).sum().backward()
    for p in m.qkv.weight, m.qkv.bias:
        g, i = p.grad.clone(), 5
        with torch.no_grad():
            flat = p.view(-1)
            d = []
            for step in (1e-6, -2e-6):
                flat[i] += step
                d.append(m(x, mem).sum().item())
            flat[i] += 1e-6
        assert abs((d[0] - d[1]) / 2e-6 - g.view(-1)[i].item()) < 1e-6


def test_refusals():
    with pytest.raises(ValueError):
        MultiheadAttention(32, 4, rotary=RotaryEmbedding(16, 8))
    m = layer("plain")
    with pytest.raises(ValueError):
        m(torch.randn(1, 3, 32), positions=torch.zeros(1, 3, dtype=torch.long))
    m = layer("both")
    with pytest.raises(ValueError):
        m(torch.randn(1, 3, 32), torch.randn(1, 3, 32), positions=torch.zeros(1, 3, dtype=torch.long))
    with pytest.raises(ValueError):
        m(torch.randn(1, 65, 32))  # beyond the tables
    qkv = torch.randn(6, 3 * 8)
    with pytest.raises(ValueError):
        ops.attention_qk_norm(qkv, 2, 4, 1)
    with pytest.raises(ValueError):
        ops.cross_attention_packed(torch.randn(1, 2, 1, 8), torch.randn(1, 2, 1, 8))


def projection_refusals(device, elsewhere):
    x, mem = torch.randn(2, 3, 16, device=device), torch.randn(2, 5, 16, device=device)
    W, b = torch.randn(24, 16, device=device), torch.randn(24, device=device)
    q, kv = ops.cross_projection(x, mem, W, b)
    assert q.shape == (2, 3, 8) and kv.shape == (2, 5, 16)
    away = (lambda t: torch.empty(t.shape, device=elsewhere))
    for args in ((x[..., :8], mem, W, b), (x, mem[..., :8], W, b), (x, mem, W[:23], b[:23]), (x, mem, W, b[:16]),
                 (x, mem, W[0], None), (x, away(mem), W, b), (x, mem, away(W), b), (x, mem, W, away(b))):
        with pytest.raises(ValueError):
            ops.cross_projection(*args)
    for args in ((x[..., :8], W, b, 0, 8), (x, W, b[:8], 0, 8), (x, W, b, 8, 25), (x, W, b, -1, 8), (x, W, b, 9, 8),
                 (x, away(W), b, 0, 8), (x, W, away(b), 0, 8)):
        with pytest.raises(ValueError):
            ops.project_rows(*args)


def test_cpu_projection_refusals():
    projection_refusals("cpu", "meta")


@pytest.mark.gpu
def test_gpu_projection_refusals():
    """Host tensors among CUDA ones are refused on the host, masks and biases too."""
    projection_refusals("cuda", "cpu")
    x, W, b = torch.randn(2, 16, device="cuda"), torch.randn(8, 16, device="cuda"), torch.randn(8)
    from flodl_b200._ext import cuda_ext
    C = cuda_ext()
    with pytest.raises(RuntimeError):
        C.cast_f32_bf16(b, torch.empty(8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        C.gemm(x.bfloat16(), W.bfloat16(), torch.empty(2, 8, device="cuda"), 2, 8, 16, False, False, bias=b)
    for heads in (1, 2):  # head sizes 64 and 32
        qkv = torch.randn(6, 3 * 64, device="cuda").bfloat16()
        with pytest.raises((RuntimeError, ValueError)):
            ops.attention_packed(qkv, 2, 3, heads, False, torch.zeros(2, 3, dtype=torch.bool))


def computed_parameters(device):
    """Biases and tables that are computed, or learned, get their gradients: against
    the same on the CPU in 64 bits."""
    g = torch.Generator().manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().float()
    x, mem, W, b = rnd(2, 3, 16), rnd(2, 5, 16), rnd(24, 16), rnd(24)
    qkv, cos, sin = rnd(6, 3 * 32), rnd(8, 8), rnd(8, 8)

    def grads(dev, wide):
        to = lambda t: (t.double() if wide else t.clone()).to(dev).requires_grad_()
        a, c, d = to(b), to(cos), to(sin)
        q, kv = ops.cross_projection(to(x), to(mem), to(W), 2 * a)
        heads = to(qkv).view(2, 3, 3, 2, 16)
        y = ops.qk_norm_rope(heads[:, :, 0], heads[:, :, 1], None, None, c, d)
        (q.sum() + kv.sum() + y[0].sum() + 2 * y[1].sum()).backward()
        first = a.grad, c.grad, d.grad
        c.grad = d.grad = None
        z = to(qkv) if dev == "cpu" else qkv.bfloat16().to(dev).requires_grad_()
        ops.attention_qk_norm(z, 2, 3, 2, None, None, c, d).square().sum().backward()
        return first + (c.grad, d.grad)

    for i, (got, want) in enumerate(zip(grads(device, False), grads("cpu", True))):
        # sums of exact ones, of f32 values, and through attention of 16-bit ones (normed
        # heads, P, output and their gradients: six roundings)
        close(got.cpu(), want, 6 * T if i > 2 and device != "cpu" else 64 * 2.0 ** -24, f"gradient {i}")


def test_cpu_computed_parameters():
    computed_parameters("cpu")


@pytest.mark.gpu
def test_gpu_computed_parameters():
    computed_parameters("cuda")


def block(device=None, C=128, H=2):
    """A decoder block: self-attention with normed, rotated heads, then
    cross-attention to a memory, both with residuals."""
    torch.manual_seed(1)
    self_attn = MultiheadAttention(C, H, causal=True, device=device, qk_norm=True,
                                   rotary=RotaryEmbedding(C // H, 512, device=device))
    cross = MultiheadAttention(C, H, device=device)
    norm1, norm2 = nn.LayerNorm(C, device=device), nn.LayerNorm(C, device=device)
    mods = torch.nn.ModuleList([self_attn, cross, norm1, norm2])

    def run(x, mem, pad, plainly=False):
        if plainly:
            x = x + plain(self_attn, F.layer_norm(x, (C,), norm1.weight, norm1.bias, norm1.eps))
            return x + plain(cross, F.layer_norm(x, (C,), norm2.weight, norm2.bias, norm2.eps), mem, pad)
        x = x + self_attn(norm1(x))
        return x + cross(norm2(x), mem, key_padding_mask=pad)
    return mods, run


def test_cpu_decoder_block():
    mods, run = block(C=32)
    x, mem = torch.randn(2, 6, 32), torch.randn(2, 11, 32)
    pad = torch.arange(11)[None, :] >= torch.tensor([11, 4])[:, None]
    torch.testing.assert_close(run(x, mem, pad), run(x, mem, pad, True), rtol=1e-5, atol=1e-5)


def test_flow_builder_using_a_memory():
    g = (FlowBuilder.from_(nn.Linear(16, 32)).tag("memory").through(nn.Linear(32, 32))
         .through(MultiheadAttention(32, 4)).using(["memory"]).build())
    x = torch.randn(2, 5, 16, requires_grad=True)
    y = g(x)
    y.sum().backward()
    assert y.shape == (2, 5, 32) and torch.isfinite(x.grad).all()


# ------------------------------------------------------------------ GPU
def close(a, b, bound, what):
    err = ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-12)).item()
    assert err <= bound, f"{what}: {err:.4f} of its norm, more than {bound:.4f}"


def compare(m, run, plain_run, inputs):
    """Outputs and all gradients of the layer against its f32 formula."""
    leaves = [t.clone().requires_grad_() for t in inputs]
    y = run(*leaves)
    g = torch.randn_like(y)
    for p in m.parameters():
        p.grad = None
    y.backward(g)
    got = [y] + [t.grad for t in leaves] + [p.grad for p in m.parameters()]
    ref = [t.clone().requires_grad_() for t in inputs]
    z = plain_run(*ref)
    params = list(m.parameters())
    want = [z] + list(torch.autograd.grad(z, ref + params, g.float(), allow_unused=True))
    names = ["out"] + [f"input {i}" for i in range(len(inputs))] + [n for n, _ in m.named_parameters()]
    for n, a, b in zip(names, got, want):
        if b is not None:
            close(a, b, 4 * T if n == "out" else 12 * T, n)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["norm", "rotary", "both", "half"])
@pytest.mark.parametrize("C,H", [(256, 4), (192, 2), (160, 4)])
def test_gpu_self_attention(kind, causal, C, H):
    m = layer(kind, C, H, causal, "cuda")
    m.rotary = RotaryEmbedding(2 * m.rotary.cos.shape[1], 400, device="cuda") if m.rotary else None
    x = torch.randn(3, 150, C, device="cuda")
    compare(m, lambda a: m(a), lambda a: plain(m, a), [x])
    pad = torch.arange(150, device="cuda")[None, :] >= torch.tensor([150, 70, 3], device="cuda")[:, None]
    compare(m, lambda a: m(a, key_padding_mask=pad), lambda a: plain(m, a, pad=pad), [x])
    if m.rotary is not None:
        pos = torch.randint(0, 400, (3, 150), device="cuda")
        compare(m, lambda a: m(a, positions=pos), lambda a: plain(m, a, positions=pos), [x])


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("C,H", [(256, 4), (192, 2), (160, 4), (256, 2), (60, 3), (320, 2)])
def test_gpu_plain_self_attention(causal, C, H):
    """Head sizes 64, 96, 40, 128, and those that no kernel takes (20, 160)."""
    m = layer("plain", C, H, causal, "cuda")
    x = torch.randn(3, 150, C, device="cuda")
    compare(m, lambda a: m(a), lambda a: plain(m, a), [x])
    at = torch.arange(150, device="cuda")[None, :]
    pad = at >= torch.tensor([150, 70, 3], device="cuda")[:, None]
    compare(m, lambda a: m(a, key_padding_mask=pad), lambda a: plain(m, a, pad=pad), [x])
    pad = at < torch.tensor([0, 70, 150], device="cuda")[:, None]  # rows that see no key
    compare(m, lambda a: m(a, key_padding_mask=pad), lambda a: plain(m, a, pad=pad), [x])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "norm"])
@pytest.mark.parametrize("C,H,S,Sm", [(256, 4, 40, 170), (192, 2, 130, 90), (160, 4, 1, 300), (512, 8, 300, 300)])
def test_gpu_cross_attention(kind, C, H, S, Sm):
    m = layer(kind, C, H, device="cuda")
    x, mem = torch.randn(2, S, C, device="cuda"), torch.randn(2, Sm, C, device="cuda")
    pad = torch.arange(Sm, device="cuda")[None, :] >= torch.tensor([Sm, Sm // 3], device="cuda")[:, None]
    compare(m, lambda a, b: m(a, b, key_padding_mask=pad), lambda a, b: plain(m, a, b, pad), [x, mem])
    m.causal = True
    compare(m, lambda a, b: m(a, b), lambda a, b: plain(m, a, b), [x, mem])
    m.causal = False
    with torch.no_grad():
        kv = m.project_memory(mem)
        y = m.attend_memory(x[:, :1], kv, pad)
        close(y, plain(m, x[:, :1], mem, pad), 4 * T, "attend_memory")


@pytest.mark.gpu
def test_gpu_layer_of_unaligned_width():
    """Head and projection sizes the kernels do not take (composed forms)."""
    m = layer("plain", 60, 3, device="cuda")
    x, mem = torch.randn(2, 9, 60, device="cuda"), torch.randn(2, 14, 60, device="cuda")
    compare(m, lambda a, b: m(a, b), lambda a, b: plain(m, a, b), [x, mem])
    m = layer("both", 60, 3, device="cuda")
    compare(m, lambda a: m(a), lambda a: plain(m, a), [x])


@pytest.mark.gpu
def test_gpu_weight_listeners_fire_once():
    from flodl_b200.ops._common import add_grad_ready_listener
    m = layer("both", 128, 2, device="cuda")
    x, mem = torch.randn(2, 20, 128, device="cuda"), torch.randn(2, 30, 128, device="cuda")
    for run in (lambda: m(x), lambda: m(x, mem)):
        fired = []
        for p in m.parameters():
            p.grad, p._flodl_grad_listeners = None, []
            add_grad_ready_listener(p, lambda q: fired.append(id(q)))
        run().float().sum().backward()
        assert len(fired) == len(set(fired)) == len(list(m.parameters()))
        assert all(p.grad is not None for p in m.parameters())


@pytest.mark.gpu
def test_gpu_decoder_block_trains_captured():
    """The block's gradients against f32, then the same step captured into a
    graph and replayed: bit for bit the eager one."""
    mods, run = block("cuda")
    x, mem = torch.randn(2, 200, 128, device="cuda"), torch.randn(2, 77, 128, device="cuda")
    pad = torch.arange(77, device="cuda")[None, :] >= torch.tensor([77, 20], device="cuda")[:, None]
    leaves = [x.clone().requires_grad_(), mem.clone().requires_grad_()]
    # two blocks deep in bf16: twice a layer's roundings
    y = run(*leaves, pad)
    g = torch.randn_like(y)
    y.backward(g)
    ref = [x.clone().requires_grad_(), mem.clone().requires_grad_()]
    params = list(mods.parameters())
    z = run(*ref, pad, True)
    want = torch.autograd.grad(z, ref + params, g.float())
    got = [t.grad for t in leaves] + [p.grad for p in params]
    close(y, z, 8 * T, "out")
    names = ["x", "mem"] + [n for n, _ in mods.named_parameters()]
    for n, a, b in zip(names, got, want):
        close(a, b, 24 * T, n)
    del y, z
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        def step():
            for p in params:
                p.grad.zero_()
            out = run(x, mem, pad)
            out.backward(g)
            return out.detach()
        eager = step().clone()
        eager_grads = [p.grad.clone() for p in params]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = step()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    for p, e, n in zip(params, eager_grads, names[2:]):
        # the projections' weight gradients are split-K sums in any order
        torch.testing.assert_close(p.grad, e, rtol=1e-3, atol=1e-3 * float(e.abs().max()), msg=n)


def test_rotary_positions_are_checked():
    rope = RotaryEmbedding(8, 16)
    x = torch.randn(2, 3, 4, 8)
    at = torch.tensor([[0, 15, 3, 3], [1, 2, 3, 4]])
    y = rope.rotate(x, at)
    for b in range(2):
        for s in range(4):
            one = x.new_zeros(1, 3, 16, 8)
            one[:, :, at[b, s]] = x[b, :, s]
            assert torch.allclose(rope.rotate(one)[0, :, at[b, s]], y[b, :, s], atol=1e-6)
    for bad in (at + 1, at - 1):
        with pytest.raises(IndexError):
            rope.rotate(x, bad)
    for bad in (at.int(), at[:1], at[:, :3]):
        with pytest.raises(ValueError):
            rope.rotate(x, bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotary_rounds_once(dtype):
    """Off from the tables' rotation by half a step of the type, and for the two
    products and their sum in f32 by 2 u of their magnitudes."""
    rope = RotaryEmbedding(32, 4096)
    x = torch.randn(2, 3, 700, 40).to(dtype)
    at = torch.randint(0, 4096, (2, 700))
    for pos in (None, at):
        rows = pos if pos is not None else torch.arange(700).expand(2, 700)
        c, s = rope.cos.double()[rows][:, None], rope.sin.double()[rows][:, None]
        a, d = x.double()[..., 0:32:2], x.double()[..., 1:32:2]
        want = torch.cat((torch.stack((a * c - d * s, a * s + d * c), -1).flatten(-2), x.double()[..., 32:]), -1)
        mag = torch.cat((torch.stack(((a * c).abs() + (d * s).abs(), (a * s).abs() + (d * c).abs()),
                                     -1).flatten(-2), 0 * x.double()[..., 32:]), -1)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
        bound = torch.finfo(dtype).eps / 2 * (want.abs() + 2 * 2.0 ** -24 * mag) + 2 * 2.0 ** -24 * mag + tiny
        assert ((rope.rotate(x, pos).double() - want).abs() <= bound).all()
    with pytest.raises(ValueError):
        RotaryEmbedding(32, 699).rotate(x)


@pytest.mark.gpu
def test_gpu_rotary_position_outside_the_tables_is_nan():
    rope = RotaryEmbedding(8, 16, device="cuda")
    x = torch.randn(2, 3, 4, 8, device="cuda")
    at = torch.tensor([[0, 15, 16, 3], [1, -1, 1 << 40, 4]], device="cuda")
    y = rope.rotate(x, at)
    assert torch.isnan(y).all(1).all(-1).tolist() == [[False, False, True, False],
                                                     [False, True, True, False]]
    assert not torch.isnan(y[0, :, :2]).any()


# ------------------------------------------------------------------ forward mode
def tangents(device, dtype):
    """Forward-mode tangents of the operators against the same in 64 bits on the CPU:
    norm-wise off by no more than half a step of the type for every rounding (one at
    the end; in attention_qk_norm also of the normed queries and keys and of their
    tangents), and by f32 sums of up to 64 terms."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)
    q, k, v, kv, qkv = rnd(2, 5, 4, 16), rnd(2, 9, 2, 16), rnd(2, 9, 2, 16), rnd(2, 9, 2, 2, 16), rnd(10, 96)
    x, W, w = rnd(3, 32), rnd(96, 32).bfloat16().float(), torch.rand(16, generator=g) + 0.5
    rope = RotaryEmbedding(16, 8)
    calls = [  # dual inputs, the others, the operator, its roundings
        ((q, k, v), (), lambda a, b, c: ops.cross_attention(a, b, c), 1),
        ((v,), (q, k), lambda c, a, b: ops.cross_attention(a, b, c), 1),
        ((kv,), (q,), lambda b, a: ops.cross_attention_packed(a, b), 1),
        ((q, k[:, :5]), (w, rope.cos, rope.sin), lambda a, b, w, c, s: ops.qk_norm_rope(a, b, w, w, c, s)[1], 1),
        ((w,), (q, k[:, :5]), lambda w, a, b: ops.qk_norm_rope(a, b, w, w)[0], 1),
        ((qkv,), (w, rope.cos, rope.sin), lambda a, w, c, s: ops.attention_qk_norm(a, 2, 5, 2, w, w, c, s), 5),
        ((x,), (W,), lambda a, W: ops.project_rows(a, W, None, 32, 96), 1),
    ]
    for duals, others, f, roundings in calls:
        steps = [rnd(*t.shape) for t in duals]

        def run(dev, wide, leaves):
            cast = lambda t: (t.double() if wide else t).to(dev)
            with forward_ad.dual_level():
                made = [forward_ad.make_dual(cast(t).detach().requires_grad_(leaves), cast(d.to(t.dtype)))
                        for t, d in zip(duals, steps)]
                y = f(*made, *(cast(t) for t in others))
                t = forward_ad.unpack_dual(y).tangent
                return None if t is None else t.detach()

        want = run("cpu", True, False)
        for leaves in (False, True):
            got = run(device, False, leaves)
            assert got is not None, "the tangent is lost"
            close(got.cpu(), want, roundings * torch.finfo(got.dtype).eps / 2 + 64 * 2.0 ** -24, "tangent")


def test_cpu_tangents():
    tangents("cpu", torch.float32)


@pytest.mark.gpu
def test_gpu_tangents():
    tangents("cuda", torch.bfloat16)
    with pytest.raises(Exception):  # the fused projections have no forward mode, and say so
        from torch.autograd import forward_ad
        m = layer("plain", device="cuda")
        with forward_ad.dual_level():
            x = torch.randn(1, 3, 32, device="cuda")
            m(forward_ad.make_dual(x, x), x)
