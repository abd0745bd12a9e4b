"""What is measured of the attention operators with separate queries, keys and
values: attention over a memory of another length, and the per-head norm of
queries and keys with the position rotation.

Each case is one pass of one operator, ``fwd`` (serving) or ``train`` (forward
and backward). The plain forms are elementary torch operations in 32 bits,
rounded once; ``exact`` is the definition in 64 bits, gradients by formula.

Layouts: queries ``[B, Sq, H, D]``, keys and values ``[B, Sk, Hk, D]`` with
query head h reading memory head ``h // (H // Hk)``; a padding mask is bool
``[B, Sk]``, True = hidden, and a query that sees no key gives zeros.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
EPS = 1e-5


# ------------------------------------------------------------------ cases
def _attn(name, mode, dtype, B, H, Hk, D, Sq, Sk, pad=0.0, empty=False, causal=False, gain=1.0):
    return dict(name=name, op="attn", mode=mode, dtype=dtype, B=B, H=H, Hk=Hk, D=D, Sq=Sq, Sk=Sk,
                pad=pad, empty=empty, causal=causal, gain=gain)


def _qk(name, mode, dtype, B, S, H, Hk, D, R, positions=False):
    return dict(name=name, op="qk", mode=mode, dtype=dtype, B=B, S=S, H=H, Hk=Hk, D=D, R=R,
                positions=positions)


def listed():
    return [
        # one decoder token against one short encoded sentence: launch latency
        _attn("attn-step-one", "fwd", "bf16", 1, 8, 8, 64, 1, 100),
        # a serving batch of single tokens over BERT-length memories, right-padded
        _attn("attn-step-batch", "fwd", "bf16", 32, 12, 12, 64, 1, 512, pad=0.5),
        # single tokens over a long memory with shared memory heads
        _attn("attn-step-long", "fwd", "bf16", 4, 16, 4, 128, 1, 32768),
        # a few learned queries reading a long odd memory
        _attn("attn-few-queries", "fwd", "fp16", 2, 8, 8, 64, 37, 4001),
        # evaluation of a decoder batch against padded BERT-base memories
        _attn("attn-eval", "fwd", "bf16", 32, 12, 12, 64, 256, 512, pad=0.5),
        # training step at the language model's widths (8 heads of 64, 256 positions)
        _attn("attn-train-lm", "train", "bf16", 64, 8, 8, 64, 256, 256),
        # odd lengths, head size between the tile widths, one sample without a visible key
        _attn("attn-train-ragged", "train", "fp16", 3, 6, 2, 96, 131, 777, pad=0.9, empty=True,
              gain=3.0),
        # long training sequences, shared memory heads of 128
        _attn("attn-train-long", "train", "bf16", 2, 16, 4, 128, 2048, 8192),
        # queries and keys of one new token per sequence, each at its own position
        _qk("qk-step", "fwd", "bf16", 8, 1, 8, 8, 64, 64, positions=True),
        # training at the language model's widths
        _qk("qk-train-lm", "train", "bf16", 64, 256, 8, 8, 64, 64),
        # prompt of a long sequence, shared heads of 128, half of each head rotated
        _qk("qk-long", "fwd", "bf16", 4, 8192, 16, 4, 128, 64),
        # 32-bit training with odd sizes
        _qk("qk-train-f32", "train", "f32", 3, 1001, 6, 3, 40, 40, positions=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "few", "fwd", "train", "train", "qk", "qk"])
    if kind == "qk":
        D = rng.choice([32, 40, 64, 64, 72, 96, 128, 128, 160])
        H = rng.choice([4, 6, 8, 12, 16])
        Hk = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16) if H % h == 0])
        B, S = _log(rng, 1, 48), _log(rng, 1, 8192)
        while B * S * (H + Hk) * D > 80_000_000:
            S = max(1, S // 2)
        return dict(op="qk", mode=rng.choice(["fwd", "train"]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "f32"]), B=B, S=S, H=H, Hk=Hk, D=D,
                    R=rng.choice([D, D, D // 2 // 2 * 2]), positions=rng.random() < 0.4)
    D = rng.choice([32, 64, 64, 64, 80, 96, 128, 128])
    H = rng.choice([4, 6, 8, 12, 16])
    Hk = H if rng.random() < 0.5 else rng.choice([h for h in (1, 2, 3, 4, 6, 8) if H % h == 0])
    if kind == "step":
        B, Sq, Sk = _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 3]), _log(rng, 1, 40000)
        while B * Sk * Hk * D > 67_000_000:
            Sk = max(1, Sk // 2)
    elif kind == "few":
        B, Sq, Sk = _log(rng, 1, 8), _log(rng, 4, 128), _log(rng, 64, 8192)
    else:
        B, Sq, Sk = _log(rng, 1, 48), _log(rng, 16, 2048), _log(rng, 16, 8192)
        while B * H * Sq * Sk > 400_000_000:
            B, Sk = max(1, B // 2), max(16, int(Sk / 1.5))
    causal = kind in ("fwd", "train") and rng.random() < 0.2
    if causal:
        Sk = Sq
    pad = rng.choice([0.0, 0.0, 0.5, 0.9])
    return dict(op="attn", mode="train" if kind == "train" else "fwd",
                dtype=rng.choice(["bf16", "bf16", "fp16"]), B=B, H=H, Hk=Hk, D=D, Sq=Sq, Sk=Sk,
                pad=pad, empty=pad > 0 and rng.random() < 0.3, causal=causal,
                gain=rng.choice([1.0, 1.0, 3.0]))


def _lengths(case):
    """Visible keys of each sample: right padding grows along the batch."""
    B, Sk = case["B"], case["Sk"]
    n = [max(1, Sk - int(case["pad"] * Sk * b / B)) for b in range(B)]
    if case["empty"]:
        n[-1] = 0
    return n


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dt = DT[case["dtype"]]
    B, H, Hk, D = case["B"], case["H"], case["Hk"], case["D"]
    train = case["mode"] == "train"

    def rnd(*shape, gain=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * gain).to(dt)

    def leaf(t):
        return t.detach().requires_grad_(train)

    if case["op"] == "attn":
        Sq, Sk = case["Sq"], case["Sk"]
        # keys and values are the two halves of one projection of the memory
        kv = rnd(B, Sk, 2, Hk, D)
        st = {"case": case, "q": leaf(rnd(B, Sq, H, D, gain=case["gain"])), "k": leaf(kv[:, :, 0]),
              "v": leaf(kv[:, :, 1]), "pad": None}
        if case["pad"] > 0:
            n = torch.tensor(_lengths(case), device="cuda")
            st["pad"] = torch.arange(Sk, device="cuda")[None, :] >= n[:, None]
        if train:
            st["dout"] = rnd(B, Sq, H, D)
        return st
    S, R = case["S"], case["R"]
    # queries and keys are column ranges of one packed projection
    qkv = rnd(B, S, (H + 2 * Hk) * D)
    rows = S + 500
    inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    st = {"case": case,
          "q": leaf(qkv[..., :H * D].unflatten(-1, (H, D))),
          "k": leaf(qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))),
          "qw": leaf(1 + 0.2 * torch.randn(D, device="cuda", generator=g)),
          "kw": leaf(1 + 0.2 * torch.randn(D, device="cuda", generator=g)),
          "cos": ang.cos().float().contiguous(), "sin": ang.sin().float().contiguous(),
          "positions": None}
    if case["positions"]:
        start = torch.randint(0, 500, (B, 1), device="cuda", generator=g)
        st["positions"] = start + torch.arange(S, device="cuda")[None, :]
    if train:
        st["dq"], st["dk"] = rnd(B, S, H, D), rnd(B, S, Hk, D)
    return st


# ------------------------------------------------------------------ plain forms
def _plain_attn(st, q, k, v):
    case = st["case"]
    G = case["H"] // case["Hk"]
    qf = q.float().transpose(1, 2)
    kf, vf = k.float().transpose(1, 2), v.float().transpose(1, 2)
    if G > 1:
        kf, vf = kf.repeat_interleave(G, 1), vf.repeat_interleave(G, 1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * (1.0 / math.sqrt(case["D"]))
    hide = None
    if case["causal"]:
        i = torch.arange(case["Sq"], device=s.device)
        hide = (i[None, :] > i[:, None])[None, None]
    if st["pad"] is not None:
        p = st["pad"][:, None, None, :]
        hide = p if hide is None else hide | p
    if hide is not None:
        s = s.masked_fill(hide, float("-inf"))
    m = s.amax(-1, keepdim=True).detach()
    e = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, vf) / torch.where(total == 0, torch.ones_like(total), total)
    return o.transpose(1, 2).to(q.dtype)


def _plain_norm_rotate(x, w, cos, sin):
    R = 2 * cos.shape[-1]
    xf = x.float()
    y = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS) * w
    a, b = y[..., 0:R:2], y[..., 1:R:2]
    rot = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((rot, y[..., R:]), -1).to(x.dtype)


def _plain_qk(st, q, k):
    S = st["case"]["S"]
    pos = st["positions"]
    cos, sin = (st["cos"][:S], st["sin"][:S]) if pos is None else (st["cos"][pos], st["sin"][pos])
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return (_plain_norm_rotate(q, st["qw"], cos, sin), _plain_norm_rotate(k, st["kw"], cos, sin))


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    train = case["mode"] == "train"
    if case["op"] == "attn":
        q, k, v = st["q"], st["k"], st["v"]
        with torch.set_grad_enabled(train):
            if own:
                from flodl_b200 import ops
                o = ops.cross_attention(q, k, v, key_padding=st["pad"], causal=case["causal"])
            else:
                o = _plain_attn(st, q, k, v)
        if not train:
            return o
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), st["dout"])
        return o.detach(), dq, dk, dv
    q, k = st["q"], st["k"]
    if not own:
        with torch.set_grad_enabled(train):
            yq, yk = _plain_qk(st, q, k)
        if not train:
            return yq, yk
        g = torch.autograd.grad((yq, yk), (q, k, st["qw"], st["kw"]), (st["dq"], st["dk"]))
        return (yq.detach(), yk.detach()) + tuple(g)
    from flodl_b200 import ops
    # a training loop drops the weights' gradients before each step; the
    # operator accumulates into them, as the framework's other norms do
    st["qw"].grad = st["kw"].grad = None
    with torch.set_grad_enabled(train):
        yq, yk = ops.qk_norm_rope(q, k, st["qw"], st["kw"], st["cos"], st["sin"],
                                  positions=st["positions"], eps=EPS)
    if not train:
        return yq, yk
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (st["dq"], st["dk"]))
    return yq.detach(), yk.detach(), dq, dk, st["qw"].grad, st["kw"].grad


# ------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    train = case["mode"] == "train"
    H, Hk, D, B = case["H"], case["Hk"], case["D"], case["B"]
    if case["op"] == "attn":
        n = sum(_lengths(case))  # keys that any query sees
        q, kv = B * case["Sq"] * H * D * e, 2 * n * Hk * D * e
        pairs = H * case["Sq"] * n
        if case["causal"]:
            pairs = H * sum(min(i + 1, L) for L in _lengths(case) for i in range(case["Sq"]))
        pad = B * case["Sk"] if case["pad"] > 0 else 0
        fwd_b, fwd_f = 2 * q + kv + pad, 4.0 * pairs * D
        if not train:
            return {"bytes": fwd_b, "flops": fwd_f}
        # the backward recomputes the scores: five products to the forward's two
        return {"bytes": fwd_b + 2 * q + 2 * B * case["Sk"] * Hk * D * e, "flops": 3.5 * fwd_f}
    T = B * case["S"]
    x = T * (H + Hk) * D * e
    tables = 2 * 4 * (case["S"] + (500 if case["positions"] else 0)) * (case["R"] // 2)
    tables += 8 * T if case["positions"] else 0
    b = 2 * x + tables + 8 * D
    f = 8.0 * T * (H + Hk) * D
    if train:
        b, f = b + 2 * x + 8 * D, f + 16.0 * T * (H + Hk) * D
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    train = case["mode"] == "train"
    if case["op"] == "attn":
        return _exact_attn(case, st, train)
    return _exact_qk(case, st, train)


def _exact_attn(case, st, train):
    B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
    if B * H * Sq * Sk * D * (14 if train else 4) > 6e12:
        return None
    G, c = H // Hk, D ** -0.5
    f64 = dict(dtype=torch.float64, device="cuda")
    out = torch.zeros(B, Sq, H, D, **f64)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(B, Sk, Hk, D, **f64), torch.zeros(B, Sk, Hk, D, **f64)
    with torch.no_grad():
        for b in range(B):
            seen = (~st["pad"][b]).nonzero()[:, 0] if st["pad"] is not None else torch.arange(Sk, device="cuda")
            if seen.numel() == 0:
                continue
            for h in range(H):
                K, V = st["k"][b, seen, h // G].double(), st["v"][b, seen, h // G].double()
                for lo in range(0, Sq, 1024):
                    r = slice(lo, min(lo + 1024, Sq))
                    Q = st["q"][b, r, h].double()
                    z = c * (Q @ K.T)
                    if case["causal"]:
                        rows = torch.arange(lo, r.stop, device="cuda")[:, None]
                        z[seen[None, :] > rows] = float("-inf")
                    P = torch.softmax(z, -1) if not case["causal"] else torch.nan_to_num(torch.softmax(z, -1))
                    O = P @ V
                    out[b, r, h] = O
                    if train:
                        dO = st["dout"][b, r, h].double()
                        dS = P * (dO @ V.T - (dO * O).sum(-1, keepdim=True))
                        dq[b, r, h] = c * (dS @ K)
                        dk[b, seen, h // G] += c * (dS.T @ Q)
                        dv[b, seen, h // G] += P.T @ dO
    return (out, dq, dk, dv) if train else out


def _exact_qk(case, st, train):
    S, R = case["S"], case["R"]
    pos = st["positions"]
    if pos is None:
        pos = torch.arange(S, device="cuda")[None, :].expand(case["B"], S)
    # the rotation as complex multiplication by the tables' (cos + i sin)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, :, None]

    def rotate(y, t):
        z = torch.view_as_complex(y[..., :R].unflatten(-1, (R // 2, 2)).contiguous()) * t
        return torch.cat((torch.view_as_real(z).flatten(-2), y[..., R:]), -1)

    ys, dxs, dws = [], [], []
    with torch.no_grad():
        for x, w, n in ((st["q"], st["qw"], "dq"), (st["k"], st["kw"], "dk")):
            x, w = x.double(), w.double()
            r = (x.square().sum(-1, keepdim=True) / case["D"] + EPS).pow(-0.5)
            ys.append(rotate(x * r * w, turn))
            if train:
                g = rotate(st[n].double(), turn.conj())
                dws.append((g * x * r).sum((0, 1, 2)))
                dxs.append(r * w * g - x * r ** 3 * (g * w * x).sum(-1, keepdim=True) / case["D"])
    return tuple(ys + dxs + dws)
