"""Cases of the operators that put the recurrences into a language model: linear attention with a decay for each head
(a prompt, a training step, a single token) and the layer norm of its read-out.

    S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,   o[t] = scale * q[t]^T S[t]          g: logarithm of the decay, <= 0

``run`` computes them in elementary operations, or, with ``own``, through this package's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a short prompt of a small model: what counts is the latency of the call
        dict(name="prompt short", op="prompt", dtype="bf16", form="lti", B=1, T=77, H=4, Dk=64, Dv=64, state=False,
             ragged=False, norm=False),
        # a batch of long prompts continued from a state, the read-out normalised per head
        dict(name="prompt batch", op="prompt", dtype="bf16", form="lti", B=4, T=8192, H=16, Dk=128, Dv=128, state=True,
             ragged=False, norm=True),
        # a padded batch of prompts of different lengths, gated decays, head sizes off the powers of two
        dict(name="prompt ragged", op="prompt", dtype="fp16", form="lpv", B=3, T=1999, H=6, Dk=80, Dv=48, state=True,
             ragged=True, norm=False),
        # a training step of a model with fixed decays
        dict(name="train fixed", op="train", dtype="bf16", form="lti", B=2, T=4096, H=16, Dk=128, Dv=128, state=False,
             ragged=False, norm=False),
        # a training step on one long document, few heads, learned gates (their gradient included)
        dict(name="train gated long", op="train", dtype="bf16", form="lpv", B=1, T=32768, H=4, Dk=128, Dv=128,
             state=False, ragged=False, norm=False),
        # a small float32 model with odd sizes, learned gates and a learned initial state
        dict(name="train gated odd", op="train", dtype="fp32", form="lpv", B=2, T=509, H=3, Dk=33, Dv=65, state=True,
             ragged=True, norm=False),
        # one sequence answering token by token
        dict(name="token single", op="token", dtype="bf16", form="lti", B=1, T=1, H=16, Dk=128, Dv=128, state=True,
             ragged=False, norm=False),
        # a serving batch answering token by token, gated
        dict(name="token batch", op="token", dtype="bf16", form="lpv", B=256, T=1, H=16, Dk=128, Dv=128, state=True,
             ragged=False, norm=False),
        # a few sequences of an odd-sized float32 model
        dict(name="token odd", op="token", dtype="fp32", form="lpv", B=7, T=1, H=5, Dk=33, Dv=65, state=True,
             ragged=False, norm=False),
        # the read-out of a training batch: 16 heads of 128 channels, forward and backward
        dict(name="norm heads", op="norm", dtype="bf16", rows=8192, C=2048, groups=16, affine=True),
        # whole rows of an odd width in float32
        dict(name="norm rows odd", op="norm", dtype="fp32", rows=1000, C=777, groups=1, affine=True),
        # the rows of a few tokens
        dict(name="norm few", op="norm", dtype="bf16", rows=4, C=1024, groups=1, affine=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "token", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        groups = rng.choice([1, 1, 4, 16])
        width = _spread(rng, 24, 4096 // groups)
        rows = min(_spread(rng, 1, 16384), (1 << 24) // (groups * width))
        return dict(op=op, dtype=dtype, rows=max(rows, 1), C=groups * width, groups=groups, affine=rng.random() < 0.8)
    form = rng.choice(["lti", "lpv"])
    Dk, Dv = (rng.choice([64, 128, 128, 96, 80, rng.randint(16, 128)]) for _ in range(2))
    H = rng.randint(1, 16)
    if op == "token":
        B, T = min(_spread(rng, 1, 256), (1 << 26) // (H * Dk * Dv)), 1
    else:
        B = rng.randint(1, 4)
        T = min(_spread(rng, 1, 16384), (1 << (17 if op == "train" else 18)) // (B * H))
    state = op == "token" or rng.random() < 0.5
    return dict(op=op, dtype=dtype, form=form, B=max(B, 1), T=T, H=H, Dk=Dk, Dv=Dv, state=state,
                ragged=op != "token" and rng.random() < 0.3, norm=op == "prompt" and rng.random() < 0.3)


def prepare(case, seed):
    dt, dev = _TYPES[case["dtype"]], "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)   # noqa: E731
    s = dict(case)
    if case["op"] == "norm":
        C, width = case["C"], case["C"] // case["groups"]
        x = randn(case["rows"], case["groups"], width) * (0.5 + torch.rand(case["rows"], case["groups"], 1, generator=gen,
                                                                           device=dev)) + 0.2 * randn(case["rows"], 1, 1)
        s["x"] = x.reshape(case["rows"], C).to(dt).requires_grad_()
        s["weight"] = (1 + 0.1 * randn(C)).to(dt).requires_grad_() if case["affine"] else None
        s["bias"] = (0.1 * randn(C)).to(dt).requires_grad_() if case["affine"] else None
        s["gy"] = randn(case["rows"], C).to(dt)
        return s
    B, T, H, Dk, Dv = (case[n] for n in ("B", "T", "H", "Dk", "Dv"))
    train, token = case["op"] == "train", case["op"] == "token"
    shape = (B, H) if token else (B, T, H)
    s["q"], s["k"] = randn(*shape, Dk).to(dt), randn(*shape, Dk).to(dt)
    s["v"] = randn(*shape, Dv).to(dt)
    if case["form"] == "lti":     # decays 1 - 2^-4 ... 1 - 2^-9 over the heads, a little apart from seed to seed
        e = torch.linspace(4.0, 9.0, H, device=dev) + 0.1 * randn(H)
        s["g"] = torch.log1p(-torch.exp2(-e))
    else:                          # gates: the logarithm of a sigmoid, most of them near one
        s["g"] = torch.nn.functional.logsigmoid(randn(*shape) + torch.linspace(2.0, 6.0, H, device=dev))
    s["scale"] = Dk ** -0.5
    s["zi"] = randn(B, H, Dk, Dv) if case["state"] else None
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device=dev)
        s["lengths"][0] = T
    s["weight"] = (1 + 0.1 * randn(H * Dv)).to(dt) if case["norm"] else None
    s["bias"] = (0.1 * randn(H * Dv)).to(dt) if case["norm"] else None
    if train:
        for n in ("q", "k", "v", "g", "zi"):
            if s[n] is not None:
                s[n].requires_grad_()
        s["go"] = randn(*shape, Dv).to(dt)
        s["gzf"] = randn(B, H, Dk, Dv) if case["state"] else None
    return s


# ------------------------------------------------------------------------------------------------- plain forms
_CHUNK = 64


def _differences(c):
    """exp(c_i - c_j) for i >= j, else 0, along the last axis of the running sums c (float64)."""
    d = c.unsqueeze(-1) - c.unsqueeze(-2)
    n = c.shape[-1]
    low = torch.ones(n, n, dtype=torch.bool, device=c.device).tril()
    return torch.exp(torch.where(low, d, torch.full_like(d, -math.inf))).float()


def _plain_attention(q, k, v, g, zi, scale, lengths):
    """In chunks of 64 tokens: products within a chunk, the chunks' sums joined by a product over the chunks."""
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    q, k, v, g = q.float(), k.float(), v.float(), g.double().expand(B, T, H)
    if lengths is not None:
        here = (torch.arange(T, device=q.device) < lengths[:, None])[..., None]
        g = torch.where(here, g, torch.zeros_like(g))
        q, k, v = (torch.where(here[..., None], x, torch.zeros_like(x)) for x in (q, k, v))
    N = -(-T // _CHUNK)
    pad = N * _CHUNK - T
    cut = lambda x: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, pad)).unflatten(1, (N, _CHUNK))  # noqa: E731
    q, k, v = (cut(x).permute(0, 3, 1, 2, 4) for x in (q, k, v))       # (B, H, N, chunk, D)
    g = cut(g).permute(0, 3, 1, 2)                                     # (B, H, N, chunk)
    c = g.cumsum(-1)
    whole = c[..., -1].cumsum(-1)                                      # up to the end of each chunk
    o = ((q @ k.transpose(-1, -2)) * _differences(c)) @ v
    sums = (k * torch.exp(c[..., -1:] - c).float().unsqueeze(-1)).transpose(-1, -2) @ v
    init = torch.zeros_like(sums[:, :, :1]) if zi is None else zi.float().unsqueeze(2)
    sums = torch.cat([init, sums], 2).flatten(-2)
    whole = torch.nn.functional.pad(whole, (1, 0))
    states = (_differences(whole) @ sums).unflatten(-1, (Dk, Dv))      # before each chunk, and after the last
    o = o + (q @ states[:, :, :-1]) * torch.exp(c).float().unsqueeze(-1)
    o = (o * scale).permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :T]
    return o, states[:, :, -1]


def _plain_norm(x, weight, bias, eps, groups):
    y = x.float().unflatten(-1, (groups, -1))
    m = y.mean(-1, keepdim=True)
    r = torch.rsqrt(((y - m) * (y - m)).mean(-1, keepdim=True) + eps)
    y = ((y - m) * r).flatten(-2)
    y = y if weight is None else y * weight.float()
    return y if bias is None else y + bias.float()


def _plain(s):
    if s["op"] == "norm":
        y = _plain_norm(s["x"], s["weight"], s["bias"], 1e-5, s["groups"]).to(s["x"].dtype)
        leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"])]
    dt = s["q"].dtype
    if s["op"] == "token":
        a = torch.exp(s["g"].double()).float()
        a = a.expand(s["B"], s["H"])
        new = s["zi"] * a[..., None, None] + s["k"].float().unsqueeze(-1) * s["v"].float().unsqueeze(-2)
        s["zi"].copy_(new)
        return [((s["q"].float().unsqueeze(-1) * new).sum(-2) * s["scale"]).to(dt), s["zi"]]
    o, zf = _plain_attention(s["q"], s["k"], s["v"], s["g"], s["zi"], s["scale"], s["lengths"])
    if s["op"] == "train":
        o = o.to(dt)
        leaves = [s[n] for n in ("q", "k", "v", "g", "zi") if s[n] is not None]
        outs, grads = ([o, zf], [s["go"], s["gzf"]]) if s["state"] else ([o], [s["go"]])
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, grads)]
    if s["norm"]:
        o = _plain_norm(o.flatten(-2), s["weight"], s["bias"], 1e-5, s["H"]).unflatten(-1, (s["H"], -1))
    return [o.to(dt), zf]


# ------------------------------------------------------------------------------------------------- the package's calls
def _calls(s):
    import philtorch_b200 as ptb

    if s["op"] == "norm":
        y = ptb.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5, groups=s["groups"])
        leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"])]
    side = ptb.lti if s["form"] == "lti" else ptb.lpv
    if s["op"] == "token":
        return [side.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["zi"], scale=s["scale"]), s["zi"]]
    if s["op"] == "train":
        out = side.linear_attention(s["q"], s["k"], s["v"], s["g"], s["zi"], scale=s["scale"], lengths=s["lengths"])
        leaves = [s[n] for n in ("q", "k", "v", "g", "zi") if s[n] is not None]
        outs, grads = (list(out), [s["go"], s["gzf"]]) if s["state"] else ([out], [s["go"]])
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, grads)]
    norm = dict(norm_eps=1e-5, norm_weight=s["weight"], norm_bias=s["bias"]) if s["norm"] else {}
    o, zf = side.linear_attention(s["q"], s["k"], s["v"], s["g"], s["zi"], scale=s["scale"], lengths=s["lengths"],
                                  return_state=True, **norm)
    return [o, zf]


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- bytes and operations
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["C"]
        # x in, y out; x and dy in, dx out; the parameters and their gradients
        return {"bytes": 5 * n * e + (4 * case["C"] * e if case["affine"] else 0), "flops": 20 * n}
    B, T, H, Dk, Dv = (case[n] for n in ("B", "T", "H", "Dk", "Dv"))
    tokens = B * T * H
    gates = 4 * (tokens if case["form"] == "lpv" else H)
    states = 4 * B * H * Dk * Dv
    forward = tokens * (2 * Dk + 2 * Dv) * e + gates
    if case["op"] == "token":
        return {"bytes": forward + 2 * states, "flops": tokens * 5 * Dk * Dv}
    if case["op"] == "prompt":
        return {"bytes": forward + (2 if case["state"] else 1) * states, "flops": tokens * 4 * Dk * Dv}
    backward = tokens * (4 * Dk + 3 * Dv) * e + 2 * gates
    return {"bytes": forward + backward + (5 * states if case["state"] else 0), "flops": tokens * 14 * Dk * Dv}


# ------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Token by token, from the recurrence itself (its adjoint runs from the last token to the first)."""
    s = prepare(case, seed)
    wide = lambda n: None if s[n] is None else s[n].detach().double()   # noqa: E731
    if case["op"] == "norm":
        x, w, gy, G = wide("x"), wide("weight"), wide("gy"), case["groups"]
        rows, C = x.shape
        x = x.reshape(rows, G, -1)
        centred = x - x.mean(2, keepdim=True)
        std = (centred.square().mean(2, keepdim=True) + 1e-5).sqrt()
        unit = centred / std
        y = unit.reshape(rows, C)
        gu = gy if w is None else gy * w
        gu = gu.reshape(rows, G, -1)
        gx = (gu - gu.mean(2, keepdim=True) - unit * (gu * unit).mean(2, keepdim=True)) / std
        out = [y if w is None else y * w + wide("bias"), gx.reshape(rows, C)]
        return out if w is None else out + [(gy * y).sum(0), gy.sum(0)]
    B, T, H, Dk, Dv = (case[n] for n in ("B", "T", "H", "Dk", "Dv"))
    if case["op"] != "token" and T > 40000:
        return None
    q, k, v, g, scale = wide("q"), wide("k"), wide("v"), wide("g"), s["scale"]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=q.device) if s["zi"] is None else wide("zi")
    if case["op"] == "token":
        S = S * g.exp().expand(B, H)[:, :, None, None] + torch.einsum("bhi,bhj->bhij", k, v)
        return [scale * torch.einsum("bhi,bhij->bhj", q, S), S]
    a = g.exp().expand(B, T, H)
    if s["lengths"] is not None:      # behind a sequence's end: no decay, nothing added, nothing read
        on = (torch.arange(T, device=q.device)[None, :] < s["lengths"][:, None]).double()
        a = a * on[..., None] + (1 - on[..., None])
        q, k, v = (x * on[:, :, None, None] for x in (q, k, v))
    else:
        on = torch.ones(B, T, dtype=torch.float64, device=q.device)
    train = case["op"] == "train"
    o = torch.empty(B, T, H, Dv, dtype=torch.float64, device=q.device)
    gq = torch.empty_like(q)
    go = wide("go") * on[:, :, None, None] if train else None
    for t in range(T):
        S.mul_(a[:, t, :, None, None]).addcmul_(k[:, t].unsqueeze(-1), v[:, t].unsqueeze(-2))
        o[:, t] = torch.matmul(q[:, t].unsqueeze(-2), S).squeeze(-2)
        if train:
            gq[:, t] = torch.matmul(S, go[:, t].unsqueeze(-1)).squeeze(-1)
    o *= scale
    if not train:
        if case["norm"]:
            centred = o - o.mean(-1, keepdim=True)
            o = centred / (centred.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            o = o * wide("weight").reshape(H, Dv) + wide("bias").reshape(H, Dv)
        return [o, S]
    gq *= scale
    R = wide("gzf") if case["state"] else torch.zeros_like(S)
    last = (R * S).sum((-1, -2))                                        # <dL/dS_T, S_T>
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    for t in range(T - 1, -1, -1):
        R.addcmul_(q[:, t].unsqueeze(-1) * scale, go[:, t].unsqueeze(-2))
        gk[:, t] = torch.matmul(R, v[:, t].unsqueeze(-1)).squeeze(-1)
        gv[:, t] = torch.matmul(k[:, t].unsqueeze(-2), R).squeeze(-2)
        R.mul_(a[:, t, :, None, None])
    gq, gk, gv = (x * on[:, :, None, None] for x in (gq, gk, gv))
    # <R_t, a_t S_{t-1}> = <R_T, S_T> + sum_{u >= t} (q_u . dq_u - k_u . dk_u)
    gg = ((q * gq).sum(-1) - (k * gk).sum(-1)).flip(1).cumsum(1).flip(1) + last[:, None]
    gg = gg * on[..., None]
    if case["form"] == "lti":
        gg = gg.sum((0, 1))
    return [o, S, gq, gk, gv, gg, R] if case["state"] else [o, gq, gk, gv, gg]
