"""The operators of a long-context attention block and the sizes at which their speed is tracked.

  attn       causal attention over a sliding window with a few first tokens that stay visible: `attention_packed(..., window,
             sinks)` on the packed projection output, or `window_attention(q, k, v, ...)` on separate tensors
  rotary     rotation of all heads by their positions: half or interleaved pairs, the whole head or its first part
  norm       RMS norm of every query and key head with the rotation in the same pass

`direction` "fwd" is the call without gradients (evaluation, scoring), "bwd" the call and its gradients, as in a training step.
Queries, keys, values and incoming gradients are what reaches the operators in a block: the projections of normalised
activations, about unit normal, and gradients of a mean over many tokens.
"""
from __future__ import annotations

import math

import torch

own = False
EPS = 1e-6


def _attn(name, batch, seq, q, kv, dim, window, sinks, direction, packed=True):
    return dict(name=name, op="attn", batch=batch, seq=seq, q_heads=q, kv_heads=kv, dim=dim, window=window, sinks=sinks,
                direction=direction, packed=packed)


def _rows(name, op, batch, seq, q, kv, dim, rotated, interleaved, first, per_batch, direction):
    """`first`: position of the first token; `per_batch`: every sequence of the batch has its own positions."""
    return dict(name=name, op=op, batch=batch, seq=seq, q_heads=q, kv_heads=kv, dim=dim, rotated=rotated,
                interleaved=interleaved, first=first, per_batch=per_batch, direction=direction)


def listed():
    return [
        # one token of each of eight sequences: launch and latency
        _attn("attn_one_token", 8, 1, 16, 8, 64, 1024, 4, "fwd"),
        # the plumbing configuration (8 query / 2 KV heads of 32, 2 x 256 tokens), a short window
        _attn("attn_tiny", 2, 256, 8, 2, 32, 64, 4, "bwd"),
        # text windows of a length nobody chose for the hardware, separate tensors
        _attn("attn_ragged", 3, 1001, 12, 4, 64, 333, 5, "bwd", packed=False),
        # evaluation with heads of 128, no sinks
        _attn("attn_hd128", 2, 4096, 16, 4, 128, 2048, 0, "fwd"),
        # the launch scripts' heads (32 query / 4 KV of dim 32) at their micro-batch
        _attn("attn_shipped_hd32", 8, 4096, 32, 4, 32, 512, 4, "bwd"),
        # the benchmark's heads (16 / 8 of 64) at its micro-batch
        _attn("attn_headline_hd64", 8, 4096, 16, 8, 64, 1024, 4, "bwd"),
        # the same heads on one long sequence
        _attn("attn_long_32k", 1, 32768, 16, 8, 64, 1024, 16, "bwd"),
        # one token of each of sixteen sequences at positions of their own
        _rows("norm_one_token", "norm", 16, 1, 16, 8, 64, 64, False, 30000, True, "fwd"),
        # a ragged micro-batch, interleaved pairs on half of the head
        _rows("norm_ragged", "norm", 3, 1001, 12, 4, 64, 32, True, 0, False, "bwd"),
        # the benchmark's heads at its micro-batch
        _rows("norm_headline", "norm", 8, 4096, 16, 8, 64, 64, False, 0, False, "bwd"),
        # the launch scripts' heads, interleaved
        _rows("rotary_shipped_hd32", "rotary", 8, 4096, 32, 4, 32, 32, True, 0, False, "bwd"),
        # a late piece of a very long text: far positions, a quarter of the head rotated
        _rows("rotary_far", "rotary", 1, 32768, 16, 4, 128, 32, False, 1 << 20, False, "fwd"),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, dim):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([r for r in (1, 2, 3, 4, 8) if kv * r * dim <= 2048]), kv


def _draw_once(rng):
    op = rng.choice(["attn", "attn", "attn", "norm", "rotary"])
    dim = rng.choice([32, 64, 64, 128])
    q, kv = _heads(rng, dim)
    batch = rng.choice([1, 1, 2, 3, 4, 8])
    direction = rng.choice(["fwd", "bwd", "bwd"])
    seq = _log_int(rng, 1, 32768 // batch)
    if rng.random() < 0.4:
        seq = max(1, seq // 128 * 128)
    if op == "attn":
        window = _log_int(rng, 1, 4096)
        if rng.random() < 0.4:
            window = max(64, window // 64 * 64)
        sinks = rng.choice([0, 1, 4, 4, 16, rng.randint(1, 200)])
        # rows that see one key only have no gradient for queries and keys: relative to the packed gradient's size, not to zero
        packed = rng.random() < 0.6 or seq == 1 or window + sinks == 1
        return _attn("", batch, seq, q, kv, dim, window, sinks, direction, packed)
    if op == "rotary":
        dim = rng.choice([32, 64, 96, 128, 256])
    rotated = rng.choice([dim, dim, dim // 2, dim // 4])
    return _rows("", op, batch, seq, q, kv, dim, rotated, rng.random() < 0.5, rng.choice([0, 0, 1000, 1 << 20]),
                 rng.random() < 0.3, direction)


def _scores(c):
    """Elements of one matrix of the plain form's scores."""
    w = max(1, min(c["window"], c["seq"]))
    return c["batch"] * c["q_heads"] * (-(-c["seq"] // w) * w) * (2 * w + c["sinks"])


def draw(rng):
    most = {op: max(work(c)["bytes"] if op != "attn" else work(c)["flops"] for c in listed() if c["op"] == op)
            for op in ("attn", "norm", "rotary")}
    while True:
        c = _draw_once(rng)
        cost = work(c)["flops"] if c["op"] == "attn" else work(c)["bytes"]
        if cost <= most[c["op"]] and (c["op"] != "attn" or _scores(c) <= 1.2 * 2 ** 30):
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------ states
class _State:
    pass


def prepare(case, seed):
    c, s = case, _State()
    s.case = c
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).bfloat16()

    B, T, Hq, Hkv, d = c["batch"], c["seq"], c["q_heads"], c["kv_heads"], c["dim"]
    grads = c["direction"] == "bwd"
    if c["op"] == "attn":
        qkv = normal(B, T, Hq + 2 * Hkv, d)
        if c["packed"]:
            s.inputs = [qkv]
        else:                                       # queries and keys of a tensor of their own, values where they were projected
            s.inputs = [qkv[:, :, :Hq].contiguous(), qkv[:, :, Hq:Hq + Hkv].contiguous(), qkv[:, :, Hq + Hkv:]]
        if grads:
            s.inputs = [t.detach().requires_grad_() for t in s.inputs]
            s.dy = normal(B, T, Hq, d, scale=1e-3)
        return s
    H = Hq + Hkv
    # the query and key heads of a packed projection output, where they lie
    s.x = normal(B, T, H + Hkv, d)[:, :, :H]
    if grads:
        s.x = s.x.detach().requires_grad_()
        s.dy = normal(B, T, H, d, scale=1e-3)
    s.positions = torch.arange(c["first"], c["first"] + T, device="cuda")
    if c["per_batch"]:
        s.positions = s.positions + torch.randint(0, 4096, (B, 1), generator=gen, device="cuda")
    half = c["rotated"] // 2
    s.inv_freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    if c["op"] == "norm":
        s.weights = [(1 + 0.3 * torch.randn(d, generator=gen, device="cuda")).bfloat16() for _ in range(2)]
        if grads:
            s.weights = [torch.nn.Parameter(w) for w in s.weights]
            s.main_grad = torch.zeros(2, d, device="cuda")         # the flat gradient buffer of a training step
            for w, g in zip(s.weights, s.main_grad):
                w.main_grad = g
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_attention(q, k, v, window, sinks):
    """fp32 `[B, T, H, d]`. Queries in blocks of `window`: a block sees itself, the block before it and the sinks."""
    B, T, Hq, d = q.shape
    Hkv = k.shape[2]
    w = max(1, min(window, T))
    S = min(sinks, T)
    n = -(-T // w)

    def blocks(t, heads):
        t = torch.nn.functional.pad(t.permute(0, 2, 1, 3), (0, 0, 0, n * w - T))
        return t.reshape(B, Hkv, heads // Hkv, n, w, d)

    def with_previous(t):
        t = blocks(t, Hkv)
        return torch.cat([torch.nn.functional.pad(t, (0, 0, 0, 0, 1, 0))[:, :, :, :-1], t], dim=4)

    qb, kb, vb = blocks(q, Hq), with_previous(k), with_previous(v)
    ks, vs = (t[:, :S].permute(0, 2, 1, 3)[:, :, None, None] for t in (k, v))
    i = torch.arange(n * w, device=q.device).view(n, w, 1)
    j = torch.arange(n, device=q.device).view(n, 1, 1) * w + torch.arange(-w, w, device=q.device)
    near = (j >= 0) & (j <= i) & (i - j < w)
    far = i - torch.arange(S, device=q.device) >= w
    scores = torch.cat([(qb @ kb.transpose(-1, -2)).masked_fill(~near, -math.inf),
                        (qb @ ks.transpose(-1, -2)).masked_fill(~far, -math.inf)], dim=-1) / math.sqrt(d)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p[..., :2 * w] @ vb + p[..., 2 * w:] @ vs
    return o.reshape(B, Hq, n * w, d)[:, :, :T].permute(0, 2, 1, 3)


def _plain_rotary(x, positions, inv_freq, interleaved):
    r = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq               # [T, r/2] or [B, T, r/2]
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], dim=-1).flatten(-2) if interleaved else torch.cat([ya, yb], dim=-1)
    return torch.cat([y, x[..., r:]], dim=-1)


def _plain(s):
    c = s.case
    grads = c["direction"] == "bwd"
    with torch.set_grad_enabled(grads):
        if c["op"] == "attn":
            leaves = [t.detach().float().requires_grad_(grads) for t in s.inputs]
            qkv = leaves[0].split([c["q_heads"], c["kv_heads"], c["kv_heads"]], dim=2) if c["packed"] else leaves
            y = _plain_attention(*qkv, c["window"], c["sinks"])
        else:
            leaves = [s.x.detach().float().requires_grad_(grads)]
            x = leaves[0]
            if c["op"] == "norm":
                leaves += [w.detach().float().requires_grad_(grads) for w in s.weights]
                x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
                x = torch.cat([x[:, :, :c["q_heads"]] * leaves[1], x[:, :, c["q_heads"]:] * leaves[2]], dim=2)
            y = _plain_rotary(x, s.positions, s.inv_freq, c["interleaved"])
        if not grads:
            return {"y": y.bfloat16()}
        dx = torch.autograd.grad(y, leaves, s.dy.float())
    out = {"y": y.detach().bfloat16()}
    if c["op"] == "norm":
        return {**out, "dx": dx[0].bfloat16(), "dw": torch.stack(dx[1:])}
    return {**out, "dx": [g.bfloat16() for g in dx]} if c["op"] == "attn" else {**out, "dx": dx[0].bfloat16()}


def _own(s):
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    c = s.case
    grads = c["direction"] == "bwd"
    with torch.set_grad_enabled(grads):
        if c["op"] == "attn":
            if c["packed"]:
                y = F_ops.attention_packed(s.inputs[0], c["q_heads"], c["kv_heads"], window=c["window"], sinks=c["sinks"])
            else:
                y = F_ops.window_attention(*s.inputs, window=c["window"], sinks=c["sinks"])
            return {"y": y.detach(), "dx": list(torch.autograd.grad(y, s.inputs, s.dy))} if grads else {"y": y}
        if c["op"] == "rotary":
            y = F_ops.rotary(s.x, s.positions, s.inv_freq, interleaved=c["interleaved"])
            return {"y": y.detach(), "dx": torch.autograd.grad(y, s.x, s.dy)[0]} if grads else {"y": y}
        y = F_ops.qk_norm_rotary(s.x, c["q_heads"], *s.weights, s.positions, s.inv_freq, eps=EPS, interleaved=c["interleaved"])
        if not grads:
            return {"y": y}
        s.main_grad.zero_()
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s.x, s.dy)[0], "dw": s.main_grad}


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    grads = c["direction"] == "bwd"
    if c["op"] == "attn":
        return _exact_attention(c, [t.detach() for t in s.inputs], s.dy if grads else None)
    x, r = s.x.detach().double(), c["rotated"]
    T, H = x.shape[1:3]
    angle = (s.positions.double()[..., None] * s.inv_freq).reshape(-1, T, 1, r // 2)
    turn = torch.polar(torch.ones_like(angle), angle)

    def pairs(t):
        t = t[..., :r]
        return torch.complex(t[..., 0::2], t[..., 1::2]) if c["interleaved"] else torch.complex(t[..., :r // 2], t[..., r // 2:])

    def turned(t, by):
        z = pairs(t) * by
        out = t.clone()
        if c["interleaved"]:
            out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
        else:
            out[..., :r // 2], out[..., r // 2:r] = z.real, z.imag
        return out

    if c["op"] == "rotary":
        return {"y": turned(x, turn), "dx": turned(s.dy.double(), turn.conj())} if grads else {"y": turned(x, turn)}
    is_q = (torch.arange(H, device=x.device) < c["q_heads"])[:, None]
    w = torch.where(is_q, s.weights[0].detach().double(), s.weights[1].detach().double())
    rstd = ((x ** 2).sum(-1, keepdim=True) / c["dim"] + EPS) ** -0.5
    hat = x * rstd
    y = turned(hat * w, turn)
    if not grads:
        return {"y": y}
    du = turned(s.dy.double(), turn.conj())
    dw = (du * hat).sum((0, 1))
    g = du * w
    dx = rstd * (g - hat * (g * hat).sum(-1, keepdim=True) / c["dim"])
    return {"y": y, "dx": dx, "dw": torch.stack([dw[:c["q_heads"]].sum(0), dw[c["q_heads"]:].sum(0)])}


def _exact_attention(c, inputs, dy):
    Hq, Hkv, T, W, S = c["q_heads"], c["kv_heads"], c["seq"], c["window"], min(c["sinks"], c["seq"])
    q, k, v = inputs[0].split([Hq, Hkv, Hkv], dim=2) if c["packed"] else inputs
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    B, d, rep = q.shape[0], q.shape[3], Hq // Hkv
    y, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    rows = max(1, min(T, 2 ** 27 // (B * Hq * (W + S + 1024)), 1024))
    for r0 in range(0, T, rows):
        r1 = min(T, r0 + rows)
        lo = max(0, r0 - W + 1)
        keys = torch.cat([torch.arange(min(S, lo), device=q.device), torch.arange(lo, r1, device=q.device)])
        i = torch.arange(r0, r1, device=q.device)[:, None]
        seen = (keys <= i) & ((i - keys < W) | (keys < S))
        ki, vi = (t[:, :, keys].repeat_interleave(rep, dim=1) for t in (k, v))
        a = torch.einsum("bhid,bhjd->bhij", q[:, :, r0:r1], ki) * d ** -0.5
        p = torch.softmax(torch.where(seen, a, torch.full_like(a, -math.inf)), dim=-1)
        y[:, :, r0:r1] = torch.einsum("bhij,bhjd->bhid", p, vi)
        if dy is not None:
            g = dy[:, r0:r1].double().transpose(1, 2)
            dp = torch.einsum("bhid,bhjd->bhij", g, vi)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * d ** -0.5
            dq[:, :, r0:r1] = torch.einsum("bhij,bhjd->bhid", ds, ki)
            n = keys.numel()
            dk.index_add_(2, keys, torch.einsum("bhij,bhid->bhjd", ds, q[:, :, r0:r1]).view(B, Hkv, rep, n, d).sum(2))
            dv.index_add_(2, keys, torch.einsum("bhij,bhid->bhjd", p, g).view(B, Hkv, rep, n, d).sum(2))
    out = {"y": y.transpose(1, 2)}
    if dy is None:
        return out
    dx = [t.transpose(1, 2) for t in (dq, dk, dv)]
    return {**out, "dx": [torch.cat(dx, dim=2)] if c["packed"] else dx}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    B, T, Hq, Hkv, d = c["batch"], c["seq"], c["q_heads"], c["kv_heads"], c["dim"]
    grads = c["direction"] == "bwd"
    row = 2 * B * T * d                                             # bytes of one head
    if c["op"] == "attn":
        full = min(c["window"], T)                                  # rows that see fewer than `window` keys, then the others
        pairs = full * (full + 1) // 2 + (T - full) * full
        sinks = min(c["sinks"], T)
        late = T - full                                             # rows that see sinks besides their window: one more each
        pairs += sum(min(sinks, n) for n in range(1, min(late, sinks) + 1)) + max(0, late - sinks) * sinks
        # q, k, v in, o out; do in, their gradients out. Two products, five more for the gradients
        heads = (Hq + 2 * Hkv) * (2 if grads else 1) + Hq * (2 if grads else 1)
        return {"bytes": heads * row, "flops": (14 if grads else 4) * d * B * Hq * pairs}
    H = Hq + Hkv
    moved = H * row * (4 if grads else 2) + 8 * T * (B if c["per_batch"] else 1)
    return {"bytes": moved, "flops": (20 if c["op"] == "norm" else 8) * H * B * T * d}
