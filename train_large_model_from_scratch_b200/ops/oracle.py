"""Plain-PyTorch definitions of every op in the model, written for clarity.

These are the numerical oracle for the CUDA kernels (tests compare a kernel
with the function here evaluated in fp32) and the execution path on CPU
(Gloo runs, fp32). They restate the math of the reference modules:
RMSNorm `model/modules/norm.py:14-19`, the RoPE variant of
`model/modules/attn.py:12-68`, GQA causal attention `attn.py:71-88,160-163`,
SwiGLU `model/modules/mlp.py:44`, top-k-then-softmax routing `mlp.py:100-103`,
and the masked-sum cross-entropy of `model/modules/loss.py:19-36`.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return weight.float() * (xf * rstd)


def rope_tables(positions: torch.Tensor, head_dim: int, theta: float = 10000.0,
                variant: str = "reference") -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables `[T, head_dim]` in fp32.

    variant "reference": frequency i occupies ADJACENT slots (2i, 2i+1) —
    `[c0,c0,c1,c1,...]` — while the rotation still pairs slot j with j +- hd/2.
    That is what the reference computes; it is a fixed linear map per position
    but not the usual norm-preserving rotation.
    variant "standard": frequency i occupies slots i and i + hd/2.
    """
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=positions.device) / head_dim))
    freqs = torch.outer(positions.float(), inv_freq)            # [T, hd/2]
    if variant == "reference":
        full = freqs.repeat_interleave(2, dim=-1)                # c0,c0,c1,c1,...
    else:
        full = torch.cat([freqs, freqs], dim=-1)                 # c0..c_{hd/2-1}, c0..
    return full.cos(), full.sin()


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def rotate_half_t(x: torch.Tensor) -> torch.Tensor:
    """Transpose of `rotate_half` (used by the RoPE backward)."""
    h = x.shape[-1] // 2
    return torch.cat((x[..., h:], -x[..., :h]), dim=-1)


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x: [B, T, H, hd]; cos/sin: [T, hd]. fp32 math, fp32 result."""
    xf = x.float()
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    return xf * c + rotate_half(xf) * s


def rope_bwd(dy: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    df = dy.float()
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    return df * c + rotate_half_t(df * s)


ROPE_SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 4096, device=None) -> tuple[torch.Tensor, float]:
    """Frequencies (float64 `[rotary_dim / 2]`, radians per position) and the factor on cos and sin, for `rotary`.

    scaling "linear": positions are divided by `factor`. "ntk": theta grows so that the slowest pair turns `factor` times slower.
    "yarn": pairs that turn more than 32 times within `original_length` stay, those below one turn are divided by `factor`, with
    a linear ramp over the pair index between, which may end behind the last pair (where that turns more than once); cos and sin
    are multiplied by 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, not {rotary_dim}")
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}: one of {ROPE_SCALINGS}")
    if theta <= 1.0 or factor < 1.0 or original_length < 1:
        raise ValueError("theta has to be above 1, factor at least 1, original_length positive")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("scaling 'ntk' needs a rotary_dim of at least 4")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    freq = theta ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    if scaling != "yarn":
        return freq, 1.0

    def pair_of(turns: float) -> float:           # index of the pair that turns so often within original_length
        return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(0, math.floor(pair_of(32.0))), min(rotary_dim - 1, math.ceil(pair_of(1.0)))
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
    return freq * (1.0 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
           inverse: bool = False) -> torch.Tensor:
    """x: `[B, T, H, hd]`; positions `[T]` or `[B, T]`; the first 2 * len(inv_freq) of a head turn, pairs (i, i + len) or (2i, 2i + 1).
    `inverse`: the transposed map (backward). Angles in 64 bits, the rest in 32."""
    r = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    cos, sin = (scale * f(angle).float()[..., None, :] for f in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    xf = x.float()
    a, b = (xf[..., 0:r:2], xf[..., 1:r:2]) if interleaved else (xf[..., :r // 2], xf[..., r // 2:r])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], dim=-1).flatten(-2) if interleaved else torch.cat([ya, yb], dim=-1)
    return torch.cat([y, xf[..., r:]], dim=-1)


def window_mask(T: int, window: int, sinks: int, device=None) -> torch.Tensor:
    """`[T, T]` bool: does query row see key column? `window` 0: every key up to the query."""
    i, j = torch.arange(T, device=device)[:, None], torch.arange(T, device=device)
    seen = j <= i
    return seen if window <= 0 else seen & ((i - j < window) | (j < sinks))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
              q_offset: int = 0) -> torch.Tensor:
    """q: [B, Tq, Hq, hd], k/v: [B, Tk, Hkv, hd] -> [B, Tq, Hq, hd].
    Query row i sits at absolute position `q_offset + i`; key j at j."""
    B, Tq, Hq, hd = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    rep = Hq // Hkv
    qf = q.float().permute(0, 2, 1, 3)                                   # B,Hq,Tq,hd
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    s = qf @ kf.transpose(-1, -2) / math.sqrt(hd)
    if causal:
        qi = torch.arange(Tq, device=q.device)[:, None] + q_offset
        kj = torch.arange(Tk, device=q.device)[None, :]
        s = s.masked_fill(kj > qi, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return (p @ vf).permute(0, 2, 1, 3)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """gate_up: [..., 2I] with gate in the first half -> silu(gate) * up."""
    g, u = gate_up.float().chunk(2, dim=-1)
    return F.silu(g) * u


def mlp(x, w_gate, w_up, w_down):
    xf = x.float()
    return (F.silu(xf @ w_gate.float().t()) * (xf @ w_up.float().t())) @ w_down.float().t()


def router_topk(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """top-k on raw logits, THEN softmax over the k winners."""
    vals, idx = torch.topk(logits.float(), k, dim=-1)
    return torch.softmax(vals, dim=-1), idx


def moe(x: torch.Tensor, w_router, w_gate, w_up, w_down, k: int) -> torch.Tensor:
    """Dropless MoE, all experts local. x: [M, D]; w_gate/up: [E, I, D]; w_down: [E, D, I]."""
    xf = x.float()
    weights, experts = router_topk(xf @ w_router.float().t(), k)
    out = torch.zeros_like(xf)
    for e in range(w_gate.shape[0]):
        tok, slot = (experts == e).nonzero(as_tuple=True)
        if tok.numel() == 0:
            continue
        y = mlp(xf[tok], w_gate[e], w_up[e], w_down[e])
        out.index_add_(0, tok, y * weights[tok, slot, None])
    return out


def moe_aux_stats(logits: torch.Tensor, experts: torch.Tensor, num_experts: int) -> torch.Tensor:
    """Switch-style load-balance term  E * sum_e f_e * p_e  with f_e the fraction
    of routed slots that chose e and p_e the mean full-softmax probability."""
    probs = torch.softmax(logits.float(), dim=-1).mean(0)
    frac = torch.bincount(experts.reshape(-1), minlength=num_experts).float() / experts.numel()
    return num_experts * (frac * probs).sum()


def cross_entropy_sum(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100):
    """(sum of per-token CE over valid targets, number of valid targets), fp32."""
    per_tok = F.cross_entropy(logits.float(), targets, ignore_index=ignore_index, reduction="none")
    valid = targets != ignore_index
    return (per_tok * valid).sum(), valid.sum().float()


def adamw_step(p, g, m, v, step: int, lr: float, beta1: float, beta2: float, eps: float, wd: float,
               grad_scale: float = 1.0):
    """One decoupled-weight-decay Adam step on fp32 tensors, in place.
    Same update as `torch.optim.AdamW` (non-amsgrad)."""
    g = g * grad_scale
    p.mul_(1.0 - lr * wd)
    m.mul_(beta1).add_(g, alpha=1.0 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1.0 - beta2)
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
    p.addcdiv_(m, denom, value=-lr / bc1)
