"""GQA causal self-attention with RoPE and optional Ulysses sequence parallelism.

What the reference does in `model/modules/attn.py:126-176` with three GEMMs, a
K/V expansion to Hq heads, a freshly built fp32 RoPE table per call, stack /
transpose copies around two all-to-alls and a library SDPA call is done here as:

  one GEMM against the fused `[Hq*hd + 2*Hkv*hd, D]` weight (q|k|v are adjacent
  in the flat parameter buffer) -> RoPE on the q and k heads of the packed
  `[B, T, Hq+2Hkv, hd]` tensor (table cached per position range) -> (SP only)
  seq->head exchange of un-expanded heads -> flash attention that reads KV head
  `h // (Hq/Hkv)` directly -> (SP only) head->seq exchange -> output GEMM.

State-dict keys (`q_proj.weight`, `k_proj.weight`, `v_proj.weight`,
`c_proj.weight`) and shapes equal the reference's.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ...ops import functional as F_ops
from ...ops import oracle
from ...parallel import parallel_state
from ...parallel.flat import fuse_adjacent
from ...parallel.sequence_parallel import ulysses
from .init import seeded_normal


def rope_impl(q: torch.Tensor, k: torch.Tensor, position_ids: torch.Tensor, rope_theta: float = 10000.0,
              variant: str = "reference"):
    """Functional RoPE on `[B, H, T, hd]` tensors (API of the reference's
    `rope_impl`, `attn.py:12-68`); fp32 result."""
    pos = position_ids[0] if position_ids.dim() > 1 else position_ids
    cos, sin = oracle.rope_tables(pos, q.shape[-1], rope_theta, variant)
    qe = oracle.rope(q.transpose(1, 2), cos, sin).transpose(1, 2)
    ke = oracle.rope(k.transpose(1, 2), cos, sin).transpose(1, 2)
    return qe, ke


def gqa_impl(k: torch.Tensor, v: torch.Tensor, num_key_value_heads: int, num_attention_heads: int):
    """Expand `[B, Hkv, T, hd]` to Hq heads. Provided for API parity
    (`attn.py:71-88`); the attention op never needs it."""
    if num_attention_heads % num_key_value_heads:
        raise ValueError("num_attention_heads must be divisible by num_key_value_heads")
    rep = num_attention_heads // num_key_value_heads
    if rep == 1:
        return k, v
    return k.repeat_interleave(rep, dim=1), v.repeat_interleave(rep, dim=1)


class _Proj(nn.Module):
    """Holder of one bias-free weight so that keys read `<name>.weight`."""

    def __init__(self, out_features: int, in_features: int, std: float, seed: int, device):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = nn.Parameter(seeded_normal((out_features, in_features), std, seed, device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        y = F_ops.linear(x.reshape(-1, shape[-1]).to(self.weight.dtype), self.weight)
        return y.view(*shape[:-1], self.out_features)


class _HeadNorm(nn.Module):
    """Weight of the RMS norm of query or key heads (`<name>.weight`); the norm itself is part of the rotation."""

    def __init__(self, head_dim: int, device):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(head_dim, device=device))


class Attention(nn.Module):
    def __init__(self, config, device=None):
        super().__init__()
        config.check_attention()
        assert config.hidden_size % config.num_attention_heads == 0
        self.config = config
        self.num_attention_heads = config.num_attention_heads
        self.num_key_value_heads = config.num_key_value_heads
        self.head_dim = config.hidden_size // config.num_attention_heads
        self.n_embd = config.hidden_size
        self.dropout = config.dropout           # > 0: training steps take the library attention path (see forward)
        hd, D = self.head_dim, config.hidden_size
        self.q_proj = _Proj(self.num_attention_heads * hd, D, config.init_std, config.seed, device)
        self.k_proj = _Proj(self.num_key_value_heads * hd, D, config.init_std, config.seed, device)
        self.v_proj = _Proj(self.num_key_value_heads * hd, D, config.init_std, config.seed, device)
        self.c_proj = _Proj(D, D, config.init_std, config.seed, device)
        self.window, self.sinks = config.attn_window, config.attn_sinks
        self.rotary_op = config.rotary_op       # the rotation (and norm) is an operator of its own, behind the projection
        self.norm_epsilon = 1e-6
        if config.qk_norm:
            self.q_norm, self.k_norm = _HeadNorm(hd, device), _HeadNorm(hd, device)
        self._qkv_weight = None
        self._turn_cache: dict = {}
        self._rope_cache: dict = {}
        self._rope_cache_full: dict = {}
        self._rope_cache_fp16: dict = {}

    def _post_flatten(self) -> None:
        self._qkv_weight = fuse_adjacent([self.q_proj.weight, self.k_proj.weight, self.v_proj.weight])

    def _tables(self, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        c = self.config
        if c.rope_scaling == "none":
            return oracle.rope_tables(pos, self.head_dim, c.rope_theta, c.rope_variant)
        freq, scale = self._frequencies(pos.device)
        angle = (pos.double()[:, None] * freq).repeat(1, 2)
        return (scale * angle.cos()).float(), (scale * angle.sin()).float()

    def _frequencies(self, device) -> tuple[torch.Tensor, float]:
        c = self.config
        return oracle.rotary_frequencies(c.rotary_dim, c.rope_theta, c.rope_scaling, c.rope_scaling_factor, c.rope_original_length, device)

    def _rope(self, T_local: int, device) -> tuple[torch.Tensor, torch.Tensor]:
        start = parallel_state.get_sep_rank() * T_local
        key = (start, T_local, str(device))
        if key not in self._rope_cache:
            self._rope_cache = {key: self._tables(torch.arange(start, start + T_local, device=device))}
        return self._rope_cache[key]

    def _turn(self, T_local: int, device):
        """(positions, frequencies, factor) of this rank's tokens for the rotary operator."""
        start = parallel_state.get_sep_rank() * T_local
        key = (start, T_local, str(device))
        if key not in self._turn_cache:
            self._turn_cache = {key: (torch.arange(start, start + T_local, device=device), *self._frequencies(device))}
        return self._turn_cache[key]

    def _rope_fp16(self, T_local: int, device) -> torch.Tensor:
        """(cos, sin) pairs in fp16 for the fused projection epilogue."""
        from ...ops import native
        key = (parallel_state.get_sep_rank() * T_local, T_local, str(device))
        if key not in self._rope_cache_fp16:
            self._rope_cache_fp16 = {key: native.rope_table_fp16(*self._rope(T_local, device))}
        return self._rope_cache_fp16[key]

    def _rope_full(self, T_full: int, device) -> tuple[torch.Tensor, torch.Tensor]:
        key = ("full", T_full, str(device))
        if key not in self._rope_cache_full:
            self._rope_cache_full = {key: self._tables(torch.arange(0, T_full, device=device))}
        return self._rope_cache_full[key]

    def _symm_ok(self, x: torch.Tensor) -> bool:
        if not (x.is_cuda and x.dtype == torch.bfloat16):
            return False
        from ...parallel import symm
        return symm.use_symm()

    def _peer_path(self, qkv: torch.Tensor, sp: int) -> bool:
        from ...parallel.sequence_parallel import ulysses_peer
        return self._symm_ok(qkv) and ulysses_peer.supported(self.num_attention_heads, self.num_key_value_heads, sp,
                                                             self.head_dim)

    def forward(self, h: torch.Tensor, B: int | None = None, T_local: int | None = None) -> torch.Tensor:
        """h: `[B*T_local, D]` (or `[B, T_local, D]`) in the compute dtype -> same shape."""
        shape = h.shape
        if h.dim() == 3:
            B, T_local = shape[0], shape[1]
            h = h.reshape(-1, shape[-1])
        Hq, Hkv, hd = self.num_attention_heads, self.num_key_value_heads, self.head_dim
        h = h.to(self.q_proj.weight.dtype)
        sp = parallel_state.get_sep_world_size()
        group = parallel_state.get_sep_group()
        if self.rotary_op:
            return self._forward_rotary(h, B, T_local, sp, group).view(shape)
        cos, sin = self._rope(T_local, h.device)
        dropout_p = self.dropout if self.training else 0.0      # reference: attn.py:159
        if dropout_p > 0.0:
            return self._forward_with_dropout(h, B, T_local, cos, sin, dropout_p, sp, group).view(shape)
        if F_ops.qkv_project_fused_ok(h, self._qkv_weight, hd, T_local):
            # CUDA: projection + RoPE (+ the seq->head exchange) are one GEMM with a head-scatter epilogue
            if sp == 1:
                o = F_ops.qkv_attention(h, self._qkv_weight, cos, sin, self._rope_fp16(T_local, h.device), B, T_local,
                                        Hq, Hkv, hd, self.window, self.sinks)
                y = F_ops.linear(o.reshape(B * T_local, Hq * hd), self.c_proj.weight)
                return y.view(shape)
            from ...parallel.sequence_parallel import ulysses_peer
            if self.window == 0 and self._symm_ok(h) and ulysses_peer.fused_ok(Hq, Hkv, sp, hd, T_local):      # incl. Hkv < sp (replicated KV heads)
                cos_f, sin_f = self._rope_full(T_local * sp, h.device)
                y = ulysses_peer.attention_block(h, self._qkv_weight, self.c_proj.weight, Hq, Hkv, hd, B, T_local,
                                                 self._rope_fp16(T_local, h.device), cos_f, sin_f, id(self), group)
                return y.view(shape)
        qkv = self._project(h).view(B, T_local, Hq + 2 * Hkv, hd)
        if sp > 1 and self.window == 0 and self._peer_path(qkv, sp):
            # RoPE + seq->head exchange in one kernel writing into the head owners' memory,
            # attention, then the head->seq exchange; see parallel/sequence_parallel/ulysses_peer.py
            from ...parallel.sequence_parallel import ulysses_peer
            cos_f, sin_f = self._rope_full(T_local * sp, h.device)
            qkv_l = ulysses_peer.seq_to_head(qkv, Hq, Hkv, cos, sin, cos_f, sin_f, id(self), group)
            o = F_ops.attention_packed(qkv_l, Hq // sp, Hkv // sp, True)
            o = ulysses_peer.head_to_seq(o, Hq, id(self), group)
            y = F_ops.linear(o.reshape(B * T_local, Hq * hd), self.c_proj.weight)
            return y.view(shape)
        qkv = F_ops.rope_qk(qkv, cos, sin, Hq + Hkv)
        y = F_ops.linear(self._attend(qkv, sp, group).reshape(B * T_local, Hq * hd), self.c_proj.weight)
        return y.view(shape)

    def _project(self, h: torch.Tensor) -> torch.Tensor:
        if self._qkv_weight is not None:
            return F_ops.linear(h, self._qkv_weight)
        return torch.cat([F_ops.linear(h, self.q_proj.weight), F_ops.linear(h, self.k_proj.weight),
                          F_ops.linear(h, self.v_proj.weight)], dim=-1)

    def _attend(self, qkv: torch.Tensor, sp: int, group) -> torch.Tensor:
        """Attention on packed heads that have been rotated, with the exchanges of sequence parallelism around it."""
        if sp == 1:
            return F_ops.attention_packed(qkv, self.num_attention_heads, self.num_key_value_heads, True, self.window, self.sinks)
        qkv_l, q_l, kv_l = ulysses.seq_to_head(qkv, self.num_attention_heads, self.num_key_value_heads, group)
        return ulysses.head_to_seq(F_ops.attention_packed(qkv_l.contiguous(), q_l, kv_l, True, self.window, self.sinks), group)

    def _forward_rotary(self, h, B, T_local, sp, group) -> torch.Tensor:
        """`rotary_op`: projection, then norm and rotation in one pass, then attention."""
        Hq, Hkv, hd = self.num_attention_heads, self.num_key_value_heads, self.head_dim
        qkv = self._project(h).view(B, T_local, Hq + 2 * Hkv, hd)
        positions, freq, scale = self._turn(T_local, h.device)
        weights = (self.q_norm.weight, self.k_norm.weight) if self.config.qk_norm else None
        turn = dict(interleaved=self.config.rope_layout == "interleaved", scale=scale)
        if sp == 1 and F_ops.window_attention_ok(qkv):
            o = F_ops.rotary_attention(qkv, Hq, Hkv, positions, freq, norm_weights=weights, eps=self.norm_epsilon, window=self.window,
                                       sinks=self.sinks, **turn)
        else:
            qk, v = qkv.split([Hq + Hkv, Hkv], dim=2)
            if weights is not None:
                qk = F_ops.qk_norm_rotary(qk, Hq, *weights, positions, freq, eps=self.norm_epsilon, **turn)
            else:
                qk = F_ops.rotary(qk, positions, freq, **turn)
            o = self._attend(torch.cat([qk, v], dim=2), sp, group)
        return F_ops.linear(o.reshape(B * T_local, Hq * hd), self.c_proj.weight)

    def _forward_with_dropout(self, h, B, T_local, cos, sin, dropout_p, sp, group) -> torch.Tensor:
        """Attention-probability dropout (`--dropout > 0`, training mode). The flash kernels of this package carry no
        dropout mask, so this configuration runs projection, RoPE and the Ulysses exchanges as separate ops and the
        library's scaled-dot-product attention with `dropout_p` (what the reference calls, `attn.py:159-163`); every
        reference script trains with 0.0, which takes the fused path."""
        import warnings
        Hq, Hkv, hd = self.num_attention_heads, self.num_key_value_heads, self.head_dim
        warnings.warn("attention dropout > 0: using the library attention kernel instead of the sm_100a flash kernels",
                      stacklevel=2)
        qkv = F_ops.rope_qk(self._project(h).view(B, T_local, Hq + 2 * Hkv, hd), cos, sin, Hq + Hkv)
        q_l, kv_l = Hq, Hkv
        if sp > 1:
            qkv, q_l, kv_l = ulysses.seq_to_head(qkv, Hq, Hkv, group)
        q, k, v = qkv.split([q_l, kv_l, kv_l], dim=2)
        o = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), dropout_p=dropout_p, is_causal=True,
            enable_gqa=q_l != kv_l).transpose(1, 2).contiguous()
        if sp > 1:
            o = ulysses.head_to_seq(o, group)
        return F_ops.linear(o.reshape(B * T_local, Hq * hd), self.c_proj.weight)
