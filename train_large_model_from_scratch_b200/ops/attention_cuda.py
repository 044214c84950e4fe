"""CUDA attention entry points used by `ops.native`: the tcgen05 flash-attention
kernels for head dims 32, 64 and 128.

Other head dims (and non-causal calls) go to the library SDPA kernels through
ATen (a library call, like a cuBLAS GEMM).
"""
from __future__ import annotations

import functools
import math

import torch

from . import native


def _native_ok(hd: int) -> bool:
    return hd in (32, 64, 128)


_WARNED: set = set()


def _warn_library_path(hd: int, causal: bool) -> None:
    """Said once per shape class: a configuration must never be measured on the library kernels unnoticed."""
    key = (hd, causal)
    if key not in _WARNED:
        _WARNED.add(key)
        import warnings
        warnings.warn(f"attention with head dim {hd}, causal={causal} is outside the tcgen05 kernels "
                      f"(head dims 32 / 64 / 128, causal): running the library SDPA kernels instead",
                      RuntimeWarning, stacklevel=3)


def fwd(qkv: torch.Tensor, n_q: int, n_kv: int, causal: bool):
    """qkv `[B, T, n_q + 2 n_kv, hd]` bf16 -> (o `[B, T, n_q, hd]` bf16, lse `[B, n_q, T]` fp32)."""
    B, T, _, hd = qkv.shape
    if causal and _native_ok(hd):
        assert qkv.is_contiguous()
        o = torch.empty(B, T, n_q, hd, dtype=torch.bfloat16, device=qkv.device)
        lse = torch.empty(B, n_q, T, dtype=torch.float32, device=qkv.device)
        native._check(native.lib().tlm_attn_fwd(qkv.data_ptr(), o.data_ptr(), lse.data_ptr(), B, T, n_q, n_kv, hd,
                                                1.0 / math.sqrt(hd), native._stream()), "attn_fwd")
        return o, lse
    _warn_library_path(hd, causal)
    q, k, v = _split(qkv, n_q, n_kv)
    out = torch.ops.aten._scaled_dot_product_flash_attention(q, k, v, 0.0, causal, False)
    return out[0].transpose(1, 2).contiguous(), out[1]


def fwd_scatter(qkv: torch.Tensor, n_q: int, n_kv: int, dst_ptrs, n_dst: int, dst_rows: int, dst_heads: int,
                dst_head0: int):
    """Causal attention (head dims 32 / 64 / 128) whose epilogue also stores each output row into
    `dst[t // dst_rows][b, t % dst_rows, dst_head0 + h, :]` (`dst_ptrs`: ctypes array of device addresses of
    bf16 `[B, dst_rows, dst_heads, hd]` tensors, typically peers' symmetric buffers)."""
    B, T, _, hd = qkv.shape
    assert _native_ok(hd) and qkv.is_contiguous()
    o = torch.empty(B, T, n_q, hd, dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty(B, n_q, T, dtype=torch.float32, device=qkv.device)
    native._check(native.lib().tlm_attn_fwd_scatter(qkv.data_ptr(), o.data_ptr(), lse.data_ptr(), B, T, n_q, n_kv, hd,
                                                    1.0 / math.sqrt(hd), dst_ptrs, n_dst, dst_rows, dst_heads,
                                                    dst_head0, native._stream()), "attn_fwd_scatter")
    return o, lse


def bwd_scatter(do, qkv, o, lse, n_q: int, n_kv: int, rope, dst_ptrs, n_dst: int, dst_rows: int, dst_heads: int,
                dst_q0: int, dst_k0: int, dst_v0: int) -> None:
    """Causal attention backward (head dims 32 / 64 / 128) whose gradient rows are stored straight into the sequence
    owners' packed gradient tensors: row t of local q head s -> `dst[t // dst_rows][b, t % dst_rows, dst_q0 + s]`,
    k -> `dst_k0 + s`, v -> `dst_v0 + s` (`dst_ptrs`: ctypes array of device addresses of bf16
    `[B, dst_rows, dst_heads, hd]` tensors, typically peers' symmetric buffers). `rope = (cos, sin)` fp32 `[T, hd]`
    or None: transposed rotation of dQ / dK on the way."""
    B, T, _, hd = qkv.shape
    assert _native_ok(hd) and qkv.is_contiguous()
    do, o = do.contiguous(), o.contiguous()
    dq_acc = torch.empty(B, n_q, T, hd, dtype=torch.float32, device=qkv.device)
    delta = torch.empty(B, n_q, T, dtype=torch.float32, device=qkv.device)
    cos, sin = rope if rope is not None else (None, None)
    native._check(native.lib().tlm_attn_bwd_scatter(
        qkv.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(), dq_acc.data_ptr(), delta.data_ptr(), B, T, n_q, n_kv,
        hd, 1.0 / math.sqrt(hd), native._ptr(cos), native._ptr(sin), dst_ptrs, n_dst, dst_rows, dst_heads, dst_q0, dst_k0,
        dst_v0, native._stream()), "attn_bwd_scatter")


def _split(qkv, n_q, n_kv):
    q = qkv[:, :, :n_q].transpose(1, 2)
    k = qkv[:, :, n_q:n_q + n_kv].transpose(1, 2)
    v = qkv[:, :, n_q + n_kv:].transpose(1, 2)
    rep = n_q // n_kv
    if rep > 1:
        k, v = k.repeat_interleave(rep, dim=1), v.repeat_interleave(rep, dim=1)
    return q, k, v


def bwd(do, qkv, o, lse, n_q: int, n_kv: int, causal: bool, rope=None):
    """-> dqkv `[B, T, n_q + 2 n_kv, hd]` bf16 (gradient of the packed input). With `rope = (cos, sin)` (fp32
    `[T, hd]`) the q and k parts are the gradient of the UN-rotated heads (transposed RoPE applied in the kernels)."""
    B, T, _, hd = qkv.shape
    if causal and _native_ok(hd):
        do, o = do.contiguous(), o.contiguous()
        dqkv = torch.empty_like(qkv)
        dq_acc = torch.empty(B, n_q, T, hd, dtype=torch.float32, device=qkv.device)
        delta = torch.empty(B, n_q, T, dtype=torch.float32, device=qkv.device)
        cos, sin = rope if rope is not None else (None, None)
        if cos is not None:
            assert cos.dtype == torch.float32 and cos.shape == (T, hd) and cos.is_contiguous() and sin.is_contiguous()
        native._check(native.lib().tlm_attn_bwd(qkv.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(),
                                                dqkv.data_ptr(), dq_acc.data_ptr(), delta.data_ptr(), B, T, n_q, n_kv,
                                                hd, 1.0 / math.sqrt(hd), native._ptr(cos), native._ptr(sin),
                                                native._stream()), "attn_bwd")
        return dqkv
    assert rope is None, "the transposed rotation is part of the tcgen05 kernels only"
    _warn_library_path(hd, causal)
    rep = n_q // n_kv
    q, k, v = _split(qkv, n_q, n_kv)
    zero = torch.zeros((), dtype=torch.int64, device=qkv.device)
    dq, dk, dv = torch.ops.aten._scaled_dot_product_flash_attention_backward(
        do.transpose(1, 2), q, k, v, o.transpose(1, 2), lse, None, None, T, T, 0.0, causal, zero, zero)
    if rep > 1:
        dk = dk.reshape(B, n_kv, rep, T, hd).sum(2)
        dv = dv.reshape(B, n_kv, rep, T, hd).sum(2)
    return torch.cat([dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2)], dim=2).contiguous()


def _tiled(t: torch.Tensor) -> torch.Tensor:
    """`t [B, T, H, hd]` as tiles can be loaded from it: rows contiguous, 16-byte aligned, at strides of whole 16 bytes. Anything
    else is copied (a broadcast tensor, an odd slice)."""
    b, r, h, c = t.stride()
    ok = c == 1 and t.data_ptr() % 16 == 0 and b > 0 and r > 0 and h > 0 and (b | r | h) % 8 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _window_fwd(q: int, k: int, v: int, strides, B: int, T: int, n_q: int, n_kv: int, hd: int, window: int, sinks: int, device,
                rest: bool):
    o = torch.empty((B, T, n_q, hd), dtype=torch.bfloat16, device=device)
    o_rest = torch.empty((B, _rest_rows(T, min(window, T), min(sinks, T)), n_q, hd), dtype=torch.bfloat16, device=device) if rest else None
    lse = torch.empty((B, n_q, T), dtype=torch.float32, device=device)
    native._check(native.lib().tlm_attn_window_fwd(q, k, v, strides, o.data_ptr(), native._ptr(o_rest), lse.data_ptr(), B, T, n_q,
                                                   n_kv, hd, 1.0 / math.sqrt(hd), min(window, T), min(sinks, T), native._stream()), "attn_window_fwd")
    return o, lse, o_rest


@functools.lru_cache(maxsize=1024)
def _rest_rows(T: int, window: int, sinks: int) -> int:
    return native.lib().tlm_attn_window_rest_rows(T, window, sinks)


@functools.lru_cache(maxsize=1024)
def _part_floats(B: int, T: int, n_kv: int, hd: int, window: int, sinks: int) -> int:
    return native.lib().tlm_attn_window_part_floats(B, T, n_kv, hd, window, sinks)


def _window_bwd(do, q: int, k: int, v: int, strides, o, lse, o_rest, dq: int, dk: int, dv: int, out_strides, B: int, T: int, n_q: int, n_kv: int,
                hd: int, window: int, sinks: int, rope) -> None:
    do = _aligned(do)
    window, sinks = min(window, T), min(sinks, T)
    l = native.lib()
    rows = B * n_q * T                                       # scratch: dQ in fp32, sums of the sink rows, delta
    part = rows * hd
    delta = part + _part_floats(B, T, n_kv, hd, window, sinks)
    work = torch.empty(delta + rows, dtype=torch.float32, device=do.device)
    w = work.data_ptr()
    cos, sin = (t.data_ptr() for t in rope) if rope is not None else (None, None)
    native._check(l.tlm_attn_window_bwd(q, k, v, strides, o.data_ptr(), native._ptr(o_rest), do.data_ptr(), lse.data_ptr(), dq, dk, dv, out_strides, w,
                                        w + 4 * delta, w + 4 * part, B, T, n_q, n_kv, hd, 1.0 / math.sqrt(hd), cos, sin, window, sinks,
                                        native._stream()), "attn_window_bwd")


def _packed(qkv: torch.Tensor, n_q: int, n_kv: int):
    """Addresses of the q, k and v heads of a packed tensor, and their strides (the same three times)."""
    s = qkv.stride()[:3]
    head = qkv.element_size() * s[2]
    p = qkv.data_ptr()
    return p, p + n_q * head, p + (n_q + n_kv) * head, native._LL9(*s, *s, *s)


def window_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int, rest: bool = False):
    """Causal attention of `q [B, T, Hq, hd]` over `k`, `v [B, T, Hkv, hd]` (bf16, hd 32 / 64 / 128, strided) where a query sees
    `window` keys, itself included (0: all), and the first `sinks`. -> o `[B, T, Hq, hd]` bf16, lse `[B, Hq, T]` fp32 and, with `rest`,
    what rounding took off o in the first rows, or in all where none sees many keys (bf16, for the backward)."""
    q, k, v = _tiled(q), _tiled(k), _tiled(v)
    B, T, n_q, hd = q.shape
    strides = native._LL9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    return _window_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, B, T, n_q, k.shape[2], hd, window, sinks, q.device,
                       rest)


def window_fwd_packed(qkv: torch.Tensor, n_q: int, n_kv: int, window: int, sinks: int, rest: bool = False):
    """The same on the heads of `qkv [B, T, n_q + 2 n_kv, hd]`."""
    qkv = _tiled(qkv)
    B, T, _, hd = qkv.shape
    return _window_fwd(*_packed(qkv, n_q, n_kv), B, T, n_q, n_kv, hd, window, sinks, qkv.device, rest)


def window_bwd(do, q, k, v, o, lse, o_rest, window: int, sinks: int, out, rope=None) -> None:
    """Gradients of `window_fwd` into `out = (dq, dk, dv)` (bf16, rows contiguous, 16-byte aligned). `rope`: as in `bwd`."""
    q, k, v = _tiled(q), _tiled(k), _tiled(v)
    B, T, n_q, hd = q.shape
    strides, out_strides = (native._LL9(*a.stride()[:3], *b.stride()[:3], *c.stride()[:3]) for a, b, c in ((q, k, v), out))
    _window_bwd(do, q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, o, lse, o_rest, *(t.data_ptr() for t in out), out_strides, B, T, n_q,
                k.shape[2], hd, window, sinks, rope)


def window_bwd_packed(do, qkv, o, lse, o_rest, n_q: int, n_kv: int, window: int, sinks: int, rope=None) -> torch.Tensor:
    """-> gradient of the packed tensor."""
    qkv = _tiled(qkv)
    B, T, H, hd = qkv.shape
    dqkv = torch.empty((B, T, H, hd), dtype=torch.bfloat16, device=qkv.device)
    _window_bwd(do, *_packed(qkv, n_q, n_kv), o, lse, o_rest, *_packed(dqkv, n_q, n_kv), B, T, n_q, n_kv, hd, window, sinks, rope)
    return dqkv
