"""Window attention with sinks, rotary positions, norms of queries and keys: the torch path (fp32) against autograd of the definitions in
64 bits, refusals, configuration, and the layer through the trainer on several ranks."""
import math
import shutil
import tempfile

import pytest
import torch

from dist_utils import TINY, run_trainer
from train_large_model_from_scratch_b200.models import GPT
from train_large_model_from_scratch_b200.ops import functional as Fo
from train_large_model_from_scratch_b200.ops import oracle
from train_large_model_from_scratch_b200.training import build_config, parse_args
from train_large_model_from_scratch_b200.training.config import ModelConfig


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _attention(q, k, v, window, sinks):
    rep = q.shape[2] // k.shape[2]
    q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(rep, 1), v.transpose(1, 2).repeat_interleave(rep, 1)
    T = q.shape[2]
    seen = torch.tensor([[j <= i and (window == 0 or i - j < window or j < sinks) for j in range(T)] for i in range(T)], dtype=torch.bool).view(T, T)
    p = torch.softmax((q @ k.mT / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf), -1)
    return (p @ v).transpose(1, 2)


def _turned(x, pos, freq, interleaved, scale):
    out = x.clone()
    r = 2 * len(freq)
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            at = float(pos[b, t] if pos.dim() == 2 else pos[t])
            for i, f in enumerate(freq.tolist()):
                a, c = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
                co, si = scale * math.cos(at * f), scale * math.sin(at * f)
                out[b, t, :, a] = x[b, t, :, a] * co - x[b, t, :, c] * si
                out[b, t, :, c] = x[b, t, :, c] * co + x[b, t, :, a] * si
    return out


def _grads(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("T,window,sinks", [(1, 3, 1), (9, 1, 0), (9, 1, 2), (9, 4, 0), (9, 4, 2), (9, 4, 100), (9, 100, 3), (9, 0, 0)])
def test_window_attention(T, window, sinks):
    qkv, do = _randn(2, T, 8, 4, seed=1), _randn(2, T, 4, 4, seed=2)
    x64 = qkv.double().requires_grad_()
    o64 = _attention(*x64.split([4, 2, 2], 2), window, sinks)
    (g64,) = _grads(o64, x64, do.double())
    x = qkv.requires_grad_()
    o = Fo.attention_packed(x, 4, 2, window=window, sinks=sinks)
    torch.testing.assert_close(o.double(), o64, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(_grads(o, x, do)[0].double(), g64, rtol=1e-4, atol=1e-5)
    leaves = [t.detach().clone().requires_grad_() for t in qkv.split([4, 2, 2], 2)]
    o = Fo.window_attention(*leaves, window=window, sinks=sinks)
    torch.testing.assert_close(torch.cat(_grads(o, leaves, do), 2).double(), g64, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("r,per_batch", [(8, False), (4, True), (2, False)])
def test_rotary_and_norm(interleaved, r, per_batch):
    x, dy = _randn(2, 3, 5, 8, seed=3), _randn(2, 3, 5, 8, seed=4)
    pos = torch.tensor([[0, 5, -7], [1, 1 << 20, 3]]) if per_batch else torch.tensor([0, 1, 1000])
    freq = 100.0 ** (-torch.arange(r // 2, dtype=torch.float64) * 2 / r)
    x64 = x.double().requires_grad_()
    y64 = _turned(x64, pos, freq, interleaved, 1.5)
    leaf = x.clone().requires_grad_()
    y = Fo.rotary(leaf, pos, freq, interleaved=interleaved, scale=1.5)
    torch.testing.assert_close(y.double(), y64, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(_grads(y, leaf, dy)[0].double(), _grads(y64, x64, dy.double())[0], rtol=1e-5, atol=1e-5)

    w = [1 + _randn(8, seed=5 + i) for i in range(2)]
    w64 = [t.double().requires_grad_() for t in w]
    u = x64 * torch.rsqrt(x64.pow(2).mean(-1, keepdim=True) + 1e-6)
    u = torch.cat([u[:, :, :3] * w64[0], u[:, :, 3:] * w64[1]], 2)
    y64 = _turned(u, pos, freq, interleaved, 1.5)
    want = _grads(y64, [x64, *w64], dy.double())
    params = [torch.nn.Parameter(t.clone()) for t in w]
    y = Fo.qk_norm_rotary(leaf, 3, *params, pos, freq, interleaved=interleaved, scale=1.5)
    got = [_grads(y, leaf, dy)[0], *(p.main_grad for p in params)]
    torch.testing.assert_close(y.double(), y64, rtol=1e-5, atol=1e-5)
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("norm", [False, True])
def test_rotary_attention_is_the_two_in_a_row(norm):
    qkv, do = _randn(2, 6, 8, 8, seed=7), _randn(2, 6, 4, 8, seed=8)
    pos, freq = torch.arange(6), torch.tensor([1.0, 0.1], dtype=torch.float64)
    weights = [1 + 0.5 * _randn(8, seed=9 + i) for i in range(2)]
    results = []
    for fused in (True, False):
        x = qkv.clone().requires_grad_()
        params = [torch.nn.Parameter(t.clone()) for t in weights] if norm else None
        if fused:
            o = Fo.rotary_attention(x, 4, 2, pos, freq, interleaved=True, scale=1.25, norm_weights=params, window=3, sinks=1)
        else:
            qk, v = x.split([6, 2], 2)
            qk = Fo.qk_norm_rotary(qk, 4, *params, pos, freq, interleaved=True, scale=1.25) if norm else Fo.rotary(qk, pos, freq, interleaved=True, scale=1.25)
            o = Fo.window_attention(qk[:, :, :4], qk[:, :, 4:], v, 3, 1)
        results.append([o.detach(), *_grads(o, x, do), *(p.main_grad for p in params or [])])
    for a, b in zip(*results):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_a_buffer_changed_between_forward_and_backward_is_noticed():
    pos = torch.arange(4)
    y = Fo.rotary(_randn(1, 4, 1, 4).requires_grad_(), pos, torch.ones(2, dtype=torch.float64))
    pos += 1
    with pytest.raises(RuntimeError, match="modified in place"):
        y.sum().backward()


def test_frequencies():
    base, one = oracle.rotary_frequencies(8, 10000.0)
    torch.testing.assert_close(base, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12, atol=0)
    assert one == 1.0
    torch.testing.assert_close(oracle.rotary_frequencies(8, 10000.0, "linear", 4.0)[0], base / 4, rtol=1e-12, atol=0)
    ntk = oracle.rotary_frequencies(8, 10000.0, "ntk", 4.0)[0]
    assert ntk[0] == 1.0 and abs(ntk[-1] / base[-1] - 0.25) < 1e-12          # the slowest pair turns four times slower
    yarn, factor = oracle.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096)
    plain = oracle.rotary_frequencies(64, 10000.0)[0]
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40]) and torch.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 8)
    assert (yarn <= plain).all() and (yarn >= plain / 8).all() and abs(factor - (0.1 * math.log(8) + 1)) < 1e-12
    for bad in (dict(rotary_dim=3), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="linear", factor=0.5), dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            oracle.rotary_frequencies(**bad)


@pytest.mark.parametrize("dim,theta,length,factor,low,high", [
    # low, high: the pairs floor(dim ln(length / 64 pi) / 2 ln(theta)) and ceil(dim ln(length / 2 pi) / 2 ln(theta)), worked out by hand
    (8, 10000.0, 8192, 8.0, 1, 4),           # 1.61 and 3.12: the last pair (3) turns 1.30 times and is on the ramp
    (64, 10000.0, 131072, 8.0, 22, 35),      # 22.51 and 34.55
    (16, 10000.0, 32768, 4.0, 4, 8),         # 4.42 and 7.43
    (64, 10000.0, 4096, 8.0, 10, 23),        # 10.47 and 22.51: ends inside the head
    (4, 10.0, 1 << 20, 2.0, 7, 3)])          # 7.43 and 10.45, at most dim - 1: every pair turns more than 32 times and stays
def test_the_ramp_may_end_behind_the_last_pair(dim, theta, length, factor, low, high):
    freq = oracle.rotary_frequencies(dim, theta, "yarn", factor, length)[0].tolist()
    for i, f in enumerate(freq):
        part = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)          # of the way from 1 to 1 / factor
        assert abs(f * theta ** (2 * i / dim) - (1 - part + part / factor)) < 1e-12, i


def test_refusals():
    qkv, pos, freq, w = _randn(1, 4, 4, 8), torch.arange(4), torch.ones(4, dtype=torch.float64), torch.ones(8)
    for call, match in (
            (lambda: Fo.attention_packed(qkv, 2, 1, causal=False, window=2), "causal"),
            (lambda: Fo.attention_packed(qkv, 3, 1, window=2), "qkv has to be"),
            (lambda: Fo.attention_packed(qkv, 2, 1, sinks=2), "sinks need a window"),
            (lambda: Fo.attention_packed(qkv, 2, 1, window=-1), "negative"),
            (lambda: Fo.window_attention(qkv[:, :, :3], qkv[:, :, :2], qkv[:, :, :2], 2), "multiple"),
            (lambda: Fo.window_attention(qkv, qkv[:, :2], qkv[:, :2], 2), "expected"),
            (lambda: Fo.window_attention(qkv, qkv.double(), qkv.double(), 2), "one type"),
            (lambda: Fo.rotary(qkv[0], pos, freq), "x has to be"),
            (lambda: Fo.rotary(qkv[..., :7], pos, freq), "head dim 7"),
            (lambda: Fo.rotary(_randn(1, 4, 1, 258), pos, freq), "head dim 258"),
            (lambda: Fo.rotary(qkv, pos.int(), freq), "positions"),
            (lambda: Fo.rotary(qkv, pos[:3], freq), "positions"),
            (lambda: Fo.rotary(qkv, pos, freq.float()), "inv_freq"),
            (lambda: Fo.rotary(qkv, pos, torch.ones(5, dtype=torch.float64)), "inv_freq"),
            (lambda: Fo.qk_norm_rotary(qkv, 5, w, w, pos, freq), "n_q 5"),
            (lambda: Fo.qk_norm_rotary(qkv, 2, w, torch.ones(4), pos, freq), "weights"),
            (lambda: Fo.rotary_attention(qkv, 3, 1, pos, freq), "qkv has to be")):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("eps", [-1e-6, float("nan")])
def test_a_negative_eps_is_refused(eps):
    qkv, pos, freq, w = _randn(1, 4, 4, 8), torch.arange(4), torch.ones(4, dtype=torch.float64), torch.ones(8)
    with pytest.raises(ValueError, match="eps"):
        Fo.qk_norm_rotary(qkv, 2, w, w, pos, freq, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        Fo.rotary_attention(qkv, 2, 1, pos, freq, norm_weights=(w, w), eps=eps)


def test_a_window_without_a_kernel_is_refused_when_the_model_is_built():
    with pytest.raises(ValueError, match="head dim 8"):
        GPT(_tiny(attn_window=4), device="cuda")
    GPT(_tiny(attn_window=4), device="cpu")


def _with_tangent(call, x, *others):
    """`call` on `x` with a tangent, under forward-mode derivatives; the tangent of the result."""
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        return fwad.unpack_dual(call(fwad.make_dual(x, torch.ones_like(x)), *others)).tangent


def test_a_tangent_is_followed_or_refused(monkeypatch):
    """The torch path differentiates forward; the kernels (stood in for here) cannot, and say so."""
    from train_large_model_from_scratch_b200.ops import attention_cuda, native
    qkv, pos, freq, w = _randn(1, 4, 4, 32), torch.arange(4), torch.ones(16, dtype=torch.float64), torch.ones(32)
    calls = [(lambda x: Fo.rotary(x, pos, freq), qkv), (lambda x: Fo.qk_norm_rotary(x, 2, w, w, pos, freq), qkv),
             (lambda x: Fo.qk_norm_rotary(qkv, 2, x, w, pos, freq), w), (lambda x: Fo.attention_packed(x, 2, 1, window=2), qkv),
             (lambda x: Fo.window_attention(qkv[:, :, :2], x, qkv[:, :, 3:], 2), qkv[:, :, 2:3])]
    for call, x in calls:
        t, h = _with_tangent(call, x), 1e-2
        # the third derivative of a softmax or a norm of size 1, times h^2 / 6, and 2^-24 / h of the results
        torch.testing.assert_close(t, (call(x + h) - call(x - h)) / (2 * h), rtol=1e-2, atol=1e-3)
    monkeypatch.setattr(Fo, "_use_native", lambda *a: True)
    monkeypatch.setattr(native, "qk_rotary", lambda x, *a, **k: x.clone())
    monkeypatch.setattr(attention_cuda, "window_fwd", lambda q, *a, **k: (q.clone(), q.new_zeros(()), None))
    monkeypatch.setattr(attention_cuda, "window_fwd_packed", lambda x, n_q, *a, **k: (x[:, :, :n_q].clone(), x.new_zeros(()), None))
    grads = qkv.clone().requires_grad_()
    calls += [(lambda x: Fo.qk_norm_rotary(grads, 2, x, w, pos, freq), w), (lambda x: Fo.rotary_attention(x, 2, 1, pos, freq), qkv),
              (lambda x: Fo.rotary_attention(grads, 2, 1, pos, freq, norm_weights=(w, x)), w)]
    for call, x in calls:
        with pytest.raises(RuntimeError, match="jvp"):
            _with_tangent(call, x)


def test_derivatives_by_the_frequencies_are_refused():
    import torch.autograd.forward_ad as fwad
    qkv, pos, w = _randn(1, 4, 4, 8), torch.arange(4), torch.ones(8)
    freq = torch.ones(4, dtype=torch.float64, requires_grad=True)
    calls = (lambda f: Fo.rotary(qkv, pos, f), lambda f: Fo.qk_norm_rotary(qkv, 2, w, w, pos, f), lambda f: Fo.rotary_attention(qkv, 2, 1, pos, f))
    for call in calls:
        with pytest.raises(ValueError, match="constant"):
            call(freq)
        with torch.no_grad():
            call(freq)
        with fwad.dual_level(), pytest.raises(ValueError, match="constant"):
            call(fwad.make_dual(freq.detach(), torch.ones(4, dtype=torch.float64)))


def test_config():
    flags = ["--rope_variant", "standard", "--qk_norm", "--rope_layout", "interleaved", "--rope_fraction", "0.5", "--rope_scaling", "yarn",
             "--rope_scaling_factor", "4", "--attn_window", "64", "--attn_sinks", "4"]
    m = build_config(parse_args(flags)).model
    assert (m.attn_window, m.attn_sinks, m.qk_norm, m.rope_layout, m.rotary_dim, m.rope_scaling) == (64, 4, True, "interleaved", m.head_dim // 2, "yarn")
    assert not ModelConfig().rotary_op and not build_config(parse_args([])).model.rotary_op
    for bad in (dict(attn_sinks=4), dict(attn_window=-1), dict(rope_layout="other"), dict(rope_scaling="other"), dict(rope_scaling_factor=0.5),
                dict(rope_fraction=0.0), dict(rope_fraction=0.3), dict(qk_norm=True, rope_variant="reference"), dict(qk_norm=True, dropout=0.1),
                dict(attn_window=8, dropout=0.1)):
        with pytest.raises(ValueError):
            ModelConfig(**{"rope_variant": "standard", "hidden_size": 64, "num_attention_heads": 4, "num_key_value_heads": 2, **bad}).check_attention()


def _tiny(**kw):
    return ModelConfig(**{**dict(num_layer=2, hidden_size=32, num_attention_heads=4, num_key_value_heads=2, intermediate_size=64, vocab_size=64,
                                 block_size=32, rope_variant="standard"), **kw})


def test_scaled_tables_are_the_rotary_operator():
    """Scaling alone stays on the projection's tables; the same layer by the operator gives the same logits."""
    kw = dict(rope_scaling="yarn", rope_scaling_factor=4.0, rope_original_length=16)
    ids = torch.randint(0, 64, (2, 20), generator=torch.Generator().manual_seed(0))
    a = GPT(_tiny(**kw), device="cpu")
    b = GPT(_tiny(**kw), device="cpu")
    for block in b.blocks:
        block.attn.rotary_op = True
    torch.testing.assert_close(a(ids)[0], b(ids)[0], rtol=1e-4, atol=1e-5)
    assert not torch.allclose(a(ids)[0], GPT(_tiny(), device="cpu")(ids)[0], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("kw", [dict(attn_window=5, attn_sinks=2), dict(qk_norm=True), dict(rope_layout="interleaved", rope_fraction=0.5),
                                dict(attn_window=3, qk_norm=True, rope_layout="interleaved", rope_scaling="linear", rope_scaling_factor=2.0)])
def test_model_gradients_against_differences(kw):
    """Along the gradient itself the directional derivative is its length. Central differences over a hundredth, of a loss of size 4 that
    fp32 rounds by 1e-6, are off by 1e-4 from that, and by the third derivative."""
    m = GPT(_tiny(**kw), device="cpu")
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(0.3 * _randn(*p.shape, seed=p.numel()) + (1 if p.dim() == 1 else 0))
    ids = torch.randint(0, 64, (2, 21), generator=torch.Generator().manual_seed(1))
    loss = lambda: m(ids[:, :-1], ids[:, 1:])[1]  # noqa: E731
    m.zero_grad_buffers()
    loss().backward()
    names = [n for n, _ in m.named_parameters()]
    assert any("q_norm" in n for n in names) == bool(kw.get("qk_norm"))
    for part in ("attn", ""):
        ps = [p for n, p in m.named_parameters() if part in n]
        g = [p.main_grad.clone() for p in ps]
        norm = math.sqrt(sum(float(t.pow(2).sum()) for t in g))
        assert all(t.abs().max() > 0 for t in g)
        with torch.no_grad():
            h, vals = 1e-2 / norm, []
            for sign in (1, -2):
                for p, t in zip(ps, g):
                    p.add_(t, alpha=sign * h)
                vals.append(float(loss()))
            for p, t in zip(ps, g):
                p.add_(t, alpha=h)
        assert abs((vals[0] - vals[1]) / (2 * h) / norm ** 2 - 1) < 0.02


@pytest.mark.parametrize("kw", [dict(qk_norm=True), dict(attn_window=4, qk_norm=True, tied_lm_head=False), dict(rope_fraction=0.5)])
def test_exact_number_of_parameters(kw):
    from train_large_model_from_scratch_b200.utils.model import count_exact_params
    cfg = _tiny(**kw)
    assert count_exact_params(cfg) == sum(p.numel() for p in GPT(cfg, device="cpu").parameters())


def test_flop_count_of_a_window():
    full, part = (GPT(_tiny(attn_window=w), device="cpu").get_exact_flops_per_fwd_bwd(1, 32) for w in (0, 4))
    assert part < full


@pytest.mark.parametrize("T,W,S", [(32, 4, 0), (32, 4, 3), (32, 4, 14), (32, 4, 28), (32, 4, 1000), (32, 1, 31), (32, 31, 1), (32, 32, 5), (31, 7, 11)])
def test_flop_count_is_that_of_the_visible_pairs(T, W, S):
    """Attention's part: 14 multiplications and additions for each pair, head and element; a triangle of n rows counts as n^2 / 2 pairs, as in
    the causal form: W / 2 for the window's, one of S for the sinks'."""
    count = lambda **kw: GPT(_tiny(**kw), device="cpu").get_exact_flops_per_fwd_bwd(1, T)  # noqa: E731
    layers, hidden = 2, 32
    causal, pairs = T * T / 2, int(oracle.window_mask(T, W, S).sum())
    got = (count(attn_window=W, attn_sinks=S) - count()) / (14 * layers * hidden) + causal
    assert abs(got - pairs) <= (min(W, T) + min(S, T - W)) / 2 + 1e-6, (got, pairs)


def test_ranks_of_a_sequence_group_agree():
    """sep = 2 (heads and sequence exchanged) against one rank, all options on: same losses and gradient norms."""
    tmp = tempfile.mkdtemp(prefix="tlm_test_")
    try:
        flags = TINY + ["--log_dir", tmp, "--total_batch_size", "512", "--debug", "--batch_size", "4", "--use_distributed_optimizer", "--rope_variant", "standard",
                        "--attn_window", "7", "--attn_sinks", "2", "--qk_norm", "--rope_layout", "interleaved", "--rope_fraction", "0.5"]
        a = run_trainer(1, flags + ["--sep_size", "1"])
        b = run_trainer(2, flags + ["--sep_size", "2"])
        assert len(a["losses"]) == len(b["losses"]) > 0
        for key in ("losses", "norms"):
            for step in a[key]:
                assert abs(a[key][step] - b[key][step]) <= 2e-4 * max(1.0, abs(a[key][step])), (key, step)
    finally:
        shutil.rmtree(tmp, ignore_errors=True)


def test_a_step_that_exchanges_heads_through_the_library_is_not_recorded():
    from types import SimpleNamespace
    from train_large_model_from_scratch_b200.training import Trainer

    def eligible(sp, **model):
        cfg = build_config(parse_args(["--rope_variant", "standard"] + [f for k, v in model.items() for f in (f"--{k}", str(v))]))
        return Trainer._graph_eligible(SimpleNamespace(_graph_disabled=False, use_cuda=True, config=cfg, world_size=2, _symm=True, sp_world_size=sp,
                                                       _compute_dtype=lambda p: torch.bfloat16))

    assert eligible(2) and eligible(1, attn_window=8) and eligible(1, rope_fraction=0.5)
    assert not eligible(2, attn_window=8) and not eligible(2, rope_fraction=0.5)
