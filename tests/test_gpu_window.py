"""Window attention with sinks on the GPU, against the definition in 64 bits. Tolerances are sums of the roundings that the kernels
make on purpose: bf16 probabilities and dS (half a step each, 2^-8 of the value), outputs rounded once (2^-8), the row term
delta = sum do * o from the rounded o; everything else is 32 bits and covered by a factor of 1.05 and 1e-5 of the largest."""
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -8


def _reference(q, k, v, do, window, sinks):
    """o, dq, dk, dv in 64 bits, each with the bound on its error."""
    from train_large_model_from_scratch_b200.ops import oracle
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, do))
    n_kv, rep, T, d = k.shape[1], q.shape[1] // k.shape[1], q.shape[2], q.shape[3]
    k, v = (t.repeat_interleave(rep, dim=1) for t in (k, v))
    seen = oracle.window_mask(T, window, sinks, q.device)
    p = torch.softmax((q @ k.mT / math.sqrt(d)).masked_fill(~seen, -math.inf), dim=-1)
    o = p @ v
    eo = H * (p @ v.abs() + o.abs())
    if min(T, (window or T) + sinks) < 128:
        # divided by the sum of the rounded probabilities: sum p (1 + e_j) v_j / sum p (1 + e_j) = o + sum p e_j (v_j - o) + O(e^2), |e_j| <= H,
        # and |v_j - o| <= |v_j| + |o|
        eo = eo + H * o.abs()
    dp = do @ v.mT
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    eds = H * ds.abs() + p * (do.abs() * eo).sum(-1, keepdim=True)
    shared = lambda t: t.unflatten(1, (n_kv, rep)).sum(2)  # noqa: E731
    dq, edq = ds @ k / math.sqrt(d), eds @ k.abs() / math.sqrt(d)
    dk, edk = (shared(a.mT @ b / math.sqrt(d)) for a, b in ((ds, q), (eds, q.abs())))
    dv, edv = (shared(a.mT @ b) for a, b in ((p, do), (H * p, do.abs())))
    out = [(o, eo)] + [(t, e + H * t.abs()) for t, e in ((dq, edq), (dk, edk), (dv, edv))]
    return [(t.transpose(1, 2), e.transpose(1, 2)) for t, e in out]


def _check(got, want, what):
    for name, g, (t, e) in zip(("o", "dq", "dk", "dv"), got, want):
        assert g.shape == t.shape
        over = (g.double() - t).abs() - 1.05 * e - 1e-5 * t.abs().max() - 1e-30
        assert torch.isfinite(g).all() and over.max().item() <= 0, (what, name, over.max().item(), (g.double() - t).abs().max().item())


def _poison(elements):
    """Memory that the allocator hands out next holds NaN."""
    t = torch.full((elements,), float("nan"), device="cuda")
    del t


def _inputs(B, T, n_q, n_kv, d, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, T, n_q + 2 * n_kv, d, generator=gen, device="cuda").bfloat16(),
            torch.randn(B, T, n_q, d, generator=gen, device="cuda").bfloat16())


def _run_packed(qkv, do, n_q, n_kv, window, sinks):
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    x = qkv.detach().requires_grad_()
    _poison(qkv.numel() * 4)
    o = F_ops.attention_packed(x, n_q, n_kv, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, x, do)
    native.raise_on_device_status()
    return [o.detach(), *g.split([n_q, n_kv, n_kv], dim=2)]


SHAPES = [(1, 1, 2, 1, 64), (3, 1, 4, 4, 32), (2, 2, 2, 2, 128), (1, 127, 4, 2, 64), (2, 128, 2, 1, 32), (1, 129, 3, 1, 128),
          (1, 257, 4, 4, 64), (2, 320, 8, 2, 32), (1, 640, 6, 2, 64), (1, 700, 4, 1, 128)]


@pytest.mark.parametrize("B,T,n_q,n_kv,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (64, 4), (127, 0), (128, 1), (129, 130), (300, 7), (100000, 4), (5, 100000)])
def test_against_the_definition(B, T, n_q, n_kv, d, window, sinks):
    qkv, do = _inputs(B, T, n_q, n_kv, d)
    got = _run_packed(qkv, do, n_q, n_kv, window, sinks)
    _check(got, _reference(*qkv.split([n_q, n_kv, n_kv], dim=2), do, window, sinks), (window, sinks))


@pytest.mark.parametrize("split", ["1", "2", "4", "8"])
@pytest.mark.parametrize("T,n_q,n_kv,d,window,sinks", [(1500, 4, 2, 64, 100, 4), (1500, 2, 2, 128, 256, 200), (1400, 4, 1, 32, 1, 20), (2100, 2, 1, 64, 130, 1)])
def test_blocks_that_share_a_tile(split, T, n_q, n_kv, d, window, sinks, monkeypatch):
    monkeypatch.setenv("TLM_ATTN_BWD_SPLIT", split)
    qkv, do = _inputs(1, T, n_q, n_kv, d, seed=1)
    got = _run_packed(qkv, do, n_q, n_kv, window, sinks)
    _check(got, _reference(*qkv.split([n_q, n_kv, n_kv], dim=2), do, window, sinks), split)


def _layouts(q, k, v):
    yield "contiguous", [t.contiguous() for t in (q, k, v)]
    yield "heads before tokens", [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    yield "one token's rows apart", [torch.cat([t, t], dim=2)[:, :, :t.shape[2]] for t in (q, k, v)]
    yield "every second head", [torch.stack([t, t], dim=3).flatten(2, 3)[:, :, ::2] for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        odd.append(flat[1:].view(t.shape).copy_(t))
    yield "addresses that are no multiples of 16 bytes", odd
    yield "rows that are no whole pieces apart", [torch.nn.functional.pad(t, (0, 3))[..., :t.shape[3]] for t in (q, k, v)]


def test_layouts():
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    qkv, do = _inputs(2, 200, 4, 2, 64, seed=2)
    q, k, v = qkv.split([4, 2, 2], dim=2)
    want = _reference(q, k, v, do, 70, 3)
    for name, views in _layouts(q, k, v):
        leaves = [t.detach().requires_grad_() for t in views]
        o = F_ops.window_attention(*leaves, window=70, sinks=3)
        for g in (do, do.transpose(1, 2).contiguous().transpose(1, 2)):
            got = [o.detach(), *torch.autograd.grad(o, leaves, g, retain_graph=True)]
            native.raise_on_device_status()
            _check(got, want, name)


def test_broadcast_keys_and_values():
    """One KV head for all batch entries: the gradient that autograd sums is that of every entry."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    qkv, do = _inputs(3, 150, 2, 1, 64, seed=3)
    q, k, v = qkv.split([2, 1, 1], dim=2)
    k1, v1 = (t[:1].detach().requires_grad_() for t in (k, v))
    o = F_ops.window_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), window=20, sinks=2)
    dk, dv = torch.autograd.grad(o, [k1, v1], do)
    want = _reference(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), do, 20, 2)
    for g, (t, e) in ((dk, want[2]), (dv, want[3])):
        t, e = t.sum(0, keepdim=True), e.sum(0, keepdim=True) * 1.05
        assert ((g.double() - t).abs() <= e + 3 * H * t.abs() + 1e-5 * t.abs().max()).all()


def test_without_a_window_it_is_the_causal_operator():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    qkv, do = _inputs(2, 300, 4, 2, 64, seed=4)
    q, k, v = qkv.split([4, 2, 2], dim=2)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = F_ops.window_attention(*leaves)
    _check([o.detach(), *torch.autograd.grad(o, leaves, do)], _reference(q, k, v, do, 0, 0), "no window")


@pytest.mark.parametrize("d,variant", [(32, "standard"), (64, "reference"), (128, "standard")])
def test_transposed_rotation_on_the_way_out(d, variant):
    """`rope`: dQ and dK leave as gradients of the un-rotated heads, the sink rows of dK among them."""
    from train_large_model_from_scratch_b200.ops import attention_cuda, native, oracle
    T, n_q, n_kv = 1500, 2, 1
    qkv, do = _inputs(1, T, n_q, n_kv, d, seed=5)
    q, k, v = qkv.split([n_q, n_kv, n_kv], dim=2)
    cos, sin = oracle.rope_tables(torch.arange(T, device="cuda"), d, 10000.0, variant)
    o, lse, rest = attention_cuda.window_fwd(q, k, v, 100, 5, rest=True)
    plain, turned = ([torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)] for _ in range(2))
    attention_cuda.window_bwd(do, q, k, v, o, lse, rest, 100, 5, plain)
    attention_cuda.window_bwd(do, q, k, v, o, lse, rest, 100, 5, turned, rope=(cos, sin))
    native.raise_on_device_status()
    assert torch.equal(plain[2], turned[2])
    for a, b in zip(plain[:2], turned[:2]):
        want = oracle.rope_bwd(a, cos, sin)
        pair = a.float().abs() + oracle.rotate_half(a.float()).abs()
        # a was rounded too, dQ's sums come in another order each time
        assert ((b.float() - want).abs() <= H * want.abs() + 2 * H * pair + 1e-4 * pair.max()).all()


def test_hidden_keys_may_hold_anything_finite():
    """The largest finite values in hidden keys: their weight is zero, not small."""
    qkv, do = _inputs(1, 600, 2, 1, 64, seed=6)
    n_q, n_kv = 2, 1
    base = _run_packed(qkv, do, n_q, n_kv, 40, 2)
    bad = qkv.clone()
    bad[:, 300:301, n_q:n_q + 1] *= 1e30                      # visible to rows 300 .. 339 only
    bad[:, 300:301, n_q + 1:] = 3e38
    got = _run_packed(bad, do, n_q, n_kv, 40, 2)
    for rows in (slice(0, 300), slice(340, 600)):
        assert torch.equal(got[0][:, rows], base[0][:, rows])


@pytest.mark.parametrize("split", ["1", "2"])
@pytest.mark.parametrize("at,window,sinks", [(300, 40, 2), (1, 40, 1), (599, 40, 0), (300, 1000, 0), (130, 140, 130)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradients_beside_a_hidden_value_of_any_size(d, at, window, sinks, split, monkeypatch):
    """do * v of a hidden key may overflow: neither the gradients of the queries that do not see it, nor those of the keys that none
    of its queries sees, know of it. dq is reduced in hardware order: one rounding to either side."""
    from train_large_model_from_scratch_b200.ops import oracle
    monkeypatch.setenv("TLM_ATTN_BWD_SPLIT", split)
    n_q, n_kv, T = 2, 1, 600
    qkv, do = _inputs(1, T, n_q, n_kv, d, seed=11)
    base = _run_packed(qkv, do, n_q, n_kv, window, sinks)
    bad = qkv.clone()
    bad[:, at, n_q + 1] = 3e38
    got = _run_packed(bad, do, n_q, n_kv, window, sinks)
    seen = oracle.window_mask(T, window, sinks, "cuda")
    rows = ~seen[:, at]
    keys = ~seen[~rows].any(0)
    assert torch.equal(got[0][:, rows], base[0][:, rows])
    if rows.any():
        a, b = got[1][:, rows].float(), base[1][:, rows].float()
        assert ((a - b).abs() <= 2 * H * b.abs() + 1e-5 * base[1].abs().max()).all()
    for a, b in zip(got[2:], base[2:]):
        assert torch.equal(a[:, keys], b[:, keys])


@pytest.mark.parametrize("d", [32, 64, 128])
def test_a_key_of_nan_reaches_the_rows_that_see_it(d):
    """... and no others: a hidden score is hidden whatever it is."""
    n_q, n_kv, window, sinks = 2, 1, 40, 3
    qkv, do = _inputs(1, 400, n_q, n_kv, d, seed=10)
    base = _run_packed(qkv, do, n_q, n_kv, window, sinks)[0]
    for at in (1, 130, 131, 135, 139, 250, 399):
        bad = qkv.clone()
        bad[:, at, n_q] = float("nan")
        from train_large_model_from_scratch_b200.ops import functional as F_ops
        with torch.no_grad():
            o = F_ops.attention_packed(bad, n_q, n_kv, window=window, sinks=sinks)
        row = torch.arange(400, device="cuda")
        sees = (row >= at) & ((row - at < window) | (at < sinks))
        assert torch.isnan(o[:, sees]).all() and torch.equal(o[:, ~sees], base[:, ~sees]), at


@pytest.mark.parametrize("T,window,sinks", [(2, 9, 0), (3, 9, 0), (4, 2, 1), (300, 2, 0), (300, 1, 1), (129, 3, 4)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_rows_with_few_keys_keep_their_gradients(T, window, sinks, d):
    """Where a row sees a few keys only, delta and do * v nearly cancel, and an error of delta relative to its own size would be much of the
    gradients of q and k (with delta from a rounded o, 0.4 of them in one of 200 random cases of two keys). delta is a weighted mean
    of the row's do * v, so what is left are three roundings relative to the result: the weights of that mean, dS, the result itself,
    half a bf16 step each."""
    worst = 0.0
    for seed in range(6):
        qkv, do = _inputs(2, T, 16, 8, d, seed=20 + seed)
        got = _run_packed(qkv, do, 16, 8, window, sinks)
        want = _reference(*qkv.split([16, 8, 8], dim=2), do, window, sinks)
        for g, (t, _) in zip(got[1:3], want[1:3]):
            worst = max(worst, ((g.double() - t).norm() / t.norm()).item())
    assert worst <= 3 * H, worst


@pytest.mark.parametrize("T,window,sinks", [(128, 1000, 0), (129, 128, 0), (300, 1000, 0), (300, 200, 4), (260, 100, 60), (700, 1, 127)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_the_first_rows_of_a_long_window_keep_their_gradients(T, window, sinks, d):
    """A sequence's first rows see few keys whatever the window. Row by row, dS = p (dp - delta): delta is a weighted mean of dp whose
    weights are off by half a bf16 step each, so off by at most that of sum p |dp - delta|; dS and dq are rounded once; o in delta is
    held to 2^-17, sums of products to 2^-18 of their terms."""
    qkv, do = _inputs(2, T, 16, 8, d, seed=40)
    got = _run_packed(qkv, do, 16, 8, window, sinks)
    from train_large_model_from_scratch_b200.ops import oracle
    q, k, v = (t.double().transpose(1, 2) for t in qkv.split([16, 8, 8], dim=2))
    do = do.double().transpose(1, 2)
    k, v = (t.repeat_interleave(2, dim=1) for t in (k, v))
    seen = oracle.window_mask(T, window, sinks, "cuda")
    p = torch.softmax((q @ k.mT / math.sqrt(d)).masked_fill(~seen, -math.inf), dim=-1)
    dp = do @ v.mT
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_delta = H * ds.abs().sum(-1, keepdim=True) + 2.0 ** -16 * (do.abs() * (p @ v.abs())).sum(-1, keepdim=True)
    e_ds = 1.05 * H * ds.abs() + p * (1.05 * e_delta + 2.0 ** -18 * (do.abs() @ v.abs().mT))
    dq, e = ds @ k / math.sqrt(d), e_ds @ k.abs() / math.sqrt(d)
    over = (got[1].double().transpose(1, 2) - dq).abs() - e - H * (dq.abs() + e)
    assert over[:, :, :128].max().item() <= 0, [(i, over[:, :, i].max().item()) for i in range(128) if over[:, :, i].max().item() > 0][:5]


def test_same_bits_again_and_in_a_graph():
    """o, dk and dv do not depend on the order in which blocks run (dq is reduced in hardware order); a captured call replays on
    new inputs, beside another captured call and eager ones on another stream."""
    n_q, n_kv, window, sinks = 4, 2, 100, 3
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    sets = [_inputs(1, 1500, n_q, n_kv, 64, seed=s) for s in (7, 8)]
    want = [_run_packed(*s, n_q, n_kv, window, sinks) for s in sets]
    again = _run_packed(*sets[0], n_q, n_kv, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip([want[0][i] for i in (0, 2, 3)], [again[i] for i in (0, 2, 3)]))
    x = [sets[0][0].clone().requires_grad_() for _ in range(2)]
    do = [sets[0][1].clone() for _ in range(2)]
    outs, graphs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):                                        # warm-up off the capture
            o = F_ops.attention_packed(x[i], n_q, n_kv, window=window, sinks=sinks)
            torch.autograd.grad(o, x[i], do[i])
    torch.cuda.current_stream().wait_stream(side)
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = F_ops.attention_packed(x[i], n_q, n_kv, window=window, sinks=sinks)
            outs.append((o, torch.autograd.grad(o, x[i], do[i])[0]))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for i, s in zip(range(2), order):
            with torch.no_grad():
                x[i].copy_(sets[s][0])
                do[i].copy_(sets[s][1])
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            eager = _run_packed(*sets[1], n_q, n_kv, window, sinks)
        graphs[1].replay()
        torch.cuda.synchronize()
        native.raise_on_device_status()
        assert torch.equal(eager[0], want[1][0])
        for i, s in zip(range(2), order):
            o, dx = outs[i]
            assert torch.equal(o.detach(), want[s][0])
            dq, dk, dv = dx.split([n_q, n_kv, n_kv], dim=2)
            assert torch.equal(dk, want[s][2]) and torch.equal(dv, want[s][3])
            assert ((dq.float() - want[s][1].float()).abs() <= 2 * H * dq.float().abs() + 1e-5 * dq.abs().max()).all()


def test_first_call_of_a_thread():
    """Tensor maps are made through the driver, which a thread's first CUDA call has to have prepared."""
    import threading
    got = []
    x = torch.zeros(1, 77, 4, 64, device="cuda", dtype=torch.bfloat16)

    def call():
        from train_large_model_from_scratch_b200.ops import attention_cuda
        got.append(attention_cuda.window_fwd(x[:, :, :2], x[:, :, 2:3], x[:, :, 3:], 11, 1)[0])

    t = threading.Thread(target=call)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and (got[0] == 0).all()


def test_gradients_against_differences():
    """The gradient of sum(o * do) along a random direction, against central differences of the definition."""
    from train_large_model_from_scratch_b200.ops import oracle
    n_q, n_kv, d, window, sinks = 2, 1, 32, 30, 3
    qkv, do = _inputs(1, 200, n_q, n_kv, d, seed=9)
    got = torch.cat(_run_packed(qkv, do, n_q, n_kv, window, sinks)[1:], dim=2).double()

    def f(x):
        q, k, v = (t.transpose(1, 2) for t in x.split([n_q, n_kv, n_kv], dim=2))
        k, v = (t.repeat_interleave(n_q // n_kv, dim=1) for t in (k, v))
        s = (q @ k.mT / math.sqrt(d)).masked_fill(~oracle.window_mask(200, window, sinks, x.device), -math.inf)
        return ((torch.softmax(s, -1) @ v).transpose(1, 2) * do.double()).sum().item()

    gen = torch.Generator(device="cuda").manual_seed(1)
    want = _reference(*qkv.split([n_q, n_kv, n_kv], dim=2), do, window, sinks)
    err = torch.cat([e for _, e in want[1:]], dim=2)
    for _ in range(4):
        u = torch.randn(qkv.shape, generator=gen, device="cuda", dtype=torch.float64)
        diff = (f(qkv.double() + 1e-4 * u) - f(qkv.double() - 1e-4 * u)) / 2e-4
        assert abs((got * u).sum().item() - diff) <= 1.05 * (err * u.abs()).sum().item()


def test_refusals():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    qkv, _ = _inputs(1, 10, 2, 1, 48)
    with pytest.raises(ValueError, match="head dim 48"):
        F_ops.attention_packed(qkv, 2, 1, window=4)
    q, k, v = _inputs(1, 10, 2, 1, 64)[0].split([2, 1, 1], dim=2)
    with pytest.raises(ValueError, match="different devices"):
        F_ops.window_attention(q, k.cpu(), v, window=4)
    empty = F_ops.window_attention(q[:, :0], k[:, :0], v[:, :0], window=4)
    assert empty.shape == (1, 0, 2, 64)


def test_offsets_beyond_32_bits():
    """The last rows of a tensor of more than 2^31 elements: as those of its end alone, which no earlier key reaches. Probabilities, dS
    and each output row's terms are the same; sums in another order may round to the other side: one bf16 step."""
    T, n, n_q, n_kv, d, window = 140032, 512, 104, 8, 128, 100
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    qkv, do = _inputs(1, T, n_q, n_kv, d)
    want = _run_packed(qkv[:, -n:].contiguous(), do[:, -n:].contiguous(), n_q, n_kv, window, 0)
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    o = F_ops.attention_packed(qkv.requires_grad_(), n_q, n_kv, window=window)
    (g,) = torch.autograd.grad(o, qkv, do)
    native.raise_on_device_status()
    assert qkv.numel() > 2 ** 31 and g.shape == qkv.shape
    for name, a, b in zip(("o", "dq", "dk", "dv"), (o.detach(), *g.split([n_q, n_kv, n_kv], dim=2)), want):
        a, b = a[:, 128 - n:].double(), b[:, 128:].double()
        assert ((a - b).abs() <= 2 * H * b.abs() + 2.0 ** -18 * b.abs().max()).all(), name
