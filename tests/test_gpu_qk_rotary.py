"""Rotary positions and norms of queries and keys on the GPU, against the definition in 64 bits. Outputs are rounded once (half a bf16
step, 2^-8 of the value); the 32-bit arithmetic before it is off by a few 2^-24 of a row's largest terms (2^-18 is allowed), sums
for the weights by 2^-24 for each of the at most 64 additions in a row that a partial sum goes through (2^-17 of the absolute sum)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -8


def _turn(x, positions, inv_freq, interleaved, scale, inverse=False):
    r = 2 * inv_freq.numel()
    angle = (positions.double()[..., None] * inv_freq).reshape(-1, x.shape[1], 1, r // 2)
    turn = torch.polar(torch.full_like(angle, scale), -angle if inverse else angle)
    out = x.double().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(out[..., a], out[..., b]) * turn
    out[..., a], out[..., b] = z.real, z.imag
    return out


def _close(got, want, terms, rel=H):
    """`terms`: size of what is added up for each row."""
    over = (got.double() - want).abs() - 1.01 * rel * want.abs() - 2.0 ** -18 * terms
    assert torch.isfinite(got).all() and over.max().item() <= 0, (over.max().item(), (got.double() - want).abs().max().item())


def _rowmax(t):
    return t.abs().amax(-1, keepdim=True)


def _case(B, T, heads, d, r, per_batch, first=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, heads + 2, d, generator=gen, device="cuda").bfloat16()
    dy = torch.randn(B, T, heads, d, generator=gen, device="cuda").bfloat16()
    pos = torch.arange(first, first + T, device="cuda")
    if per_batch:
        pos = pos + torch.randint(-50, 5000, (B, 1), generator=gen, device="cuda")
    w = [(1 + 0.5 * torch.randn(d, generator=gen, device="cuda")).bfloat16() for _ in range(2)]
    return x[:, :, :heads], dy, pos, 10000.0 ** (-torch.arange(r // 2, device="cuda", dtype=torch.float64) * 2 / r), w


CASES = [(1, 1, 1, 64, 64, False), (16, 1, 24, 64, 64, True), (2, 5, 3, 32, 32, False), (3, 33, 12, 64, 32, True), (1, 100, 5, 128, 128, False),
         (2, 17, 6, 128, 32, False), (1, 40, 20, 256, 256, False), (2, 9, 7, 96, 96, True), (1, 7, 3, 80, 40, False), (1, 7, 4, 48, 22, True),
         (2, 3, 2, 2, 2, False), (1, 11, 40, 16, 16, False), (1, 9, 2, 130, 64, False), (1, 1500, 4, 64, 64, False)]


@pytest.mark.parametrize("B,T,heads,d,r,per_batch", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(B, T, heads, d, r, per_batch, interleaved):
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, dy, pos, freq, _ = _case(B, T, heads, d, r, per_batch)
    leaf = x.detach().requires_grad_()
    y = F_ops.rotary(leaf, pos, freq, interleaved=interleaved, scale=1.25)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    _close(y.detach(), _turn(x, pos, freq, interleaved, 1.25), 2.5 * _rowmax(x.double()))
    _close(dx, _turn(dy, pos, freq, interleaved, 1.25, inverse=True), 2.5 * _rowmax(dy.double()))


@pytest.mark.parametrize("B,T,heads,d,r,per_batch", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_and_rotary(B, T, heads, d, r, per_batch, interleaved):
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, dy, pos, freq, w = _case(B, T, heads, d, r, per_batch, seed=1)
    n_q = heads - heads // 3
    leaf, params = x.detach().requires_grad_(), [torch.nn.Parameter(t) for t in w]
    y = F_ops.qk_norm_rotary(leaf, n_q, *params, pos, freq, eps=1e-5, interleaved=interleaved)
    for p in params:
        p.main_grad = torch.full((d,), 3.0, device="cuda")
    (dx,) = torch.autograd.grad(y, leaf, dy)
    is_q = (torch.arange(heads, device="cuda") < n_q)[:, None]
    wt = torch.where(is_q, w[0].double(), w[1].double())
    rstd = (x.double().pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = x.double() * rstd
    _close(y.detach(), _turn(hat * wt, pos, freq, interleaved, 1.0), 4 * _rowmax(hat * wt))
    du = _turn(dy, pos, freq, interleaved, 1.0, inverse=True)
    g = du * wt
    dot = (g * hat).mean(-1, keepdim=True)
    _close(dx, rstd * (g - hat * dot), rstd * 4 * (_rowmax(g) + _rowmax(hat) * (g * hat).abs().mean(-1, keepdim=True)))
    for p, heads_of in zip(params, (slice(0, n_q), slice(n_q, None))):
        terms = (du * hat)[:, :, heads_of]
        assert ((p.main_grad.double() - 3.0 - terms.sum((0, 1, 2))).abs() <= 2.0 ** -17 * (3.0 + terms.abs().sum((0, 1, 2)))).all()


@pytest.mark.parametrize("B,T,heads,d", [(1, 1, 1, 64), (1, 7, 12, 64), (2, 5, 3, 32), (1, 33, 5, 128), (3, 3, 7, 96), (1, 3, 2, 22), (1, 700, 5, 256)])
@pytest.mark.parametrize("eps", [0.0, 1e-60])
def test_an_eps_of_zero(B, T, heads, d, eps):
    """... or one that is zero in 32 bits: places of a block that have no row add nothing to the weights' gradients."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, dy, pos, freq, w = _case(B, T, heads, d, d, False, seed=6)
    n_q = heads - heads // 3
    leaf, params = x.detach().requires_grad_(), [torch.nn.Parameter(t) for t in w]
    y = F_ops.qk_norm_rotary(leaf, n_q, *params, pos, freq, eps=eps)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    is_q = (torch.arange(heads, device="cuda") < n_q)[:, None]
    wt = torch.where(is_q, w[0].double(), w[1].double())
    rstd = x.double().pow(2).mean(-1, keepdim=True).rsqrt()
    hat = x.double() * rstd
    _close(y.detach(), _turn(hat * wt, pos, freq, False, 1.0), 4 * _rowmax(hat * wt))
    du = _turn(dy, pos, freq, False, 1.0, inverse=True)
    g = du * wt
    _close(dx, rstd * (g - hat * (g * hat).mean(-1, keepdim=True)), rstd * 4 * (_rowmax(g) + _rowmax(hat) * (g * hat).abs().mean(-1, keepdim=True)))
    for p, heads_of in zip(params, (slice(0, n_q), slice(n_q, None))):
        # du is a difference of two products of dy, each off by a few 2^-24 of its own size
        terms, size = (du * hat)[:, :, heads_of], (2 * _rowmax(dy.double()) * hat.abs())[:, :, heads_of]
        assert ((p.main_grad.double() - terms.sum((0, 1, 2))).abs() <= 2.0 ** -17 * terms.abs().sum((0, 1, 2)) + 2.0 ** -20 * size.sum((0, 1, 2))).all()


def test_far_positions_keep_their_angle():
    """Around 2^32 a 32-bit angle would say nothing."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, _, pos, freq, _ = _case(1, 64, 2, 64, 64, False, first=1 << 32)
    pos = torch.cat([pos[:32], -pos[32:]])
    # 64-bit angles around 2^32 are themselves off by 2^-21
    _close(F_ops.rotary(x, pos, freq), _turn(x, pos, freq, False, 1.0), 16 * _rowmax(x.double()))


def test_layouts_and_the_same_weight_twice():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, dy, pos, freq, w = _case(2, 50, 4, 64, 64, False, seed=2)
    base = None
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
    for view in (x, x.contiguous(), x.transpose(1, 2).contiguous().transpose(1, 2), odd, torch.nn.functional.pad(x, (0, 1))[..., :64],
                 x.transpose(2, 3).contiguous().transpose(2, 3)):
        leaf, p = view.detach().requires_grad_(), torch.nn.Parameter(w[0])
        y = F_ops.qk_norm_rotary(leaf, 3, p, p, pos, freq)
        (dx,) = torch.autograd.grad(y, leaf, dy.transpose(1, 2).contiguous().transpose(1, 2))
        got = (y.detach(), dx, p.main_grad)
        base = base or got
        assert torch.equal(got[0], base[0])
        # the element-by-element form adds a row up in the same lanes, but may contract differently: one rounding of the result
        assert ((got[1].float() - base[1].float()).abs() <= 2 * H * base[1].float().abs() + 1e-6).all()
        torch.testing.assert_close(got[2], base[2], rtol=1e-5, atol=1e-4)


def test_a_row_of_zeros_and_large_rows():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, dy, pos, freq, w = _case(1, 8, 2, 64, 64, False, seed=3)
    x = x.clone()
    x[:, 0] = 0
    x[:, 1] *= 2.0 ** 60
    x[:, 2] *= 2.0 ** -60
    leaf = x.requires_grad_()
    y = F_ops.qk_norm_rotary(leaf, 1, *[torch.nn.Parameter(t) for t in w], pos, freq)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert torch.isfinite(y).all() and torch.isfinite(dx).all() and (y[:, 0] == 0).all()


def test_deterministic_and_captured():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    sets = [_case(2, 700, 12, 64, 64, True, seed=s) for s in (4, 5)]
    want = []
    for x, dy, pos, freq, w in sets:
        for _ in range(2):
            leaf, params = x.detach().requires_grad_(), [torch.nn.Parameter(t) for t in w]
            y = F_ops.qk_norm_rotary(leaf, 8, *params, pos, freq)
            (dx,) = torch.autograd.grad(y, leaf, dy)
            got = (y.detach(), dx, params[0].main_grad, params[1].main_grad)
        want.append(got)
        first = F_ops.qk_norm_rotary(x, 8, *params, pos, freq)
        assert torch.equal(first, got[0])
    x, dy, pos, freq, w = [t.clone() if torch.is_tensor(t) else t for t in sets[0]]
    leaf, params = x.detach().requires_grad_(), [torch.nn.Parameter(t.clone()) for t in w]
    for p in params:
        p.main_grad = torch.zeros(64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(F_ops.qk_norm_rotary(leaf, 8, *params, pos, freq), leaf, dy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for p in params:
            p.main_grad.zero_()
        y = F_ops.qk_norm_rotary(leaf, 8, *params, pos, freq)
        (dx,) = torch.autograd.grad(y, leaf, dy)
    for s in (1, 0, 1):
        with torch.no_grad():
            for dst, src in zip((leaf, dy, pos, *params), (*sets[s][:3], *sets[s][4])):
                dst.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((y.detach(), dx, params[0].main_grad, params[1].main_grad), want[s]):
            assert torch.equal(a, b)


def test_refusals():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    x, _, pos, freq, w = _case(2, 8, 4, 64, 64, False)
    with pytest.raises(ValueError, match="different devices"):
        F_ops.rotary(x, pos.cpu(), freq)
    with pytest.raises(ValueError, match="weights"):
        F_ops.qk_norm_rotary(x, 2, w[0].float(), w[1], pos, freq)
    assert F_ops.rotary(x[:, :0], pos[:0], freq).shape == (2, 0, 4, 64)


def test_offsets_beyond_32_bits():
    """The last rows of a tensor of more than 2^31 elements, as they come out alone."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    T, heads, d, n = 140032, 120, 128, 40
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, T, heads, d, generator=gen, device="cuda").bfloat16()
    pos, freq = torch.arange(T, device="cuda"), 10000.0 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
    w = [(1 + 0.5 * torch.randn(d, generator=gen, device="cuda")).bfloat16() for _ in range(2)]
    for leaf_w in w:
        leaf_w.main_grad = torch.zeros(d, device="cuda")

    def run(x, pos):
        x = x.detach().requires_grad_()
        y = F_ops.qk_norm_rotary(x, 96, *w, pos, freq)
        (dx,) = torch.autograd.grad(y, x, x.detach())
        return y.detach()[:, -n:].clone(), dx[:, -n:].clone(), F_ops.rotary(x.detach(), pos, freq)[:, -n:].clone()

    got, want = run(x, pos), run(x[:, -n:].contiguous(), pos[-n:])
    native.raise_on_device_status()
    assert x.numel() > 2 ** 31
    for a, b in zip(got, want):
        assert torch.equal(a, b)
