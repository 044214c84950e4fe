"""The long-context options of the attention layer on the GPU: norms and rotation, window attention and the projection as they run
together, against the same layer in 64 bits, on the torch path, and captured in a graph."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -8

OPTIONS = [dict(attn_window=100, attn_sinks=4), dict(qk_norm=True), dict(rope_layout="interleaved", rope_fraction=0.5),
           dict(attn_window=64, qk_norm=True, rope_fraction=0.25), dict(rope_scaling="yarn", rope_scaling_factor=4.0, rope_original_length=64),
           dict(attn_window=130, attn_sinks=130, qk_norm=True, rope_layout="interleaved", rope_scaling="linear", rope_scaling_factor=2.0)]


def _case(B, T, n_q, n_kv, d, norm, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(B, T, n_q + 2 * n_kv, d, generator=gen, device="cuda").bfloat16()
    do = torch.randn(B, T, n_q, d, generator=gen, device="cuda").bfloat16()
    w = [torch.nn.Parameter((1 + 0.3 * torch.randn(d, generator=gen, device="cuda")).bfloat16()) for _ in range(2)] if norm else None
    return qkv, do, w


def _chain(qkv, weights, n_q, n_kv, pos, freq, interleaved, window, sinks):
    """In 64 bits, for autograd."""
    from train_large_model_from_scratch_b200.ops import oracle
    q, k, v = qkv.split([n_q, n_kv, n_kv], dim=2)
    if weights is not None:
        q, k = (t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w for t, w in zip((q, k), weights))
    r = 2 * freq.numel()
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
        y = [a * cos - b * sin, b * cos + a * sin]
        return torch.cat([torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1), x[..., r:]], -1)

    q, k, v = (t.transpose(1, 2) for t in (turn(q), turn(k), v))
    k, v = (t.repeat_interleave(n_q // n_kv, dim=1) for t in (k, v))
    s = (q @ k.mT / math.sqrt(q.shape[-1])).masked_fill(~oracle.window_mask(q.shape[2], window, sinks, q.device), -math.inf)
    return (torch.softmax(s, -1) @ v).transpose(1, 2)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("norm,interleaved,r_of,window,sinks", [(True, False, 1, 100, 4), (True, True, 2, 0, 0), (False, True, 1, 1, 3), (False, False, 4, 300, 0)])
def test_norm_rotation_and_window_in_a_row(d, norm, interleaved, r_of, window, sinks):
    """Relative to the size of each result: rotated heads, probabilities, dS, o (in delta), dQ / dK between the kernels and the result
    are rounded, half a bf16 step each. A rounding of the heads moves a score by at most 2 * 2^-8 |q| |k| / sqrt(d), which is 2^-7 times the
    spread of the scores here, and through that a result by as much again: nine half steps at most if all of them pointed one way."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    B, T, n_q, n_kv = 2, 500, 4, 2
    qkv, do, w = _case(B, T, n_q, n_kv, d, norm)
    r = d // r_of
    pos, freq = torch.arange(1000, 1000 + T, device="cuda"), 10000.0 ** (-torch.arange(r // 2, device="cuda", dtype=torch.float64) * 2 / r)
    x = qkv.detach().requires_grad_()
    o = F_ops.rotary_attention(x, n_q, n_kv, pos, freq, interleaved=interleaved, norm_weights=w, window=window, sinks=sinks)
    (dx,) = torch.autograd.grad(o, x, do)
    native.raise_on_device_status()
    x64 = qkv.double().requires_grad_()
    w64 = [t.detach().double().requires_grad_() for t in w] if norm else None
    o64 = _chain(x64, w64, n_q, n_kv, pos, freq, interleaved, window, sinks)
    want = torch.autograd.grad(o64, [x64, *(w64 or [])], do.double())
    pairs = [(o, o64.detach())] + list(zip(dx.split([n_q, n_kv, n_kv], 2), want[0].split([n_q, n_kv, n_kv], 2)))
    if window == 1:
        pairs = [pairs[0], pairs[3]]                       # most rows see a key or two: their dQ and dK are differences of equal numbers
    else:
        pairs += list(zip([p.main_grad for p in w or []], want[1:]))
    for got, ref in pairs:
        assert torch.isfinite(got).all()
        assert ((got.double() - ref).norm() / ref.norm()).item() <= 9 * H, (got.shape, ((got.double() - ref).norm() / ref.norm()).item())


def test_one_node_is_the_operators_in_a_row():
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    n_q, n_kv = 4, 2
    qkv, do, w = _case(1, 900, n_q, n_kv, 64, True, seed=1)
    pos, freq = torch.arange(900, device="cuda"), 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
    x = qkv.detach().requires_grad_()
    o = F_ops.rotary_attention(x, n_q, n_kv, pos, freq, norm_weights=w, window=200, sinks=2)
    (dx,) = torch.autograd.grad(o, x, do)
    leaf = qkv.detach().requires_grad_()
    qk, v = leaf.split([n_q + n_kv, n_kv], dim=2)
    qk = F_ops.qk_norm_rotary(qk, n_q, *[torch.nn.Parameter(t.detach().clone()) for t in w], pos, freq)
    o2 = F_ops.window_attention(qk[:, :, :n_q], qk[:, :, n_q:], v, window=200, sinks=2)
    (dx2,) = torch.autograd.grad(o2, leaf, do)
    assert torch.equal(o, o2) and torch.equal(dx[:, :, n_q:], dx2[:, :, n_q:])
    # dQ is reduced in another order each time: another rounding before the norm, whose gradient takes differences of them
    assert ((dx[:, :, :n_q].double() - dx2[:, :, :n_q].double()).norm() <= 4 * H * dx2[:, :, :n_q].double().norm()).item()


def test_a_tangent_is_refused():
    """The kernels know nothing of forward-mode derivatives: a tangent is refused, not dropped; other calls beside it run."""
    import torch.autograd.forward_ad as fwad
    from train_large_model_from_scratch_b200.ops import functional as F_ops
    qkv, _, w = _case(1, 40, 4, 2, 64, True)
    pos, freq = torch.arange(40, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    plain = F_ops.rotary(qkv, pos, freq)
    for call in (lambda x: F_ops.rotary(x, pos, freq), lambda x: F_ops.qk_norm_rotary(x, 4, *[t.detach() for t in w], pos, freq),
                 lambda x: F_ops.attention_packed(x, 4, 2, window=7), lambda x: F_ops.rotary_attention(x, 4, 2, pos, freq, window=7),
                 lambda x: F_ops.window_attention(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], 7)):
        with fwad.dual_level():
            with pytest.raises(RuntimeError, match="jvp"):
                call(fwad.make_dual(qkv, torch.ones_like(qkv)))
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                call(fwad.make_dual(qkv, torch.ones_like(qkv)))
            assert torch.equal(F_ops.rotary(qkv, pos, freq), plain)


def _models(over):
    from train_large_model_from_scratch_b200.models import GPT
    from train_large_model_from_scratch_b200.models.modules.init import clear_init_cache
    from train_large_model_from_scratch_b200.training.config import ModelConfig
    clear_init_cache()
    cfg = ModelConfig(**{**dict(num_layer=2, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512, vocab_size=4096,
                                block_size=512, rope_variant="standard"), **over})
    return GPT(cfg, device="cuda"), GPT(cfg, device="cpu", compute_dtype=torch.float32)


@pytest.mark.parametrize("over", OPTIONS)
@pytest.mark.parametrize("heads", [4, 8, 2])
def test_model_against_the_torch_path(over, heads):
    from train_large_model_from_scratch_b200.ops import native
    gpu, cpu = _models({**over, "num_attention_heads": heads, "num_key_value_heads": heads // 2})
    cpu.dense_buf.params.copy_(gpu.dense_buf.params.float().cpu())
    data = torch.randint(0, 4096, (2, 258), generator=torch.Generator().manual_seed(0))
    x, y = data[:, :-1].contiguous(), data[:, 1:].contiguous()
    _, lg, _ = gpu(x.cuda(), y.cuda())
    lg.backward()
    _, lc, _ = cpu(x, y)
    lc.backward()
    native.raise_on_device_status()
    assert abs(lg.item() - lc.item()) < 2e-2
    gg, gc = gpu.dense_buf.main_grad.cpu(), cpu.dense_buf.main_grad
    for name, (off, n, _) in cpu.dense_buf.layout.items():
        a, b = gg[off:off + n], gc[off:off + n]
        c = torch.nn.functional.cosine_similarity(a, b, dim=0).item()
        assert c > 0.98, (name, c)
    with torch.no_grad():                                  # scoring: without gradients, with a window or norms op by op
        assert gpu._one_call_ok(gpu.wte(x.cuda()), 257) == ("rope_scaling" in over and len(over) == 3)
        logits = gpu(x.cuda())[0]
        torch.testing.assert_close(logits, gpu(x.cuda())[0], rtol=0, atol=0)
    ref = cpu(x)[0]
    assert ((logits.cpu().float() - ref).norm() / ref.norm()).item() < 2e-2


def test_captured_step():
    """A micro-step captured and replayed on new tokens gives the eager gradients."""
    from train_large_model_from_scratch_b200.ops import native
    model, _ = _models(OPTIONS[-1])
    data = [torch.randint(0, 4096, (2, 301), generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2)]
    x, y = data[0][:, :-1].contiguous(), data[0][:, 1:].contiguous()

    def step():
        model.zero_grad_buffers()
        _, loss, _ = model(x, y)
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for d in (data[1], data[0]):
        x.copy_(d[:, :-1])
        y.copy_(d[:, 1:])
        graph.replay()
        torch.cuda.synchronize()
        loss, grads = captured.clone(), model.dense_buf.main_grad.clone()
        eager = step()
        torch.cuda.synchronize()
        assert abs(loss.item() - eager.item()) < 1e-5
        # reductions in hardware order round differently, half a step of bf16 in dQ
        assert ((grads - model.dense_buf.main_grad).norm() <= 2 * H * grads.norm()).item()
    native.raise_on_device_status()


@pytest.mark.parametrize("which", ["window", "norm", "all"])
def test_captured_beside_an_eager_graph_of_the_same_parameters(which):
    """Forward and backward of an operator captured while an eager graph of the same weights lives: they are no inputs of its node."""
    from train_large_model_from_scratch_b200.ops import functional as F_ops, native
    n_q, n_kv = 4, 2
    qkv, do, w = _case(1, 300, n_q, n_kv, 64, True, seed=2)
    pos, freq = torch.arange(300, device="cuda"), 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
    for p in w:
        p.main_grad = torch.zeros(64, device="cuda")

    def call(x):
        if which == "window":
            return F_ops.attention_packed(x, n_q, n_kv, window=60, sinks=2)
        if which == "norm":
            return F_ops.qk_norm_rotary(x[:, :, :n_q], 2, *w, pos, freq)
        return F_ops.rotary_attention(x, n_q, n_kv, pos, freq, norm_weights=w, window=60, sinks=2)

    def step():
        for p in w:
            p.main_grad.zero_()
        x = qkv.detach().requires_grad_()
        o = call(x)
        return o.detach(), torch.autograd.grad(o, x, do)[0]

    first = qkv.detach().requires_grad_()
    alive = call(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, dx = step()
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (o, dx, *(p.main_grad for p in w))]
    want = [*step(), *(p.main_grad.clone() for p in w)]
    torch.autograd.grad(alive, first, do)
    torch.cuda.synchronize()
    native.raise_on_device_status()
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        assert ((a.double() - b.double()).norm() <= 2 * H * b.double().norm()).item()


def test_forward_at_another_length_between_recorded_steps():
    """Scoring a prompt of another length between two steps replaces the positions and frequencies that the model caches; the recorded
    step goes on reading the ones it was recorded with."""
    import tempfile
    from train_large_model_from_scratch_b200.training import Trainer
    from train_large_model_from_scratch_b200.training.config import (CheckpointConfig, Config, DataConfig, LoggingConfig, ModelConfig,
                                                                     OptimConfig, ParallelConfig, SeedConfig, TrainingConfig)
    data = torch.randint(0, 2048, (2, 257), generator=torch.Generator().manual_seed(8)).cuda()
    batch = [{"input_ids": data[:, :-1].contiguous(), "labels": data[:, 1:].contiguous()}]
    runs = []
    for other_lengths in (False, True):
        tr = Trainer(Config(
            logging=LoggingConfig(exp_name="t", log_dir=tempfile.mkdtemp(prefix="tlm_gpu_")), seed=SeedConfig(),
            data=DataConfig(use_mock_data=True, mock_data_num_samples=2),
            train=TrainingConfig(total_batch_size=512, batch_size=2, seq_len=256, max_steps=100, max_epochs=None, debug=True).with_derived(),
            optim=OptimConfig(max_lr=6e-4, min_lr=6e-5, warmup_steps=10), ckpt=CheckpointConfig(), parallel=ParallelConfig(),
            model=ModelConfig(num_layer=2, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512, vocab_size=2048,
                              block_size=512, rope_variant="standard", rope_layout="interleaved", qk_norm=True, attn_window=70, attn_sinks=2)))
        run = []
        for step in range(7):
            run.append(float(tr.train_step(step, batches=batch)["loss"]))
            if other_lengths and step >= 3:
                logits, _, _ = tr.raw_model(data[:, :100])
                del logits
                junk = [torch.full((256,), 12345, device="cuda") for _ in range(64)] + \
                       [torch.full((n,), 3.0, device="cuda", dtype=torch.float64) for n in (32, 256) for _ in range(64)]
                del junk
        assert tr._graph is not None
        runs.append(run)
    for a, b in zip(*runs):
        assert math.isfinite(a) and abs(a - b) < 5e-3 * a, runs
