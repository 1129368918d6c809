"""Self-attention with norms of queries and keys: norms and rotation in one kernel against the separate operations."""

import pytest
import torch

from scaling_b200.core.nn.attention import ParallelSelfAttention
from scaling_b200.core.nn.attention.attention import RelativePositionEmbeddingType
from scaling_b200.core.nn.masked_softmax import MaskedSoftmaxConfig
from scaling_b200.core.nn.norm import LayerNormConfig, NormType
from scaling_b200.core.nn.rotary import RotaryConfig
from scaling_b200.ops import functional as K


def _attention(norm_type, device, dtype, heads=4, kv_heads=None, rotary="rotary", rot_dims=64, seed=0):
    torch.manual_seed(seed)
    kind = RelativePositionEmbeddingType(rotary)
    m = ParallelSelfAttention(
        hidden_size=64 * heads, num_attention_heads=heads, masked_softmax_config=MaskedSoftmaxConfig(kernel="flash_attention"),
        rotary_config=RotaryConfig(dimensions=rot_dims), relative_position_embedding_type=kind, device=torch.device(device),
        dtype=dtype, norm_type=norm_type, key_query_norm=True, layernorm_config=LayerNormConfig(),
        qkv_in_one=kv_heads is None, num_kv_heads=kv_heads)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.startswith("norm_"):
                p.add_(0.2 * torch.randn_like(p))
    return m


def _step(m, x, cu, pos):
    for p in m.parameters():
        p.grad = None
    xi = x.detach().requires_grad_()
    y = m(xi, cu, pos)
    y.backward(torch.linspace(-1, 1, y.numel(), device=y.device).view_as(y).to(y.dtype))
    return y.detach(), xi.grad, {n: p.grad for n, p in m.named_parameters()}


@pytest.mark.gpu
@pytest.mark.parametrize("norm_type", [NormType.RMS, NormType.LAYERNORM])
@pytest.mark.parametrize("kv_heads,rotary,rot_dims", [(None, "rotary", 64), (2, "rotary_complex", 64), (None, "rotary", 16), (1, "none", 64)])
def test_attention_with_head_norms_in_one_kernel(norm_type, kv_heads, rotary, rot_dims, monkeypatch):
    dev = "cuda"
    m = _attention(norm_type, dev, torch.bfloat16, kv_heads=kv_heads, rotary=rotary, rot_dims=rot_dims)
    x = torch.randn(2, 40, 256, device=dev).bfloat16()
    cu = torch.tensor([0, 25, 40, 80], dtype=torch.int32, device=dev)
    pos = torch.arange(40, device=dev).repeat(2, 1)
    calls = []
    real = K.qk_norm_rope
    monkeypatch.setattr(K, "qk_norm_rope", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    fused = _step(m, x, cu, pos)
    assert len(calls) == 1
    monkeypatch.setattr(ParallelSelfAttention, "_head_norm_fused", lambda self, q: False)
    separate = _step(m, x, cu, pos)
    assert len(calls) == 1
    # Both against the same module in fp32 on the CPU.  All roundings of the fused form are also made by the separate one
    # (which makes two more per element and pass), so its distance is of the same size or smaller; a factor of two leaves
    # room for the signs in which they happen to add up.  (The distance of the two from each other has no bound in terms of
    # the result: the weights' gradients are sums in which large terms cancel.)
    ref = _attention(norm_type, "cpu", torch.float32, kv_heads=kv_heads, rotary=rotary, rot_dims=rot_dims)
    ref.load_state_dict({n: t.float().cpu() for n, t in m.state_dict().items()})
    want = _step(ref, x.float().cpu(), cu.cpu(), pos.cpu())
    triples = [(fused[0], separate[0], want[0]), (fused[1], separate[1], want[1])]
    triples += [(fused[2][n], separate[2][n], want[2][n]) for n in fused[2]]
    for a, b, w in triples:
        assert (a is None) == (b is None) == (w is None)
        if a is not None:
            dist = lambda t: (t.float().cpu() - w).norm().item()  # noqa: E731
            assert dist(a) <= 2.0 * dist(b) + 2.0 ** -8 * w.norm().item()


@pytest.mark.gpu
def test_hooks_on_the_norms_still_see_their_outputs():
    m = _attention(NormType.RMS, "cuda", torch.bfloat16)
    seen = []
    handle = m.norm_query.register_forward_hook(lambda mod, args, out: seen.append(out.shape))
    x = torch.randn(1, 16, 256, device="cuda").bfloat16()
    cu = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    a = m(x, cu, None)
    handle.remove()
    b = m(x, cu, None)
    assert seen == [(16, 4, 64)]
    assert (a.float() - b.float()).norm() <= 4 * 2.0 ** -8 * b.float().norm()


@pytest.mark.gpu
def test_backward_hooks_on_the_norms_still_run():
    m = _attention(NormType.RMS, "cuda", torch.bfloat16)
    seen = []
    m.norm_key.register_full_backward_hook(lambda mod, gi, go: seen.append(go[0].shape))
    x = torch.randn(1, 16, 256, device="cuda").bfloat16().requires_grad_()
    m(x, torch.tensor([0, 16], dtype=torch.int32, device="cuda"), None).float().sum().backward()
    assert seen == [(16, 4, 64)]


def test_separate_operations_on_the_cpu():
    m = _attention(NormType.LAYERNORM, "cpu", torch.float32)
    x = torch.randn(2, 10, 256)
    cu = torch.tensor([0, 10, 20], dtype=torch.int32)
    y, dx, grads = _step(m, x, cu, None)
    assert y.shape == x.shape and torch.isfinite(dx).all()
    assert all(g is not None and torch.isfinite(g).all() for g in grads.values())


@pytest.mark.gpu
def test_cached_generation_step_uses_the_same_kernel():
    """A prompt and then single tokens through the module's cache equal the whole sequence at once."""
    m = _attention(NormType.RMS, "cuda", torch.bfloat16)
    x = torch.randn(1, 21, 256, device="cuda").bfloat16()
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device="cuda")  # noqa: E731
    with torch.no_grad():
        whole = m(x, cu(21), None)
        parts = [m(x[:, :20], cu(20), torch.arange(20, device="cuda")[None], use_cache=True, reset_cache=True),
                 m(x[:, 20:], cu(1), torch.tensor([[20]], device="cuda"), use_cache=True)]
    got = torch.cat(parts, 1)
    assert (got.float() - whole.float()).norm() <= 4 * 2.0 ** -8 * whole.float().norm()


class _Metrics:
    """Takes the place of the logger and of the training context."""

    iterations = 0

    def __init__(self):
        self.names = set()

    def log_metrics(self, metrics, **_):
        self.names.update(metrics)

    def warning(self, *_):
        pass


@pytest.mark.gpu
def test_traced_steps_record_the_norms():
    from scaling_b200.core.logging.tensor_statistics_recorder import (TensorStatistics, TensorStatisticsRecorder,
                                                                      TensorStatisticsRecorderConfig)

    m = _attention(NormType.RMS, "cuda", torch.bfloat16)
    model = torch.nn.Module()
    model._layers = torch.nn.ModuleList([m])
    log = _Metrics()
    config = TensorStatisticsRecorderConfig(statistics=[("*", [TensorStatistics.MEAN])])
    recorder = TensorStatisticsRecorder(config, log, model, logger=log)
    x = torch.randn(1, 16, 256, device="cuda").bfloat16().requires_grad_()
    cu = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    with recorder.trace():
        m(x, cu, None).float().sum().backward()
    for norm in ("norm_query", "norm_key"):
        for mode in ("forward", "backward"):
            assert f"activation_statistics/layers.0.{norm}_{mode}_mean" in log.names


class _Half(torch.nn.Module):
    def forward(self, x):
        return 0.5 * x


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["module", "one module", "forward"])
def test_norm_modules_that_were_exchanged_are_called(how):
    """Modules put in place of the norms, and a forward of an instance's own, run instead of the kernel."""
    m = _attention(NormType.RMS, "cuda", torch.float32, rotary="none")
    x = torch.randn(1, 16, 256, device="cuda")
    cu = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    seen = {}
    core = m.scaled_dot_product_attention
    real = core.forward
    core.forward = lambda q, k, v, *a, **kw: (seen.update(q=q, k=k), real(q, k, v, *a, **kw))[1]
    with torch.no_grad():
        q, k, _ = m._project_qkv(x)
        want_k = K.rms_norm(k, m.norm_key.weight, m.norm_key.eps)
        if how == "forward":
            m.norm_query.forward = lambda t: 0.5 * t
        else:
            m.norm_query = _Half()
        if how == "module":
            m.norm_key, want_k = _Half(), 0.5 * k
        m(x, cu, None)
    assert torch.equal(seen["q"], 0.5 * q) and torch.equal(seen["k"], want_k)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [(0.5, 0.5), (0.5, 1e-5)])
def test_the_modules_own_epsilon_is_used(eps):
    m = _attention(NormType.RMS, "cuda", torch.float32, rotary="none")
    m.norm_query.eps, m.norm_key.eps = eps
    x = 0.1 * torch.randn(1, 16, 256, device="cuda")
    cu = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    seen = {}
    core = m.scaled_dot_product_attention
    real = core.forward
    core.forward = lambda q, k, v, *a, **kw: (seen.update(q=q, k=k), real(q, k, v, *a, **kw))[1]
    with torch.no_grad():
        q, k, _ = m._project_qkv(x)
        m(x, cu, None)
    for got, t, norm in ((seen["q"], q, m.norm_query), (seen["k"], k, m.norm_key)):
        want = t.double() * torch.rsqrt(t.double().pow(2).mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
        # a sum of 64 squares, the division, the root and two products: below 32 half steps of fp32
        assert ((got - want).abs() <= 32 * 2.0 ** -24 * want.abs() + 2.0 ** -120).all()


@pytest.mark.gpu
def test_floating_point_position_ids():
    m = _attention(NormType.RMS, "cuda", torch.bfloat16)
    x = torch.randn(2, 16, 256, device="cuda").bfloat16()
    cu = torch.tensor([0, 16, 32], dtype=torch.int32, device="cuda")
    pos = torch.arange(16, device="cuda").repeat(2, 1)
    with torch.no_grad():
        want = m(x, cu, pos)
        for kind in (torch.float32, torch.float64, torch.int32, torch.int16):
            assert torch.equal(m(x, cu, pos.to(kind)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", ["rotary", "rotary_complex"])
def test_far_positions_have_the_same_angles_in_every_form(rotary):
    """One kernel, or separate operations because of a hook: the same queries and keys at positions of some millions."""
    m = _attention(NormType.RMS, "cuda", torch.float32, rotary=rotary)
    x = torch.randn(1, 64, 256, device="cuda")
    cu = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    pos = torch.arange(64, device="cuda")[None] * 79190 + 10 ** 6
    seen = []
    core = m.scaled_dot_product_attention
    real = core.forward
    core.forward = lambda q, k, v, *a, **kw: (seen.append((q, k)), real(q, k, v, *a, **kw))[1]
    with torch.no_grad():
        m(x, cu, pos)
        handle = m.norm_query.register_forward_hook(lambda *a: None)
        m(x, cu, pos)
        handle.remove()
    for a, b in zip(*seen):
        # 64 half steps for the norm and the rotation in one kernel, 32 + 32 for the separate ones, of max|y|
        assert ((a - b).abs() <= 128 * 2.0 ** -24 * a.abs().amax(-1, keepdim=True) * 2.0 ** 0.5).all()


def _tensor_parallel_worker(rank, world_size, port, device, kv_heads):
    from tests.test_core_distributed import _topology

    t = _topology(rank, world_size, port, mp=world_size)
    m = ParallelSelfAttention(
        hidden_size=128, num_attention_heads=8, masked_softmax_config=MaskedSoftmaxConfig(), topology=t,
        rotary_config=RotaryConfig(dimensions=16), relative_position_embedding_type=RelativePositionEmbeddingType.ROTARY,
        norm_type=NormType.RMS, key_query_norm=True, layernorm_config=LayerNormConfig(), qkv_in_one=False,
        num_kv_heads=kv_heads)
    g = torch.Generator().manual_seed(11)
    draw = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    full = {"query": draw(128, 128) / 8, "key": draw(kv_heads * 16, 128) / 8, "value": draw(kv_heads * 16, 128) / 8}
    with torch.no_grad():
        for name, w in full.items():
            getattr(m, name).weight.copy_(w.chunk(world_size)[rank])
            getattr(m, name).bias.zero_()
        m.dense.weight.copy_((draw(128, 128) / 8).chunk(world_size, 1)[rank])
        m.dense.bias.zero_()
        m.norm_query.weight.copy_(1 + 0.2 * draw(16))
        m.norm_key.weight.copy_(1 + 0.2 * draw(16))
    x = draw(2, 12, 128).requires_grad_()
    y = m(x, torch.tensor([0, 12, 24], dtype=torch.int32), torch.arange(12).repeat(2, 1) * 7919 + 10 ** 6)
    y.square().sum().backward()
    return y.detach(), x.grad, m.norm_query.weight.grad, m.norm_key.weight.grad


@pytest.mark.dist
@pytest.mark.parametrize("kv_heads", [4])
def test_head_norms_and_far_positions_under_tensor_parallelism(kv_heads):
    """The same outputs and gradients as on one rank; fp32 sums of at most 128 terms in another order."""
    from tests.utils import dist_launcher

    (want,) = dist_launcher(_tensor_parallel_worker, 1, kv_heads=kv_heads)
    for got in dist_launcher(_tensor_parallel_worker, 2, kv_heads=kv_heads):
        for a, b in zip(got, want):
            assert (a - b).norm() <= 512 * 2.0 ** -24 * b.norm()
