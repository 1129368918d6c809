"""Per-head norm and rotation of queries and keys: the torch expression against the formulas (CPU), the kernels against
the same definition in 64 bits (GPU)."""

import math

import pytest
import torch

from scaling_b200.ops import functional as K
from scaling_b200.ops._lib import KernelError

DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative


def _turn(z, pos, rotary, sign):
    """Rotation as complex multiplication in fp64 (``z [tokens, heads, d]``)."""
    if rotary is None:
        return z.clone()
    rot, base, interleaved = rotary
    theta = pos.double()[:, None] * torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64,
                                                 device=z.device)
    unit = torch.polar(torch.ones_like(theta), sign * theta)[:, None]
    out = z.clone()
    ia = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    ib = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    c = torch.complex(z[..., ia].contiguous(), z[..., ib].contiguous()) * unit
    out[..., ia], out[..., ib] = c.real, c.imag
    return out


def definition(x, w, b, pos, rotary, eps, rms, dout=None):
    """(out, dx, dw, db) in fp64 and the sizes that their error bounds scale with."""
    x, w = x.detach().double(), w.detach().double()
    mu = torch.zeros_like(x[..., :1]) if rms else x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xhat = (x - mu) * r
    y = xhat * w + (0.0 if b is None else b.detach().double())
    out = _turn(y, pos, rotary, 1.0)
    size = (x.abs().amax(-1, keepdim=True) * r * w.abs().max()) + y.abs().amax(-1, keepdim=True)
    if dout is None:
        return out, size
    dy = _turn(dout.double(), pos, rotary, -1.0)
    g = dy * w
    gx = (g * xhat).mean(-1, keepdim=True)
    gm = torch.zeros_like(gx) if rms else g.mean(-1, keepdim=True)
    dx = r * (g - gm - xhat * gx)
    xs = x.abs().amax(-1, keepdim=True) * r
    dx_size = r * (g.abs().amax(-1, keepdim=True)) * (2.0 + xs + xs ** 2)
    return (out, size, dx, dx_size, (dy * xhat).sum((0, 1)), (dy.abs() * xs).sum((0, 1)), dy.sum((0, 1)),
            dy.abs().sum((0, 1)))


def _inputs(T, Hq, Hk, D, dtype, w_dtype, rms, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q = (mk(T, Hq, D) * torch.exp(mk(Hq, 1)) + 0.5).to(dtype).to(device)
    k = (mk(T, Hk, D) * torch.exp(mk(Hk, 1)) - 0.25).to(dtype).to(device)
    ws = [(1.0 + 0.3 * mk(D)).to(w_dtype).to(device) for _ in range(2)]
    bs = [None, None] if rms else [(0.2 * mk(D)).to(w_dtype).to(device) for _ in range(2)]
    pos = torch.randint(0, 200000, (T,), generator=g).to(device)
    gq, gk = mk(T, Hq, D).to(dtype).to(device), mk(T, Hk, D).to(dtype).to(device)
    return q, k, ws, bs, pos, gq, gk


def _close(got, want, size, steps, what):
    """|got - want| within one rounding to got's type plus `steps` fp32 half steps of `size`."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny  # below it the spacing no longer shrinks with the value
    bound = half * (want.abs() + steps * U * size) + steps * U * size + half * tiny
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: {(err / bound).max().item():.3g} of the bound"


# Error of the forward value in fp32 half steps of max|x| r max|w| + max|y|: a mean over D <= 256 elements is a chain of
# at most 16 lane additions and 5 shuffles (V = 1: 8 + 5), so 21 for mu and 21 for the sum of squares (halved by the
# square root), the division 1 each, rsqrtf 4 (2 ulp), difference, two products and the bias 4, the two products and the
# sum of the rotation 3, the sine and cosine of an angle rounded to fp32 turns (|rest| <= 1/2: 2^-26 turns, times 2 pi
# is 1.6 steps) and of 2 ulp 6: below 64 in all.
FWD_STEPS = 64
# dx: xhat as above (2 x 40), g 1 + rotation 10, two more means of 21 each against sizes that dx_size holds: below 192.
BWD_STEPS = 192

CASES = [
    # T, Hq, Hk, D, rotary, rms
    (1, 1, 1, 64, (64, 10000.0, False), True),
    (1, 32, 8, 128, (128, 10000.0, True), True),
    (7, 3, 1, 32, (16, 10000.0, False), False),
    (130, 12, 12, 64, (64, 10000.0, False), False),
    (257, 8, 2, 128, (32, 500000.0, True), True),
    (65, 5, 5, 80, (20, 10000.0, False), True),      # rotated half of 10: not whole 16-byte chunks
    (33, 4, 2, 96, (96, 10000.0, True), False),
    (33, 4, 2, 96, (36, 10000.0, True), False),      # the rotated part ends inside a chunk
    (19, 2, 1, 256, (256, 10000.0, False), False),
    (19, 2, 1, 256, None, True),
    (40, 3, 3, 50, (6, 10000.0, False), True),       # rows that are no multiple of 16 bytes
    (23, 2, 2, 7, (4, 10000.0, True), False),        # odd head size
    (300, 71, 1, 64, (64, 10000.0, False), True),
]


@pytest.mark.parametrize("T,Hq,Hk,D,rotary,rms", CASES)
def test_torch_expression_follows_the_definition(T, Hq, Hk, D, rotary, rms):
    q, k, ws, bs, pos, gq, gk = _inputs(T, Hq, Hk, D, torch.float64, torch.float64, rms, "cpu")
    leaves = [t.requires_grad_() for t in (q, k, *ws, *(b for b in bs if b is not None))]
    outs = K.qk_norm_rope(q, k, ws[0], ws[1], q_bias=bs[0], k_bias=bs[1], positions=pos, rotary=rotary, eps=1e-5, rms=rms)
    grads = torch.autograd.grad(outs, leaves, (gq, gk))
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        out, _, dx, _, dw, _, db, _ = definition(x, ws[i], bs[i], pos, rotary, 1e-5, rms, g)
        assert torch.allclose(outs[i], out, rtol=1e-9, atol=1e-9)
        assert torch.allclose(grads[i], dx, rtol=1e-8, atol=1e-8)
        assert torch.allclose(grads[2 + i], dw, rtol=1e-8, atol=1e-8)
        if not rms:
            assert torch.allclose(grads[4 + i], db, rtol=1e-8, atol=1e-8)


def test_gradient_against_differences():
    q, k, ws, bs, pos, _, _ = _inputs(3, 2, 1, 6, torch.float64, torch.float64, False, "cpu")
    args = [t.requires_grad_() for t in (q, k, *ws, *bs)]
    assert torch.autograd.gradcheck(
        lambda *a: K.qk_norm_rope(a[0], a[1], a[2], a[3], q_bias=a[4], k_bias=a[5], positions=pos % 100,
                                  rotary=(4, 100.0, False), rms=False), args)


def test_equals_norm_then_rope():
    q, k, ws, bs, _, _, _ = _inputs(9, 4, 2, 16, torch.float32, torch.float32, False, "cpu")
    pos = torch.arange(9)
    got = K.qk_norm_rope(q, k, ws[0], ws[1], q_bias=bs[0], k_bias=bs[1], positions=pos, rotary=(8, 10000.0, False), rms=False)
    for x, w, b, y in ((q, ws[0], bs[0], got[0]), (k, ws[1], bs[1], got[1])):
        assert torch.allclose(y, K.rope(K.layer_norm(x, w, b), pos, 8), atol=1e-5)


def _refused(device):
    q, k, ws, bs, pos, _, _ = _inputs(5, 4, 2, 16, torch.float32, torch.float32, True, device)
    ok = dict(positions=pos, rotary=(8, 10000.0, False))
    K.qk_norm_rope(q, k, *ws, **ok)
    bad = [
        lambda: K.qk_norm_rope(q, k, None, ws[1], **ok),
        lambda: K.qk_norm_rope(q, k, ws[0][:8], ws[1], **ok),
        lambda: K.qk_norm_rope(q[0], k, *ws, **ok),
        lambda: K.qk_norm_rope(q, k[:4], *ws, **ok),
        lambda: K.qk_norm_rope(q, k[..., :8], ws[0], ws[1][:8], **ok),
        lambda: K.qk_norm_rope(q, k.bfloat16(), *ws, **ok),
        lambda: K.qk_norm_rope(q, k, *ws, q_bias=ws[0], **ok),              # a bias with RMSNorm
        lambda: K.qk_norm_rope(q, k, *ws, rotary=(8, 10000.0, False)),      # no positions
        lambda: K.qk_norm_rope(q, k, *ws, positions=pos[:3], rotary=(8, 10000.0, False)),
        lambda: K.qk_norm_rope(q, k, *ws, positions=pos.float(), rotary=(8, 10000.0, False)),
        lambda: K.qk_norm_rope(q, k, *ws, positions=pos, rotary=(7, 10000.0, False)),
        lambda: K.qk_norm_rope(q, k, *ws, positions=pos, rotary=(18, 10000.0, False)),
        lambda: K.qk_norm_rope(q, k, *ws, positions=pos, rotary=(8, 0.0, False)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_refusals():
    _refused("cpu")


def test_no_tokens():
    q = torch.zeros(0, 4, 16, requires_grad=True)
    w = torch.ones(16, requires_grad=True)
    a, b = K.qk_norm_rope(q, q[:, :2], w, w, positions=torch.zeros(0, dtype=torch.int32), rotary=(16, 10000.0, False))
    assert a.shape == (0, 4, 16) and b.shape == (0, 2, 16)
    (a.sum() + b.sum()).backward()
    assert torch.equal(w.grad, torch.zeros(16))


# ------------------------------------------------------------------------------------------------ GPU
def _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, rms):
    leaves = [t.detach().requires_grad_() for t in (q, k, *ws)] + [b.detach().requires_grad_() for b in bs if b is not None]
    bl = leaves[4:] if not rms else [None, None]
    outs = K.qk_norm_rope(*leaves[:4], q_bias=bl[0], k_bias=bl[1], positions=pos, rotary=rotary, eps=1e-5, rms=rms)
    return outs, torch.autograd.grad(outs, leaves, (gq, gk))


def _check_all(outs, grads, q, k, ws, bs, pos, gq, gk, rotary, rms):
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        out, size, dx, dx_size, dw, dw_size, db, db_size = definition(x, ws[i], bs[i], pos, rotary, 1e-5, rms, g)
        # a chain of additions: at most rows / 8 per thread (eight row groups at least), then warps, blocks and lanes
        steps = x.shape[0] * x.shape[1] / 8 + 512
        _close(outs[i], out, size, FWD_STEPS, f"out {i}")
        _close(grads[i], dx, dx_size, BWD_STEPS, f"dx {i}")
        _close(grads[2 + i], dw, dw_size, steps, f"dw {i}")
        if not rms:
            _close(grads[4 + i], db, db_size, steps, f"db {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.float32, torch.float32)])
@pytest.mark.parametrize("T,Hq,Hk,D,rotary,rms", CASES)
def test_kernel_follows_the_definition(T, Hq, Hk, D, rotary, rms, dtype, w_dtype):
    q, k, ws, bs, pos, gq, gk = _inputs(T, Hq, Hk, D, dtype, w_dtype, rms, DEV)
    outs, grads = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, rms)
    assert [o.dtype for o in outs] == [dtype] * 2 and all(o.is_contiguous() for o in outs)
    _check_all(outs, grads, q, k, ws, bs, pos, gq, gk, rotary, rms)


@pytest.mark.gpu
def test_gpu_refusals():
    _refused(DEV)
    x = torch.zeros(2, 1, 258, device=DEV)
    with pytest.raises(KernelError):
        K.qk_norm_rope(x, x, x[0, 0], x[0, 0])
    x = torch.zeros(2, 1, 64, device=DEV, dtype=torch.float64)
    with pytest.raises(KernelError):
        K.qk_norm_rope(x, x, x[0, 0], x[0, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_a_packed_projection_and_odd_strides(dtype):
    T, H, D = 67, 6, 64
    rotary = (64, 10000.0, False)
    _, _, ws, bs, pos, gq, gk = _inputs(T, H, H, D, dtype, dtype, True, DEV)
    packed = torch.randn(T, H, 3 * D, device=DEV).to(dtype)
    wide = torch.randn(T, H, D + 3, device=DEV).to(dtype)      # rows that start on any element
    turned = torch.randn(H, D, T, device=DEV).to(dtype)        # innermost dimension not contiguous
    one = torch.randn(1, H, D, device=DEV).to(dtype).expand(T, H, D)  # every token the same memory
    views = [(packed[..., :D], packed[..., D:2 * D]), (wide[..., 1:D + 1], wide[..., 3:]),
             (turned.permute(2, 0, 1), packed[..., 2 * D:]), (one, one)]
    for q, k in views:
        outs, grads = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, True)
        _check_all(outs, grads, q, k, ws, bs, pos, gq, gk, rotary, True)
    # gradients that arrive as a stride-0 expansion, and none at all for the queries
    q = views[0][0].detach().requires_grad_()
    k = views[0][1].detach().requires_grad_()
    K.qk_norm_rope(q, k, *ws, positions=pos, rotary=rotary)[1].sum().backward()
    assert torch.count_nonzero(q.grad) == 0
    _, _, dx, dx_size, *_ = definition(k, ws[1], None, pos, rotary, 1e-5, True, torch.ones_like(k))
    _close(k.grad, dx, dx_size, BWD_STEPS, "dk")


@pytest.mark.gpu
def test_shared_weight_and_persistent_gradient_buffers():
    T, Hq, Hk, D = 200, 8, 2, 64
    rotary = (64, 10000.0, True)
    q, k, ws, bs, pos, gq, gk = _inputs(T, Hq, Hk, D, torch.bfloat16, torch.float32, True, DEV)
    _, want = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, True)
    _, both = _run_gpu(q, k, [ws[0], ws[0]], bs, pos, gq, gk, rotary, True)
    start = torch.randn(D, device=DEV)
    for same in (False, True):
        params = [torch.nn.Parameter(ws[0].clone())]
        params.append(params[0] if same else torch.nn.Parameter(ws[1].clone()))
        for p in set(params):
            p.grad = start.clone()
            p.fused_grad_accumulation = True
        outs = K.qk_norm_rope(q, k, *params, positions=pos, rotary=rotary)
        torch.autograd.backward(outs, (gq, gk))
        sums = [both[2] + both[3]] if same else [want[2], want[3]]
        for p, s in zip(params, sums):
            assert torch.allclose(p.grad, start + s, rtol=1e-5, atol=1e-4 * s.abs().max().item())


@pytest.mark.gpu
def test_same_bits_every_time_and_frozen_weights():
    q, k, ws, bs, pos, gq, gk = _inputs(999, 12, 4, 64, torch.bfloat16, torch.bfloat16, False, DEV)
    rotary = (32, 10000.0, False)
    first = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, False)
    again = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, False)
    for a, b in zip(first[0] + first[1], again[0] + again[1]):
        assert torch.equal(a, b)
    ql, kl = q.detach().requires_grad_(), k.detach().requires_grad_()
    outs = K.qk_norm_rope(ql, kl, *ws, q_bias=bs[0], k_bias=bs[1], positions=pos, rotary=rotary, rms=False)
    for a, b in zip(torch.autograd.grad(outs, (ql, kl), (gq, gk)), first[1][:2]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_bad_rows_stay_alone():
    """A token with infinities or NaN spoils its own rows, nothing else; a row of zeros gives zeros (plus the bias)."""
    q, k, ws, bs, pos, gq, gk = _inputs(50, 4, 2, 128, torch.bfloat16, torch.bfloat16, True, DEV)
    rotary = (128, 10000.0, False)
    clean, _ = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, True)
    q2 = q.clone()
    q2[3, 1, 5], q2[4, 2, 7], q2[6, 0] = float("nan"), float("inf"), 0.0
    outs, grads = _run_gpu(q2, k, ws, bs, pos, gq, gk, rotary, True)
    keep = torch.ones(50, 4, dtype=torch.bool, device=DEV)
    keep[3, 1] = keep[4, 2] = keep[6, 0] = False
    assert torch.equal(outs[0][keep], clean[0][keep]) and torch.equal(outs[1], clean[1])
    assert torch.count_nonzero(outs[0][6, 0]) == 0 and torch.isfinite(grads[0][keep]).all()


@pytest.mark.gpu
def test_captured_step_and_other_stream():
    q, k, ws, bs, pos, gq, gk = _inputs(300, 6, 3, 80, torch.float16, torch.float16, True, DEV)
    rotary = (80, 10000.0, True)
    leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]

    def step():
        outs = K.qk_norm_rope(*leaves, positions=pos.int(), rotary=rotary)
        return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, leaves, (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    with torch.no_grad():
        saved = q.clone()
        leaves[0].mul_(0.5)
    graph.replay()
    changed = [t.clone() for t in static]
    assert not torch.equal(changed[2], eager[2])
    with torch.no_grad():
        leaves[0].copy_(saved)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(static, eager):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_far_positions_keep_their_angles():
    T = 64
    q, k, ws, bs, _, gq, gk = _inputs(T, 2, 1, 128, torch.float32, torch.float32, True, DEV)
    pos = torch.arange(T, device=DEV) * 7919 + 2 ** 30
    pos[0], pos[1] = -5, 2 ** 31 - 1
    rotary = (128, 10000.0, False)
    outs, grads = _run_gpu(q, k, ws, bs, pos, gq, gk, rotary, True)
    _check_all(outs, grads, q, k, ws, bs, pos, gq, gk, rotary, True)


@pytest.mark.gpu
def test_more_rows_than_32_bits_of_elements():
    """Offsets of the last rows pass 2^31 elements."""
    T, H, D = 2 ** 20 + 3, 32, 64
    x = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    x.view(-1)[:].random_(-3, 4)
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    with torch.no_grad():
        a, b = K.qk_norm_rope(x, x[:, :1], w, w, positions=pos, rotary=(64, 10000.0, False))
    for t in (0, T // 2, T - 1):
        want, size = definition(x[t:t + 1], w, None, pos[t:t + 1], (64, 10000.0, False), 1e-5, True)
        _close(a[t:t + 1], want, size, FWD_STEPS, f"token {t}")
        _close(b[t:t + 1], want[:, :1], size[:, :1], FWD_STEPS, f"token {t}")


# Rotation alone: the angle and its sine and cosine 8 steps (see above), two products and a sum of the pair 3, each of at
# most sqrt(2) max|x|: below 32 in all.
TURN_STEPS = 32


def _check_head_rotation(x, pos, rotary, g):
    leaf = x.detach().requires_grad_()
    y = K.head_rotation(leaf, pos, rotary)
    (dx,) = torch.autograd.grad(y, leaf, g)
    _close(y, _turn(x.double(), pos, rotary, 1.0), x.double().abs().amax(-1, keepdim=True), TURN_STEPS, "y")
    _close(dx, _turn(g.double(), pos, rotary, -1.0), g.double().abs().amax(-1, keepdim=True), TURN_STEPS, "dx")
    with torch.no_grad():
        assert torch.equal(K.head_rotation(x, pos, rotary), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rotary", [(16, 10000.0, False), (16, 500000.0, True), (6, 10000.0, True)])
def test_rotation_alone_torch_expression(rotary, dtype):
    q, _, _, _, pos, g, _ = _inputs(9, 3, 1, 16, dtype, dtype, True, "cpu")
    _check_head_rotation(q, pos, rotary, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D,rotary", [(1, 1, 64, (64, 10000.0, False)), (130, 12, 128, (128, 10000.0, True)),
                                          (67, 5, 80, (20, 10000.0, False)), (33, 3, 50, (6, 500000.0, True)),
                                          (9, 2, 256, (256, 10000.0, False)), (700, 71, 64, (32, 10000.0, False)),
                                          (9, 2, 320, (64, 10000.0, False))])
def test_rotation_alone_kernel(T, H, D, rotary, dtype):
    q, _, _, _, pos, g, _ = _inputs(T, H, 1, D, dtype, dtype, True, DEV)
    pos[0] = 10 ** 9
    _check_head_rotation(q, pos, rotary, g)
    turned = q.permute(1, 2, 0).contiguous().permute(2, 0, 1)  # as heads that were gathered over ranks come
    assert torch.equal(K.head_rotation(turned, pos, rotary), K.head_rotation(q, pos, rotary))


def _rotation_refused(device):
    q, _, _, _, pos, _, _ = _inputs(9, 3, 1, 16, torch.float32, torch.float32, True, device)
    rotary = (16, 10000.0, False)
    K.head_rotation(q, pos, rotary)
    K.head_rotation(q, pos.float(), rotary)
    for x, p, r in ((q, pos[:8], rotary), (q, pos[:1], rotary), (q, pos[None], rotary), (q, torch.cat((pos, pos)), rotary),
                    (q[0], pos, rotary), (q, pos, (18, 10000.0, False)), (q, pos, (7, 10000.0, False))):
        with pytest.raises(ValueError):
            K.head_rotation(x, p, r)


def test_rotation_alone_refusals():
    _rotation_refused("cpu")


@pytest.mark.gpu
def test_rotation_alone_gpu_refusals():
    _rotation_refused(DEV)
    q, _, _, _, pos, _, _ = _inputs(9, 3, 1, 16, torch.float32, torch.float32, True, DEV)
    with pytest.raises(ValueError):
        K.head_rotation(q, pos.cpu(), (16, 10000.0, False))
