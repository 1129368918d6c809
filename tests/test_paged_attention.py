"""Writes into a paged key/value cache and attention over it, against plain evaluations in 64 bits."""

import math
import random

import pytest
import torch

from scaling_b200.ops import functional as K
from scaling_b200.ops._lib import KernelError
from scaling_b200.ops.paged_attention import paged_append, paged_attention
from tests.test_qk_norm_rope import FWD_STEPS, _close, _turn, definition

DEV = "cuda"


class Batch:
    """Packed new tokens of several sequences and their pages in a cache (pages in random order, every unused entry of
    the table -1, every unused element of the caches NaN)."""

    def __init__(self, lens, new, page, kv_heads, dim, dtype, device, heads=None, spare_rows=0, seed=0, fill=float("nan"),
                 joint=False):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.page = list(lens), list(new), page
        counts = [-(-n // page) for n in self.lens]
        ids = list(range(sum(counts) + 3))
        rng.shuffle(ids)
        cols = max(counts + [1]) + 1
        table = torch.full((len(self.lens), cols), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
            at += c
        self.table_cpu = table
        self.table = table.to(device)
        cu = [0]
        for n in self.new:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=device)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.tokens = cu[-1]
        rows = self.tokens + spare_rows
        shape = (len(ids), page, kv_heads, dim)
        if joint:  # keys and values of a page side by side in one tensor
            both = torch.full((len(ids), 2, page, kv_heads, dim), fill, dtype=dtype, device=device)
            self.k_cache, self.v_cache = both[:, 0], both[:, 1]
        else:
            self.k_cache = torch.full(shape, fill, dtype=dtype, device=device)
            self.v_cache = torch.full(shape, fill, dtype=dtype, device=device)
        mk = lambda h: torch.randn(rows, h, dim, generator=g).to(dtype).to(device)  # noqa: E731
        self.q, self.k, self.v = mk(heads or kv_heads), mk(kv_heads), mk(kv_heads)

    def place(self, b, p):
        return int(self.table_cpu[b, p // self.page]), p % self.page

    def positions(self):
        return [(b, length - n + i) for b, (n, length) in enumerate(zip(self.new, self.lens)) for i in range(n)]

    def fill_history(self, seed=1, scale=1.0):
        """Random keys and values at every position of every sequence (the new ones included)."""
        g = torch.Generator().manual_seed(seed)
        kc, vc = self.k_cache.cpu(), self.v_cache.cpu()
        for b, length in enumerate(self.lens):
            for i in range(-(-length // self.page)):
                n = min(self.page, length - i * self.page)
                page = int(self.table_cpu[b, i])
                kc[page, :n] = (scale * torch.randn(n, *kc.shape[2:], generator=g)).to(kc.dtype)
                vc[page, :n] = torch.randn(n, *vc.shape[2:], generator=g).to(vc.dtype)
        self.k_cache.copy_(kc)
        self.v_cache.copy_(vc)

    def args(self):
        return self.k_cache, self.v_cache, self.table, self.cu, self.seq_lens


APPENDS = [
    # lens, new, page, heads, kv_heads, dim, rotary, norm
    ([5], [1], 16, 4, 4, 64, (64, 10000.0, False), "rms"),
    ([17, 3, 40], [1, 1, 1], 16, 8, 2, 128, (128, 10000.0, True), "rms"),
    ([30, 16, 0, 9], [30, 7, 0, 2], 8, 3, 1, 80, (20, 10000.0, False), "layer"),
    ([300, 1], [123, 1], 64, 4, 2, 64, (32, 500000.0, False), "none"),
    ([64, 65], [64, 65], 32, 2, 2, 50, None, "layer"),
    ([70, 80], [9, 80], 128, 5, 5, 32, None, "none"),
]


def _append_case(lens, new, page, heads, kv_heads, dim, rotary, norm, dtype, device, joint=False, spare=0):
    b = Batch(lens, new, page, kv_heads, dim, dtype, device, heads=heads, spare_rows=spare, joint=joint)
    g = torch.Generator().manual_seed(7)
    w = lambda base: (base + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(device)  # noqa: E731
    kw = {}
    if norm != "none":
        kw.update(q_weight=w(1.0), k_weight=w(1.0))
    if norm == "layer":
        kw.update(q_bias=w(0.0), k_bias=w(0.0))
    q = paged_append(b.k, b.v, *b.args(), q=b.q, rotary=rotary, rms=norm == "rms", **kw)
    return b, q, kw


def _check_append(b, q, kw, rotary, norm):
    pos = torch.tensor([p for _, p in b.positions()], dtype=torch.int64, device=q.device)

    def want(x, w, bias):
        x = x[:b.tokens]
        if norm == "none":
            return _turn(x.double(), pos, rotary, 1.0), x.double().abs().amax(-1, keepdim=True)
        return definition(x, w, bias, pos, rotary, 1e-5, norm == "rms")

    wq, size = want(b.q, kw.get("q_weight"), kw.get("q_bias"))
    _close(q[:b.tokens], wq, size, FWD_STEPS, "q")
    assert torch.count_nonzero(q[b.tokens:]) == 0
    wk, size = want(b.k, kw.get("k_weight"), kw.get("k_bias"))
    touched = torch.zeros(b.k_cache.shape[:2], dtype=torch.bool, device=q.device)
    places = [b.place(*p) for p in b.positions()]
    page = torch.tensor([x for x, _ in places], dtype=torch.int64, device=q.device)
    slot = torch.tensor([y for _, y in places], dtype=torch.int64, device=q.device)
    touched[page, slot] = True
    _close(b.k_cache[page, slot], wk, size, FWD_STEPS, "k")
    if rotary is None and norm == "none":
        assert torch.equal(b.k_cache[page, slot], b.k[:b.tokens]) and torch.equal(q[:b.tokens], b.q[:b.tokens])
    assert torch.equal(b.v_cache[page, slot], b.v[:b.tokens])
    for c in (b.k_cache, b.v_cache):  # everything else keeps what it held
        assert torch.isnan(c[~touched]).all()


@pytest.mark.parametrize("lens,new,page,heads,kv_heads,dim,rotary,norm", APPENDS)
def test_append_torch_expression(lens, new, page, heads, kv_heads, dim, rotary, norm):
    b, q, kw = _append_case(lens, new, page, heads, kv_heads, dim, rotary, norm, torch.float32, "cpu", spare=3)
    _check_append(b, q, kw, rotary, norm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("lens,new,page,heads,kv_heads,dim,rotary,norm", APPENDS)
def test_append_kernel(lens, new, page, heads, kv_heads, dim, rotary, norm, joint, dtype):
    b, q, kw = _append_case(lens, new, page, heads, kv_heads, dim, rotary, norm, dtype, DEV, joint=joint, spare=3)
    _check_append(b, q, kw, rotary, norm)
    K.check_status()


def _append_refused(device):
    b = Batch([20, 5], [4, 1], 16, 2, 64, torch.float32, device, heads=4)
    ok = lambda **kw: {**dict(q=b.q, rotary=(64, 10000.0, False)), **kw}  # noqa: E731
    w = torch.ones(64, device=device)
    paged_append(b.k, b.v, *b.args(), **ok())
    kc, vc, table, cu, sl = b.args()
    bad = [
        lambda: paged_append(b.k, b.v[:4], *b.args(), **ok()),
        lambda: paged_append(b.k[:, :1], b.v[:, :1], *b.args(), **ok()),
        lambda: paged_append(b.k.bfloat16(), b.v, *b.args(), **ok()),
        lambda: paged_append(b.k[..., :32], b.v, *b.args(), **ok()),
        lambda: paged_append(b.k, b.v, kc, vc[:, :8], table, cu, sl, **ok()),
        lambda: paged_append(b.k, b.v, kc[:, :12], vc[:, :12], table, cu, sl, **ok()),      # page size 12
        lambda: paged_append(b.k, b.v, kc, vc, table.long(), cu, sl, **ok()),
        lambda: paged_append(b.k, b.v, kc, vc, table, cu[:2], sl, **ok()),
        lambda: paged_append(b.k, b.v, kc, vc, table[:1], cu, sl, **ok()),
        lambda: paged_append(b.k, b.v, kc, vc, table.t(), cu, sl, **ok()),
        lambda: paged_append(b.k, b.v, *b.args(), **ok(q=b.q[:3])),
        lambda: paged_append(b.k, b.v, *b.args(), q=None, q_weight=w),
        lambda: paged_append(b.k, b.v, *b.args(), **ok(k_bias=w)),
        lambda: paged_append(b.k, b.v, *b.args(), **ok(rotary=(66, 10000.0, False))),
        lambda: paged_append(b.k, b.v, *b.args(), **ok(positions=torch.zeros(4, dtype=torch.int32, device=device))),
        lambda: paged_append(b.k, b.v, *b.args(), **ok(positions=torch.zeros(5, device=device))),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KernelError):
        paged_append(b.k.requires_grad_(), b.v, *b.args(), **ok())
    with torch.no_grad():
        paged_append(b.k, b.v, *b.args(), **ok())


def test_append_refusals():
    _append_refused("cpu")


def _bad_places(b):
    """(what is wrong, table, cu, seq_lens) of calls that name a place outside the cache or the table."""
    kc, _, table, cu, sl = b.args()
    for bad_id in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 1] = bad_id
        yield f"page {bad_id}", t, cu, sl
    for length in (2, 10 ** 6, -3):  # fewer than the new tokens, beyond the table, negative
        s = sl.clone()
        s[0] = length
        yield f"length {length}", table, cu, s


def test_append_bad_places_on_the_cpu():
    b = Batch([20, 5], [6, 1], 16, 2, 64, torch.float32, "cpu")
    for what, table, cu, sl in _bad_places(b):
        with pytest.raises(ValueError):
            paged_append(b.k, b.v, b.k_cache, b.v_cache, table, cu, sl)


@pytest.mark.gpu
def test_append_bad_places_are_reported_and_touch_nothing_else():
    for i in range(7):
        b = Batch([20, 5], [6, 1], 16, 2, 64, torch.float32, DEV)
        what, table, cu, sl = list(_bad_places(b))[i]
        paged_append(b.k, b.v, b.k_cache, b.v_cache, table, cu, sl)
        with pytest.raises(KernelError):
            K.check_status()
        K.check_status()  # the error is reported once
        page, slot = b.place(1, 4)
        assert torch.equal(b.k_cache[page, slot], b.k[6]) and torch.equal(b.v_cache[page, slot], b.v[6]), what
        written = (~torch.isnan(b.k_cache[..., 0, 0])).sum().item()
        # the rows of the first sequence that have a place: positions 14, 15 lie in the good page, 16 .. 19 in the bad one;
        # with a length of 2 only the last two of its six new tokens have a position
        assert written == (1 + 2 if what.startswith("page") or what == "length 2" else 1), what


@pytest.mark.gpu
def test_append_captured_into_a_graph_follows_new_lengths():
    b = Batch([100, 50], [1, 1], 16, 2, 64, torch.bfloat16, DEV, heads=4)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    b.seq_lens.copy_(torch.tensor([98, 48]))
    K.check_status()
    paged_append(b.k, b.v, *b.args(), q=b.q, q_weight=w, k_weight=w, rotary=(64, 10000.0, False))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = paged_append(b.k, b.v, *b.args(), q=b.q, q_weight=w, k_weight=w, rotary=(64, 10000.0, False))
    for step in (99, 100):
        b.seq_lens.copy_(torch.tensor([step, step - 50]))
        graph.replay()
        eager = paged_append(b.k, b.v, *b.args(), q=b.q, q_weight=w, k_weight=w, rotary=(64, 10000.0, False))
        assert torch.equal(q, eager)
    for pos in (97, 98, 99):
        page, slot = b.place(0, pos)
        assert torch.equal(b.v_cache[page, slot], b.v[0])


# ------------------------------------------------------------------------------------------------ attention
def attention_in_64_bits(b, causal, scale, window, q=None):
    """(out, bound): the definition key by key, and the error that the kernel's roundings may leave.

    Per probability: half a step of the 16-bit type (relative), the score's fp32 error - a chain of D products and sums,
    taken with full steps for a tensor core that truncates, times the scale - and 2^-21 for the argument and the
    exponential, twice because it enters sum and quotient; a chain of as many fp32 additions as there are keys; the output
    is rounded once."""
    q = b.q if q is None else q
    kv, d = b.k_cache.shape[2], b.k_cache.shape[3]
    group = q.shape[1] // kv
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    at = 0
    for s, (n, length) in enumerate(zip(b.new, b.lens)):
        places = [b.place(s, j) for j in range(length)]
        page = torch.tensor([x for x, _ in places], dtype=torch.int64, device=q.device)
        slot = torch.tensor([y for _, y in places], dtype=torch.int64, device=q.device)
        for i in range(n):
            pos = length - n + i
            lo = 0 if window is None else max(0, pos - window)
            hi = pos + 1 if causal else (length if window is None else min(length, pos + window + 1))
            if hi <= lo:
                continue
            k = b.k_cache[page[lo:hi], slot[lo:hi]].double()
            v = b.v_cache[page[lo:hi], slot[lo:hi]].double()
            qi = q[at + i].double().view(kv, group, d)
            z = torch.einsum("hgd,jhd->hgj", qi, k) * scale
            size = torch.einsum("hgd,jhd->hgj", qi.abs(), k.abs()).amax(-1, keepdim=True) * scale
            prob = torch.softmax(z, -1)
            out[at + i] = torch.einsum("hgj,jhd->hgd", prob, v).reshape(-1, d)
            w = torch.einsum("hgj,jhd->hgd", prob, v.abs())
            rel = half + 2 * (size * (d + 8) * 2.0 ** -23 + 2.0 ** -21) + (hi - lo) * 2.0 ** -23
            bound[at + i] = (rel * w).reshape(-1, d)
        at += n
    return out, bound + half * (out.abs() + bound) + half * torch.finfo(q.dtype).tiny


ATTENDS = [
    # lens, new, page, heads, kv_heads, dim, window, causal
    ([1], [1], 16, 1, 1, 64, None, True),
    ([5], [1], 16, 4, 4, 64, None, True),
    ([300], [1], 16, 12, 12, 64, None, True),
    ([127, 128, 129, 255, 257], [1] * 5, 16, 8, 2, 128, None, True),
    ([700, 3, 1500], [1, 1, 1], 64, 40, 1, 128, None, True),
    ([3000], [1], 8, 71, 1, 64, None, True),
    ([4100, 17], [2, 1], 128, 4, 2, 128, None, True),
    ([130, 64], [130, 64], 32, 6, 2, 64, None, True),          # whole prompts, group 3
    ([300, 333], [260, 129], 16, 4, 4, 128, None, True),       # chunks that end inside a 128-row tile
    ([600], [300], 256, 8, 8, 32, None, True),
    ([90, 0, 200, 40], [1, 0, 100, 0], 16, 9, 3, 96, None, True),   # sequences without new tokens, one without any
    ([250, 100], [70, 100], 16, 4, 2, 80, None, False),
    ([400, 1000], [200, 1], 32, 4, 2, 64, 100, True),
    ([400, 1000], [200, 3], 32, 2, 2, 128, 0, True),           # a window of the token itself
    ([500], [130], 16, 4, 1, 8, 37, False),
    ([2, 300], [5, 9], 16, 4, 2, 64, None, True),              # more new tokens than the length: rows that see nothing
    ([257] * 40, [1] * 40, 16, 4, 4, 64, None, True),          # more sequences than a warp has lanes
]


def _attend_batch(lens, new, page, heads, kv_heads, dim, dtype, device, **kw):
    b = Batch(lens, new, page, kv_heads, dim, dtype, device, heads=heads, **kw)
    b.fill_history()
    b.q = (1.5 * b.q.float()).to(dtype)
    return b


def _check_attention(b, out, causal, window, scale=None):
    scale = 1.0 / math.sqrt(b.q.shape[2]) if scale is None else scale
    want, bound = attention_in_64_bits(b, causal, scale, window)
    assert torch.isfinite(out).all()
    err = (out.double() - want).abs()
    assert (err <= bound).all(), f"{(err / bound.clamp(min=1e-300)).max().item():.3g} of the bound"


@pytest.mark.parametrize("lens,new,page,heads,kv_heads,dim,window,causal", ATTENDS)
def test_attention_torch_expression(lens, new, page, heads, kv_heads, dim, window, causal):
    b = _attend_batch(lens, new, page, heads, kv_heads, dim, torch.float64, "cpu", spare_rows=2)
    out = paged_attention(b.q, *b.args(), causal=causal, window=window)
    want, _ = attention_in_64_bits(b, causal, 1.0 / math.sqrt(dim), window)
    assert torch.allclose(out, want, rtol=1e-9, atol=1e-9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,page,heads,kv_heads,dim,window,causal", ATTENDS)
def test_attention_kernel(lens, new, page, heads, kv_heads, dim, window, causal, dtype):
    b = _attend_batch(lens, new, page, heads, kv_heads, dim, dtype, DEV, spare_rows=2)
    out = paged_attention(b.q, *b.args(), causal=causal, window=window)
    K.check_status()
    _check_attention(b, out, causal, window)
    again = paged_attention(b.q, *b.args(), causal=causal, window=window)
    assert torch.equal(out, again)


def _attention_refused(device, dtype):
    b = _attend_batch([20, 5], [4, 1], 16, 4, 2, 64, dtype, device)
    paged_attention(b.q, *b.args())
    kc, vc, table, cu, sl = b.args()
    bad = [
        lambda: paged_attention(b.q[:, :3], *b.args()),
        lambda: paged_attention(b.q[..., :32], *b.args()),
        lambda: paged_attention(b.q.double().float(), kc.double(), vc.double(), table, cu, sl),
        lambda: paged_attention(b.q, kc, vc[:, :8], table, cu, sl),
        lambda: paged_attention(b.q, kc[:, :12], vc[:, :12], table, cu, sl),
        lambda: paged_attention(b.q, kc, vc, table.long(), cu, sl),
        lambda: paged_attention(b.q, kc, vc, table, cu[:2], sl),
        lambda: paged_attention(b.q, *b.args(), scale=0.0),
        lambda: paged_attention(b.q, *b.args(), scale=float("nan")),
        lambda: paged_attention(b.q, *b.args(), scale=-1.0),
        lambda: paged_attention(b.q, *b.args(), window=-2),
        lambda: paged_attention(b.q, *b.args(), out=b.q[:3]),
        lambda: paged_attention(b.q, *b.args(), out=b.q.double()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KernelError):
        paged_attention(b.q.requires_grad_(), *b.args())
    with torch.no_grad():
        paged_attention(b.q, *b.args())


def test_attention_refusals():
    _attention_refused("cpu", torch.float32)


@pytest.mark.gpu
def test_attention_gpu_refusals():
    _attention_refused(DEV, torch.bfloat16)
    for dtype, page, dim in ((torch.float32, 16, 64), (torch.bfloat16, 4, 64), (torch.bfloat16, 16, 68), (torch.bfloat16, 16, 136)):
        b = Batch([20], [1], page, 1, dim, dtype, DEV)
        with pytest.raises(KernelError):
            paged_attention(b.q, *b.args())
    b = Batch([20], [1], 16, 1, 64, torch.bfloat16, DEV)
    wide = torch.zeros(*b.k_cache.shape[:3], 65, dtype=torch.bfloat16, device=DEV)[..., :64]
    with pytest.raises(KernelError):
        paged_attention(b.q, wide, b.v_cache, b.table, b.cu, b.seq_lens)


def test_attention_bad_pages_on_the_cpu():
    b = _attend_batch([20, 5], [6, 1], 16, 2, 2, 64, torch.float32, "cpu")
    kc, vc, table, cu, sl = b.args()
    for bad in (-1, kc.shape[0]):
        t = table.clone()
        t[0, 0] = bad
        with pytest.raises(ValueError):
            paged_attention(b.q, kc, vc, t, cu, sl)
    s = sl.clone()
    s[1] = 10 ** 6
    with pytest.raises(ValueError):
        paged_attention(b.q, kc, vc, table, cu, s)


@pytest.mark.gpu
def test_attention_bad_pages_are_reported_and_leave_other_sequences_alone():
    b = _attend_batch([200, 150], [6, 3], 16, 4, 2, 64, torch.bfloat16, DEV)
    good = paged_attention(b.q, *b.args())
    K.check_status()
    kc, vc, table, cu, sl = b.args()
    for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 3] = bad
        out = paged_attention(b.q, kc, vc, t, cu, sl)
        with pytest.raises(KernelError):
            K.check_status()
        assert torch.equal(out[6:], good[6:])
        # the same entry outside every query's window is not looked at
        near = paged_attention(b.q, kc, vc, t, cu, sl, window=90)
        K.check_status()
        assert torch.equal(near, paged_attention(b.q, kc, vc, table, cu, sl, window=90))
    for length in (10 ** 6, -4):
        s = sl.clone()
        s[0] = length
        out = paged_attention(b.q, kc, vc, table, cu, s)
        with pytest.raises(KernelError):
            K.check_status()
        want, bound = attention_in_64_bits(b, True, 0.125, None)  # another length: the work is cut at other places
        assert ((out.double() - want).abs() <= bound)[6:9].all()


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_and_given_outputs():
    b = _attend_batch([50, 300], [3, 140], 16, 4, 2, 64, torch.float16, DEV, spare_rows=5)
    plain = paged_attention(b.q, *b.args())
    assert torch.count_nonzero(plain[b.tokens:]) == 0
    wide = torch.full((b.q.shape[0], 6, 72), 7.0, dtype=torch.float16, device=DEV)
    out = paged_attention(b.q, *b.args(), out=wide[:, 1:5, :64])
    assert out.data_ptr() == wide[:, 1:5].data_ptr()
    assert torch.equal(out[:b.tokens], plain[:b.tokens])
    assert (wide[b.tokens:] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 5] == 7).all() and (wide[..., 64:] == 7).all()
    # no sequence at all
    none = paged_attention(b.q, b.k_cache, b.v_cache, b.table[:0], b.cu[:1], b.seq_lens[:0])
    assert torch.count_nonzero(none) == 0
    K.check_status()


@pytest.mark.gpu
def test_views_joint_caches_and_odd_query_strides():
    b = _attend_batch([90, 700], [1, 33], 32, 8, 2, 64, torch.bfloat16, DEV, joint=True)
    _check_attention(b, paged_attention(b.q, *b.args()), True, None)
    want = paged_attention(b.q, *b.args())
    odd = torch.zeros(b.q.shape[0], 8, 67, dtype=torch.bfloat16, device=DEV)
    odd[..., 3:] = b.q
    assert torch.equal(paged_attention(odd[..., 3:], *b.args()), want)
    turned = b.q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(paged_attention(turned, *b.args()), want)


@pytest.mark.gpu
def test_scores_far_apart_and_growing():
    """Scores of hundreds, growing along the sequence, so that the running reference moves at every tile."""
    for sign in (1.0, -1.0):
        b = _attend_batch([1500, 900], [200, 1], 16, 4, 2, 128, torch.bfloat16, DEV)
        for s, length in enumerate(b.lens):
            for j in range(length):
                page, slot = b.place(s, j)
                b.k_cache[page, slot] = sign * (j / 40.0) / 16.0
        b.q.fill_(1.0)
        out = paged_attention(b.q, *b.args(), scale=1.0)
        _check_attention(b, out, True, None, scale=1.0)


@pytest.mark.gpu
def test_attention_captured_into_a_graph_follows_lengths_tables_and_queries():
    b = _attend_batch([2000, 333, 80], [1, 1, 1], 16, 8, 2, 128, torch.bfloat16, DEV)
    args = b.args()
    paged_attention(b.q, *args)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_attention(b.q, *args))
        graphs.append(g)
    side = torch.cuda.Stream()
    for lens in ([2000, 333, 80], [17, 1, 64], [1999, 332, 79]):
        b.seq_lens.copy_(torch.tensor(lens))
        b.q.mul_(0.9)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):  # two calls at once: each graph has a workspace of its own
            graphs[1].replay()
        torch.cuda.synchronize()
        eager = paged_attention(b.q, *args)
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)


@pytest.mark.gpu
def test_cache_offsets_beyond_32_bits():
    pages = 2 ** 31 // (64 * 2 * 128) + 40  # the last pages start past 2^31 elements
    kc = torch.zeros(pages, 64, 2, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    b = Batch([150], [3], 64, 2, 128, torch.bfloat16, DEV, heads=4)
    last = torch.tensor([[pages - 1, pages - 5, pages - 2]], dtype=torch.int32, device=DEV)
    b.table, b.table_cpu, b.k_cache, b.v_cache = last, last.cpu(), kc, vc
    g = torch.Generator().manual_seed(3)
    for j in last[0].tolist():
        kc[j] = torch.randn(64, 2, 128, generator=g)
        vc[j] = torch.randn(64, 2, 128, generator=g)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    q = paged_append(b.k, b.v, *b.args(), q=b.q, q_weight=w, k_weight=w, rotary=(128, 10000.0, False))
    page, slot = b.place(0, 149)
    assert torch.equal(vc[page, slot], b.v[2])
    b.q = q
    _check_attention(b, paged_attention(q, *b.args()), True, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,heads,kv_heads,window", [(64, 12, 12, None), (128, 8, 2, None), (64, 8, 1, 60)])
def test_prompt_in_chunks_then_tokens_equals_one_pass(dim, heads, kv_heads, window):
    """Append and attend chunk by chunk and token by token, against the whole sequence at once in 64 bits."""
    dtype, page, total = torch.bfloat16, 16, 400
    g = torch.Generator().manual_seed(5)
    lens = [total, 290]
    x = [[torch.randn(n, h, dim, generator=g).to(dtype).to(DEV) for h in (heads, kv_heads, kv_heads)] for n in lens]
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(DEV) for _ in range(2))
    whole = Batch(lens, lens, page, kv_heads, dim, dtype, DEV, heads=heads)
    rotary = (dim, 10000.0, False)
    outs = [[], []]
    done = [0, 0]
    for chunk in (250, 39, 1, 1, 109):
        new = [min(chunk, n - d) for n, d in zip(lens, done)]
        starts = list(done)
        done = [d + n for d, n in zip(done, new)]
        cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=DEV)
        sl = torch.tensor(done, dtype=torch.int32, device=DEV)
        q, k, v = (torch.cat([x[s][c][starts[s]:done[s]] for s in range(2)]) for c in range(3))
        q = paged_append(k, v, whole.k_cache, whole.v_cache, whole.table, cu, sl, q=q, q_weight=wq, k_weight=wk, rotary=rotary)
        o = paged_attention(q, whole.k_cache, whole.v_cache, whole.table, cu, sl, window=window)
        outs[0].append(o[:new[0]])
        outs[1].append(o[new[0]:])
    K.check_status()
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    qn, _ = K.qk_norm_rope(torch.cat([x[0][0], x[1][0]]), torch.cat([x[0][1], x[1][1]]), wq, wk, positions=pos, rotary=rotary)
    whole.q = qn
    _check_attention(whole, torch.cat(outs[0] + outs[1]), True, window)


def _rows_that_are_not_numbers(device, dtype):
    """A query of NaN beside one that sees nothing, in a short sequence, a long one that is cut into parts, and a chunk."""
    b = _attend_batch([20, 3000, 2], [1, 1, 5], 16, 4, 2, 64, dtype, device)
    b.q[0] = float("nan")
    b.q[1, 3] = float("nan")
    return b


def _check_rows_that_are_not_numbers(b):
    out = paged_attention(b.q, *b.args())
    assert torch.isnan(out[0]).all() and torch.isnan(out[1, 3]).all()
    assert torch.count_nonzero(out[2:5]) == 0  # three more new tokens than the sequence has
    clean = b.q.nan_to_num(0.0)
    want, bound = attention_in_64_bits(b, True, 0.125, None, q=clean)
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device=out.device)
    keep[0], keep[1, 3] = False, False
    assert ((out.double() - want).abs() <= bound)[keep].all()


def test_bad_queries_stay_alone_in_the_torch_expression():
    _check_rows_that_are_not_numbers(_rows_that_are_not_numbers("cpu", torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("more", [False, True])
def test_bad_queries_stay_alone(more):
    b = _rows_that_are_not_numbers(DEV, torch.bfloat16)
    _check_rows_that_are_not_numbers(b)
    if more:  # in a chunk's rows
        b = _attend_batch([700], [300], 16, 4, 2, 64, torch.bfloat16, DEV)
        want = paged_attention(b.q, *b.args())
        b.q[100] = float("nan")
        out = paged_attention(b.q, *b.args())
        assert torch.isnan(out[100]).all()
        keep = torch.arange(300, device=DEV) != 100
        assert torch.equal(out[keep], want[keep])


def test_outputs_whose_rows_share_memory_are_refused():
    b = _attend_batch([20], [4], 16, 4, 2, 64, torch.bfloat16, "cpu")
    shared = torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(4, 4, 64)
    with pytest.raises(ValueError, match="share memory"):
        paged_attention(b.q, *b.args(), out=shared)
    with pytest.raises(KernelError, match="no backward"):
        paged_attention(b.q, *b.args(), out=torch.zeros_like(b.q).requires_grad_())


@pytest.mark.gpu
def test_rows_before_the_first_sequence():
    b = _attend_batch([50, 300], [3, 140], 16, 4, 2, 64, torch.bfloat16, DEV, spare_rows=9)
    want = paged_attention(b.q, *b.args())
    cu = b.cu + 7
    moved = torch.cat((b.q[-7:], b.q[:-7]))
    for _ in range(3):  # memory of earlier results is reused
        garbage = torch.full_like(moved, float("nan"))
        del garbage
        out = paged_attention(moved, b.k_cache, b.v_cache, b.table, cu, b.seq_lens)
        assert torch.count_nonzero(out[:7]) == 0 and torch.count_nonzero(out[7 + b.tokens:]) == 0
        assert torch.equal(out[7:7 + b.tokens], want[:b.tokens])
        del out
    K.check_status()


@pytest.mark.gpu
def test_queries_off_the_16_byte_boundary_and_in_the_place_of_the_output():
    b = _attend_batch([50, 300, 4000], [3, 140, 1], 16, 4, 2, 64, torch.bfloat16, DEV)
    want = paged_attention(b.q, *b.args())
    flat = torch.zeros(b.q.numel() + 4, dtype=torch.bfloat16, device=DEV)
    off = flat[4:].view(b.q.shape)
    off.copy_(b.q)
    assert off.is_contiguous() and off.data_ptr() % 16
    assert torch.equal(paged_attention(off, *b.args()), want)
    q = b.q.clone()
    assert paged_attention(q, *b.args(), out=q) is q
    assert torch.equal(q, want)


@pytest.mark.gpu
def test_more_work_than_32_bits_of_tiles_is_refused():
    """Prompts of a million tokens with 64 heads over one KV head: the lengths on the work line add up to more than 2^31."""
    cache = torch.zeros(1, 128, 1, 8, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(1, 2 ** 14, dtype=torch.int32, device=DEV)
    q = torch.zeros(2 ** 20, 64, 8, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, 2 ** 20], dtype=torch.int32, device=DEV)
    lens = torch.tensor([2 ** 21], dtype=torch.int32, device=DEV)
    K.check_status()
    paged_attention(q, cache, cache, table, cu, lens)
    with pytest.raises(KernelError, match="size"):
        K.check_status()
    K.check_status()


@pytest.mark.gpu
def test_page_tables_of_too_many_positions_are_refused():
    cache = torch.zeros(1, 128, 1, 8, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(1, 1, 8, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    lens = torch.tensor([5], dtype=torch.int32, device=DEV)
    paged_attention(q, cache, cache, torch.zeros(1, 2 ** 19, dtype=torch.int32, device=DEV), cu, lens)
    with pytest.raises(KernelError):
        paged_attention(q, cache, cache, torch.zeros(1, 2 ** 19 + 1, dtype=torch.int32, device=DEV), cu, lens)
    K.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 255, 256, 257, 513, 1000])
def test_append_of_many_sequences(batch):
    """Sequences with none to three new tokens, some of them empty: each token finds its own sequence."""
    rng = random.Random(batch)
    new = [rng.choice([0, 0, 1, 1, 2, 3]) for _ in range(batch)]
    lens = [n + rng.choice([0, 1, 15, 16, 40]) for n in new]
    if sum(new) == 0:
        new[0], lens[0] = 2, 20
    b = Batch(lens, new, 16, 1, 16, torch.float32, DEV, heads=2, spare_rows=4, fill=0.0)
    q = paged_append(b.k, b.v, *b.args(), q=b.q)
    want_k, want_v = torch.zeros_like(b.k_cache), torch.zeros_like(b.v_cache)
    for t, (s, pos) in enumerate(b.positions()):
        page, slot = b.place(s, pos)
        want_k[page, slot], want_v[page, slot] = b.k[t], b.v[t]
    assert torch.equal(b.k_cache, want_k) and torch.equal(b.v_cache, want_v)
    assert torch.equal(q[:b.tokens], b.q[:b.tokens]) and torch.count_nonzero(q[b.tokens:]) == 0
    K.check_status()


def _optimizer():
    from scaling_b200.core.nn.parameter_meta import CoreParameterMeta
    from scaling_b200.core.optimizer import (LearningRateSchedulerConfig, Optimizer, OptimizerConfig, OptimizerParamGroup,
                                             OptimizerParamGroupConfig)
    from scaling_b200.parallel import Topology, TopologyConfig

    topology = Topology(TopologyConfig.from_dict({
        "world_size": 1, "model_parallel_size": 1, "pipe_parallel_size": 1, "global_rank": 0, "local_slot": 0,
        "micro_batch_size": 1, "gradient_accumulation_steps": 1}))
    p = torch.nn.Parameter(torch.ones(64, device=DEV))
    CoreParameterMeta.register_on_parameter(p, is_model_parallel=False, layer_index=0, parameter_name="w")
    group = OptimizerParamGroup([("w", p, p.core_parameter_meta)], OptimizerParamGroupConfig(
        name="g", weight_decay=0.0, learning_rate_scheduler=LearningRateSchedulerConfig(
            learning_rate=0.1, learning_rate_decay_style="constant")))
    return p, Optimizer(OptimizerConfig(zero=False), [group], topology)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["append", "page", "length"])
def test_bad_places_do_not_reach_the_optimizer(what):
    """An error in a table or a length belongs to its call: the next optimizer step is taken, the error is still raised."""
    K.check_status()
    b = _attend_batch([200, 150], [6, 3], 16, 4, 2, 64, torch.bfloat16, DEV)
    kc, vc, table, cu, sl = b.args()
    p, opt = _optimizer()
    if what == "append":
        paged_append(b.k, b.v, kc, vc, table, cu, torch.full_like(sl, -3))
    elif what == "page":
        table[0, 3] = kc.shape[0]
        paged_attention(b.q, kc, vc, table, cu, sl)
    else:
        sl[0] = 10 ** 6
        paged_attention(b.q, kc, vc, table, cu, sl)
    before = p.detach().clone()
    p.grad.fill_(1.0)
    out = opt.step()
    assert not out.overflow and not torch.equal(p.detach(), before)
    with pytest.raises(KernelError):
        K.check_status()
    K.check_status()


@pytest.mark.gpu
def test_errors_outlast_replays_where_the_first_call_was_captured(monkeypatch):
    """The status words are made by the first call: inside a capture, too, they belong to no graph."""
    b = Batch([20, 5], [6, 1], 16, 2, 64, torch.bfloat16, DEV)
    paged_append(b.k, b.v, *b.args())
    K.check_status()
    monkeypatch.setattr(K, "_STATUS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_append(b.k, b.v, *b.args())
    K.check_status()
    good = b.table.clone()
    b.table[0, 1] = -1
    graph.replay()
    b.table.copy_(good)
    graph.replay()  # a good call does not take the error back
    with pytest.raises(KernelError):
        K.check_status()
    graph.replay()
    K.check_status()


@pytest.mark.gpu
def test_long_prompts_are_taken_beside_many_sequences_as_alone():
    """2^19 tokens with 16 heads per KV head: some 2^26 products of 256 rows with 128 keys, far below 2^31.  Sequences
    without new tokens do not change where the work is cut, so the outputs are equal bit by bit."""
    n, heads = 2 ** 19, 16
    g = torch.Generator(device=DEV).manual_seed(3)
    kc, vc = (torch.randn(1, 128, 1, 8, generator=g, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(n, heads, 8, generator=g, device=DEV).bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    K.check_status()
    outs = []
    for others in (0, 32):
        table = torch.zeros(1 + others, n // 128, dtype=torch.int32, device=DEV)
        outs.append(paged_attention(q, kc, vc, table, ints([0] + [n] * (1 + others)), ints([n] + [5] * others)))
        K.check_status()
    assert torch.equal(outs[0], outs[1])
    for i in (0, 1, 127, 128, 300, n - 1):  # every page is the same one: position j has key j % 128
        seen = torch.arange(i + 1, device=DEV)
        count = torch.bincount(seen % 128, minlength=128).double()
        k, v = kc[0, :, 0].double(), vc[0, :, 0].double()
        z = q[i].double() @ k.t() / 8 ** 0.5
        p = torch.exp(z - z.amax(-1, keepdim=True)) * count
        want = p @ v / p.sum(-1, keepdim=True)
        # as in attention_in_64_bits; the chain of additions has at most (i + 1) links of 2^-24 on average, full steps here
        size = (q[i].double().abs() @ k.abs().t()).amax(-1, keepdim=True) / 8 ** 0.5
        rel = 2.0 ** -8 + 2 * (size * 16 * 2.0 ** -23 + 2.0 ** -21) + (i + 1) * 2.0 ** -23
        w = p @ v.abs() / p.sum(-1, keepdim=True)
        assert ((outs[0][i].double() - want).abs() <= rel * w + 2.0 ** -8 * (want.abs() + rel * w)).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
def test_a_refused_call_leaves_zeros(given):
    """Lengths that add up to more than 2^31: nothing of what the memory held before is in the output."""
    n, heads, spare = 2 ** 20, 64, 3
    cache = torch.ones(1, 128, 1, 8, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(n + spare, heads, 8, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(1, 2 ** 14, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    lens = torch.tensor([2 ** 21], dtype=torch.int32, device=DEV)
    K.check_status()
    out = torch.full_like(q, 7.0)
    if not given:
        del out  # its memory is given to the call's result
    out = paged_attention(q, cache, cache, table, cu, lens, out=out if given else None)
    with pytest.raises(KernelError, match="size"):
        K.check_status()
    assert torch.count_nonzero(out[:n]) == 0
    assert (out[n:] == (7 if given else 0)).all()


WRONG_ROWS = [[0, 4, 9], [0, 8, 6], [-2, 3, 7], [3, 1, 7]]  # of two sequences in seven rows


@pytest.mark.parametrize("cu", WRONG_ROWS)
def test_rows_that_do_not_follow_one_another_on_the_cpu(cu):
    b = _attend_batch([20, 30], [4, 3], 16, 2, 2, 64, torch.float32, "cpu")
    kc, vc, table, _, sl = b.args()
    wrong = torch.tensor(cu, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged_append(b.k, b.v, kc, vc, table, wrong, sl)
    with pytest.raises(ValueError):
        paged_attention(b.q, kc, vc, table, wrong, sl)


@pytest.mark.gpu
@pytest.mark.parametrize("others", [0, 300])
@pytest.mark.parametrize("cu", WRONG_ROWS)
def test_rows_that_do_not_follow_one_another_are_reported(cu, others):
    b = _attend_batch([20, 30] + [9] * others, [4, 3] + [0] * others, 16, 2, 2, 64, torch.bfloat16, DEV)
    kc, vc, table, good, sl = b.args()
    last = max(cu[2], 0)
    wrong = torch.tensor(cu + [last] * others, dtype=torch.int32, device=DEV)
    for call in (lambda c: paged_append(b.k, b.v, kc, vc, table, c, sl), lambda c: paged_attention(b.q, kc, vc, table, c, sl)):
        call(wrong)
        with pytest.raises(KernelError):
            K.check_status()
        call(good)
        K.check_status()


def test_written_tensors_whose_elements_share_memory_are_refused():
    b = _attend_batch([20], [4], 16, 4, 2, 64, torch.bfloat16, "cpu")
    kc, vc, table, cu, sl = b.args()
    flat = torch.zeros(kc.numel(), dtype=torch.bfloat16)
    for shared in (kc[:, :, :1].expand(kc.shape), kc[:1].expand(kc.shape), flat.as_strided(kc.shape, (64, 64, 64, 1)),
                   flat.as_strided(kc.shape, (16 * 128 - 64, 128, 64, 1))):
        for caches in ((shared, vc), (kc, shared)):
            with pytest.raises(ValueError, match="share memory"):
                paged_append(b.k, b.v, *caches, table, cu, sl)
        paged_attention(b.q, shared, vc, table, cu, sl)  # caches that are read only may be any view
    with pytest.raises(ValueError, match="share memory"):
        paged_attention(b.q, *b.args(), out=flat.as_strided((4, 4, 64), (128, 64, 1)))
    # layouts in use: pages of keys and values side by side, heads before tokens, more columns than the head has
    for view in (torch.zeros(kc.shape[0], 2, *kc.shape[1:], dtype=torch.bfloat16)[:, 0],
                 torch.zeros(kc.shape[0], 2, 16, 64, dtype=torch.bfloat16).transpose(1, 2),
                 torch.zeros(*kc.shape[:3], 72, dtype=torch.bfloat16)[..., :64],
                 torch.zeros(kc.shape[0], 16, 2, 2, 64, dtype=torch.bfloat16)[:, :, :, 1]):
        paged_append(b.k, b.v, view, view.clone(), table, cu, sl)


def _many(batch, kind, seed):
    """(lens, new) of more sequences than a warp has lanes: the work is found by groups of 32 of them."""
    rng = random.Random(seed)
    long = lambda: rng.choice([0, 1, 15, 127, 128, 129, 640, 1500, rng.randrange(3500)])  # noqa: E731
    if kind == "tokens":  # one new token each
        new = [1] * batch
    elif kind == "mixed":  # single tokens, a few tokens, chunks of more than 64 rows
        new = [rng.choice([1, 1, 1, 2, 5, 17, 40, 90]) if b % 3 else 1 for b in range(batch)]
    else:  # runs of sequences without new tokens, longer than a group, between the others
        new = [rng.choice([1, 3, 30]) if b in (2, batch // 2, batch - 1) else 0 for b in range(batch)]
    lens = [n + long() for n in new]
    lens[rng.randrange(batch)] = 3600  # the table is wider than the plan for short ones takes
    return lens, new


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim,window", [(4, 1, 64, None), (4, 2, 128, None), (6, 2, 64, 700)])
@pytest.mark.parametrize("kind", ["tokens", "mixed", "runs"])
@pytest.mark.parametrize("batch", [33, 64, 100])
def test_more_sequences_than_lanes_with_divided_items(batch, kind, heads, kv_heads, dim, window):
    lens, new = _many(batch, kind, batch)
    b = _attend_batch(lens, new, 16, heads, kv_heads, dim, torch.bfloat16, DEV)
    out = paged_attention(b.q, *b.args(), window=window)
    K.check_status()
    _check_attention(b, out, True, window)
    assert torch.equal(out, paged_attention(b.q, *b.args(), window=window))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_captured_chunks_and_tokens_follow_new_lengths(dim):
    """Both kernels and the joining of parts in one graph, replayed with other lengths, offsets and tables."""
    lens, new = _many(40, "mixed", 5)
    b = _attend_batch(lens, new, 16, 4, 1, dim, torch.bfloat16, DEV)
    paged_attention(b.q, *b.args())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(b.q, *b.args())
    full = b.seq_lens.clone()
    half = torch.tensor([max(n, length // 2) for n, length in zip(new, lens)], dtype=torch.int32, device=DEV)
    turned = torch.tensor([0] + new[::-1], device=DEV).cumsum(0).to(torch.int32)
    for lengths, cu, table in ((full, b.cu, b.table), (half, b.cu, b.table), (full.flip(0), turned, b.table.flip(0))):
        args = (b.k_cache, b.v_cache, table.clone(), cu.clone(), lengths.clone())
        want = paged_attention(b.q, *args)
        keep = [t.clone() for t in (b.table, b.cu, b.seq_lens)]
        b.table.copy_(args[2]), b.cu.copy_(args[3]), b.seq_lens.copy_(args[4])
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)
        b.table.copy_(keep[0]), b.cu.copy_(keep[1]), b.seq_lens.copy_(keep[2])
    K.check_status()
    _check_attention(b, paged_attention(b.q, *b.args()), True, None)


@pytest.mark.gpu
@pytest.mark.parametrize("sms", [1, 7, 40])
def test_work_shared_out_over_fewer_multiprocessors(sms, monkeypatch):
    from scaling_b200.ops import paged_attention as module

    monkeypatch.setattr(module, "sm_count", lambda: sms)
    for lens, new in (([3000, 900], [1, 1]), ([3000, 900, 5], [200, 1, 5])):
        b = _attend_batch(lens, new, 16, 8, 2, 128, torch.bfloat16, DEV)
        _check_attention(b, paged_attention(b.q, *b.args()), True, None)
    K.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("length,new,heads,dim", [(2 ** 22, 1, 1, 64), (2 ** 22 + 77, 2, 20, 128),   # narrow, 1 and 40 rows
                                                  (2 ** 26, 1, 1, 64),                                # the longest table
                                                  (2 ** 20 - 3, 20, 4, 128),                          # wide, 80 rows
                                                  (2 ** 20 + 130, 40, 4, 64), (2 ** 20, 65, 4, 128)])  # 160 and 260 rows
def test_long_contexts_in_one_piece(length, new, heads, dim, monkeypatch):
    """One CTA adds up millions of keys: the sums are as exact as those of 2^14 keys.  Positions share pages, so that a key's
    weight is multiplied by how often it is seen; later keys have larger scores, so that the references move."""
    from scaling_b200.ops import paged_attention as module

    monkeypatch.setattr(module, "sm_count", lambda: 1)
    dtype, page, pages = torch.float16, 128, 48
    g = torch.Generator().manual_seed(length)
    kc = torch.randn(pages, page, 1, dim, generator=g)
    vc = 1.0 + 0.5 * torch.randn(pages, page, 1, dim, generator=g)
    kc[pages // 2:] *= 2.0
    kc, vc = (t.to(dtype).to(DEV) for t in (kc, vc))
    cols = -(-length // page)
    table = torch.arange(cols) % (pages // 2)
    table[cols // 2:] += pages // 2
    table = table.int().to(DEV)
    q = (1.5 * torch.randn(new, heads, dim, generator=g)).to(dtype).to(DEV)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    out = paged_attention(q, kc, vc, table[None], ints(0, new), ints(length))
    K.check_status()
    position = torch.arange(length, device=DEV)
    key = table[position // page].long() * page + position % page
    k, v = kc.reshape(-1, dim).double(), vc.reshape(-1, dim).double()
    half, scale = torch.finfo(dtype).eps / 2, dim ** -0.5
    for i in range(new):
        count = torch.bincount(key[:length - new + i + 1], minlength=pages * page).double()
        z = q[i].double() @ k.t() * scale
        w = torch.exp(z - z.amax(-1, keepdim=True)) * count
        w /= w.sum(-1, keepdim=True)
        want = w @ v
        # as in attention_in_64_bits, with chains of 2^14 additions, and of one rounded addition for each of these
        size = (q[i].double().abs() @ k.abs().t()).amax(-1, keepdim=True) * scale
        rel = half + 2 * (size * (dim + 8) * 2.0 ** -23 + 2.0 ** -21) + 2 ** 14 * 2.0 ** -23 + length / 2 ** 14 * 2.0 ** -24
        bound = rel * (w @ v.abs())
        bound += half * (want.abs() + bound)
        err = (out[i].double() - want).abs()
        assert (err <= bound).all(), f"{(err / bound).max().item():.3g} of the bound"


FIRST_CALL = '''
import torch
from scaling_b200.ops import functional as K
from scaling_b200.ops.paged_attention import paged_append, paged_attention

make = lambda *shape: torch.randn(*shape, device="cuda").bfloat16()
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
q, k, v, w, kc, vc = make(3, 4, 64), make(3, 2, 64), make(3, 2, 64), make(64), make(4, 16, 2, 64), make(4, 16, 2, 64)
cache = (kc, vc, ints(0, 1, 2)[None], ints(0, 3), ints(20))
rotary = dict(positions=ints(17, 18, 19), rotary=(64, 10000.0, False))
leaves = [t.clone().requires_grad_() for t in (q, k, w)]


def step():
    outs = K.qk_norm_rope(*leaves, leaves[2], **rotary)
    return outs[0].detach(), *torch.autograd.grad(outs, leaves, (q, k))


calls = {"append": lambda: (paged_append(k, v, *cache, q=q), kc.clone()), "attend": lambda: (paged_attention(q, *cache),),
         "norm": lambda: K.qk_norm_rope(q, k, w, w, **rotary), "step": step}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls["WHICH"]()
graph.replay()
K.check_status()
assert all(torch.equal(a, b) for a, b in zip(got, calls["WHICH"]()))
print("FIRST-CALL-OK")
'''


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["append", "attend", "norm", "step"])
def test_the_first_call_of_a_process_inside_a_capture(which):
    """Loading the library, binding the thread and making the status words are no part of the graph and do not break it."""
    import subprocess
    import sys
    from pathlib import Path

    res = subprocess.run([sys.executable, "-c", FIRST_CALL.replace("WHICH", which)], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent, timeout=300)
    assert res.returncode == 0 and "FIRST-CALL-OK" in res.stdout, res.stderr[-3000:]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (12, 12, 64)])
def test_chunks_with_many_items_per_multiprocessor(heads, kv_heads, dim):
    """Long chunks of many heads behind long contexts: every CTA takes several items of many tiles, most of them divided."""
    b = _attend_batch([6000, 4100], [1000, 700], 64, heads, kv_heads, dim, torch.bfloat16, DEV)
    out = paged_attention(b.q, *b.args())
    K.check_status()
    _check_attention(b, out, True, None)
