"""Workloads of three attention operators: per-head norm and rotation of queries and keys, the write of new tokens
into a paged key/value cache, and attention of new tokens over that cache.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges.  ``prepare`` makes what a program holds
before the call, ``run`` makes one pass: with ``own`` false from elementary torch operations in 32 bits (angles in 64),
with ``own`` true through the package's entry points.  ``exact`` evaluates the definition in 64 bits.

Layouts: tokens first, ``[tokens, heads, head_dim]``; caches ``[pages, page_size, kv_heads, head_dim]``; sequence ``b`` of
a call has its new tokens in rows ``cu_seqlens[b] : cu_seqlens[b + 1]``, holds ``seq_lens[b]`` tokens in all (the new ones
are its last), and position ``p`` of it lies in row ``p % page_size`` of page ``page_table[b, p // page_size]``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed() -> list[dict]:
    return [
        # one token of a request that decodes alone, heads of the 7B decoder
        dict(name="norm_rope_one_token", op="norm_rope", train=False, tokens=1, heads=32, kv_heads=8, dim=128,
             dtype="bf16", rms=True, rot=128, interleaved=True, base=10000.0, packed=False, start=1500),
        # training step of the 125M decoder: micro batch 8 x 2048, packed projection, layer norm with bias
        dict(name="norm_rope_train_125m", op="norm_rope", train=True, tokens=16384, heads=12, kv_heads=12, dim=64,
             dtype="bf16", rms=False, rot=64, interleaved=False, base=10000.0, packed=True, start=0),
        # training step of the 7B decoder: two sequences of 4096, separate projections, eight kv heads
        dict(name="norm_rope_train_7b", op="norm_rope", train=True, tokens=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", rms=True, rot=128, interleaved=True, base=10000.0, packed=False, start=0),
        # 32-bit run with one kv head, an odd token count, a head size between the usual ones, a quarter rotated
        dict(name="norm_rope_train_odd", op="norm_rope", train=True, tokens=2999, heads=40, kv_heads=1, dim=80,
             dtype="fp32", rms=False, rot=20, interleaved=False, base=500000.0, packed=False, start=100000),
        # one decoding step of 64 requests
        dict(name="append_decode", op="append", batch=64, new=1, least_new=1, context=4000, least_context=100,
             mix=1, heads=32, kv_heads=8,
             dim=128, page=16, dtype="bf16", norm="rms", rot=128, interleaved=True, base=10000.0),
        # chunks of four prompts, one kv head
        dict(name="append_chunk", op="append", batch=4, new=2048, least_new=500, context=6000, least_context=0,
             mix=2, heads=40, kv_heads=1,
             dim=128, page=64, dtype="bf16", norm="layer", rot=64, interleaved=False, base=10000.0),
        # ragged prompts of a small fp16 model without norms
        dict(name="append_ragged", op="append", batch=33, new=400, least_new=1, context=1500, least_context=0,
             mix=3, heads=12, kv_heads=12,
             dim=64, page=16, dtype="fp16", norm="none", rot=64, interleaved=False, base=10000.0),
        # one short request of the 125M decoder, the next token: latency
        dict(name="attend_one_request", op="attend", batch=1, new=1, least_new=1, context=300, least_context=300,
             mix=4, heads=12,
             kv_heads=12, dim=64, page=16, dtype="bf16", window=-1),
        # one decoding step of 64 requests of the 7B decoder
        dict(name="attend_decode", op="attend", batch=64, new=1, least_new=1, context=8000, least_context=500,
             mix=5, heads=32, kv_heads=8,
             dim=128, page=16, dtype="bf16", window=-1),
        # one decoding step of two requests with very long contexts, one kv head
        dict(name="attend_decode_long", op="attend", batch=2, new=1, least_new=1, context=130000, least_context=90000,
             mix=6, heads=40,
             kv_heads=1, dim=128, page=64, dtype="bf16", window=-1),
        # chunks of two long prompts of the 7B decoder
        dict(name="attend_chunk", op="attend", batch=2, new=2048, least_new=2048, context=8192, least_context=2000,
             mix=7, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", window=-1),
        # prompts and decoding requests in one call, local attention, fp16
        dict(name="attend_mixed", op="attend", batch=24, new=300, least_new=1, context=5000, least_context=0,
             mix=8, heads=12, kv_heads=12,
             dim=64, page=32, dtype="fp16", window=1024),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["norm_rope", "append", "attend", "attend"])
    heads, kv = rng.choice([(12, 12), (32, 8), (32, 32), (40, 1), (40, 8), (16, 2), (6, 3), (9, 3), (71, 1)])
    if op == "norm_rope":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        cap = max(1, min(16384, 42_000_000 // ((heads + kv) * dim)))
        return dict(op=op, train=rng.random() < 0.7, tokens=_log_int(rng, 1, cap), heads=heads, kv_heads=kv, dim=dim,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rms=rng.random() < 0.5,
                    rot=rng.choice([0, dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    base=rng.choice([10000.0, 500000.0]), packed=heads == kv and rng.random() < 0.6,
                    start=rng.choice([0, 0, 70000]))
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "append":
        top = rng.choice([1, 7, 130, 2048])
        batch = _log_int(rng, 1, max(1, min(128, 8192 // top)))
        return dict(op=op, batch=batch, new=top, least_new=1,
                    context=_log_int(rng, 16, 6000), least_context=0, mix=rng.randrange(10 ** 6),
                    heads=heads, kv_heads=kv, dim=dim, page=page, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    norm=rng.choice(["rms", "layer", "none"]), rot=rng.choice([0, dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]))
    while True:
        top = rng.choice([1, 1, 5, 100, 2048])
        batch = _log_int(rng, 1, max(1, min(128, 4096 // top)))
        case = dict(op=op, batch=batch, new=top, least_new=1, context=_log_int(rng, 16, 120000), least_context=0,
                    mix=rng.randrange(10 ** 6), heads=heads, kv_heads=kv, dim=dim, page=page,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    window=rng.choice([-1, -1, -1, _log_int(rng, 1, 4096)]))
        new, total = _lengths(case)
        largest = dict(listed()[-2])
        if (work(case)["flops"] <= work(largest)["flops"] and sum(total) * kv * dim <= 400_000_000
                and max(n * t for n, t in zip(new, total)) * heads <= 700_000_000):
            return case


# ------------------------------------------------------------------------------------------------ lengths and work
def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and total tokens of every sequence: log-spread over the case's ranges, the upper ends among them."""
    rng = random.Random(case["mix"])
    new, total = [], []
    for b in range(case["batch"]):
        n = case["new"] if b == 0 else _log_int(rng, case["least_new"], case["new"])
        lo, hi = case["least_context"], case["context"]
        c = hi if b == 0 else (_log_int(rng, lo + 1, hi + 1) - 1 if hi > 0 else 0)
        new.append(n)
        total.append(n + c)
    return new, total


def _pairs(n: int, length: int, window: int) -> tuple[int, int]:
    """(visible query-key pairs, keys that some query sees) of one sequence: causal, positions from the end."""
    first = length - n
    if window < 0:
        return n * first + n * (n + 1) // 2, length
    pairs = sum(min(p, window) + 1 for p in range(first, length))
    return pairs, length - max(0, first - window)


def work(case: dict) -> dict:
    h, kv, d, sz = case["heads"], case["kv_heads"], case["dim"], _SIZE[case["dtype"]]
    if case["op"] == "norm_rope":
        n = case["tokens"] * (h + kv) * d
        if case["train"]:  # forward: x -> y; backward: x, dy -> dx
            return {"bytes": 5 * n * sz + 4 * case["tokens"], "flops": 25 * n}
        return {"bytes": 2 * n * sz + 4 * case["tokens"], "flops": 9 * n}
    new, total = _lengths(case)
    if case["op"] == "append":
        t = sum(new)
        return {"bytes": 2 * t * (h + 2 * kv) * d * sz + 4 * t, "flops": 9 * t * (h + kv) * d}
    pairs = keys = 0
    for n, length in zip(new, total):
        p, k = _pairs(n, length, case["window"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * keys * kv * d * sz + 2 * sum(new) * h * d * sz + 4 * keys // case["page"],
            "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------------------------------------ inputs
def _weights(case: dict, g: torch.Generator, dtype: torch.dtype, bias: bool, grad: bool) -> dict:
    out = {}
    for name in ("q", "k"):
        w = 1.0 + 0.2 * torch.randn(case["dim"], generator=g, device="cuda")
        out[f"{name}_weight"] = w.to(dtype).requires_grad_(grad)
        b = 0.1 * torch.randn(case["dim"], generator=g, device="cuda")
        out[f"{name}_bias"] = b.to(dtype).requires_grad_(grad) if bias else None
    return out


def _activations(g: torch.Generator, tokens: int, heads: int, dim: int, dtype: torch.dtype) -> torch.Tensor:
    """Projection outputs: every head has a scale of its own, one channel of each head stands out."""
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(heads, 1, generator=g, device="cuda"))
    x[:, :, dim // 3] *= 4.0
    return x.to(dtype)


def _page_table(case: dict, total: list[int], g: torch.Generator) -> tuple[torch.Tensor, int]:
    counts = [-(-t // case["page"]) for t in total]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pages


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm_rope":
        t = case["tokens"]
        if case["packed"]:  # one projection, per head [q | k | v]
            packed = _activations(g, t, h, 3 * d, dtype)
            q, k = packed[..., :d], packed[..., d:2 * d]
        else:
            q, k = _activations(g, t, h, d, dtype), _activations(g, t, kv, d, dtype)
        q, k = q.detach().requires_grad_(case["train"]), k.detach().requires_grad_(case["train"])
        pos = torch.arange(t, device="cuda", dtype=torch.int32) % 4096 + case["start"]
        state = dict(case=case, q=q, k=k, pos=pos, **_weights(case, g, dtype, not case["rms"], case["train"]))
        if case["train"]:
            state["dq"] = torch.randn(t, h, d, generator=g, device="cuda").to(dtype)
            state["dk"] = torch.randn(t, kv, d, generator=g, device="cuda").to(dtype)
        return state
    new, total = _lengths(case)
    table, pages = _page_table(case, total, g)
    cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    state = dict(case=case, new=new, total=total, page_table=table, cu_seqlens=cu,
                 seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"))
    t = sum(new)
    shape = (pages, case["page"], kv, d)
    if case["op"] == "append":
        state.update(k_cache=torch.zeros(shape, dtype=dtype, device="cuda"),
                     v_cache=torch.zeros(shape, dtype=dtype, device="cuda"),
                     q=_activations(g, t, h, d, dtype), k=_activations(g, t, kv, d, dtype),
                     v=torch.randn(t, kv, d, generator=g, device="cuda").to(dtype))
        if case["norm"] != "none":
            state.update(_weights(case, g, dtype, case["norm"] == "layer", False))
        return state
    # normalised keys and queries: scores of unit spread and somewhat above, as trained heads have them
    state.update(k_cache=torch.randn(shape, generator=g, device="cuda", dtype=dtype),
                 v_cache=torch.randn(shape, generator=g, device="cuda", dtype=dtype),
                 q=(1.5 * torch.randn(t, h, d, generator=g, device="cuda")).to(dtype))
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x: torch.Tensor, w, b, rms: bool) -> torch.Tensor:
    if w is None:
        return x
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.float()
    return y if b is None else y + b.float()


def _plain_rotate(x: torch.Tensor, pos: torch.Tensor, rot: int, base: float, interleaved: bool) -> torch.Tensor:
    if rot == 0:
        return x
    inv = base ** (-torch.arange(0, rot, 2, device=x.device, dtype=torch.float64) / rot)
    ang = pos.double()[:, None] * inv
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_norm_rope(s: dict):
    c = s["case"]
    out = []
    for n in ("q", "k"):
        y = _plain_norm(s[n].float(), s[f"{n}_weight"], s[f"{n}_bias"], c["rms"])
        out.append(_plain_rotate(y, s["pos"], c["rot"], c["base"], c["interleaved"]).to(s[n].dtype))
    return out


def _plain_append(s: dict):
    c = s["case"]
    dev = s["q"].device
    pos = torch.cat([torch.arange(t - n, t, device=dev) for n, t in zip(s["new"], s["total"])])
    seq = torch.repeat_interleave(torch.arange(c["batch"], device=dev), torch.tensor(s["new"], device=dev))
    out = []
    for n in ("q", "k"):
        y = _plain_norm(s[n].float(), s.get(f"{n}_weight"), s.get(f"{n}_bias"), c["norm"] == "rms")
        out.append(_plain_rotate(y, pos, c["rot"], c["base"], c["interleaved"]).to(s[n].dtype))
    page = s["page_table"][seq, pos // c["page"]].long()
    s["k_cache"][page, pos % c["page"]] = out[1]
    s["v_cache"][page, pos % c["page"]] = s["v"]
    return out[0], s["k_cache"], s["v_cache"]


def _plain_attend(s: dict):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    g = h // kv
    outs, at = [], 0
    for b, (n, length) in enumerate(zip(s["new"], s["total"])):
        pages = s["page_table"][b, :-(-length // c["page"])].long()
        k = s["k_cache"][pages].reshape(-1, kv, d)[:length].float().transpose(0, 1)  # [kv, length, d]
        v = s["v_cache"][pages].reshape(-1, kv, d)[:length].float().transpose(0, 1)
        q = s["q"][at:at + n].float().reshape(n, kv, g, d).permute(1, 2, 0, 3).reshape(kv, g * n, d)
        scores = torch.matmul(q, k.transpose(1, 2)).mul_(1.0 / math.sqrt(d)).view(kv, g, n, length)
        rel = torch.arange(length, device=q.device)[None] - torch.arange(length - n, length, device=q.device)[:, None]
        hidden = rel > 0
        if c["window"] >= 0:
            hidden |= rel < -c["window"]
        scores.masked_fill_(hidden, float("-inf"))
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(p.view(kv, g * n, length), v).view(kv, g, n, d) / p.sum(-1, keepdim=True)
        outs.append(o.permute(2, 0, 1, 3).reshape(n, h, d).to(s["q"].dtype))
        at += n
    return torch.cat(outs)


# ------------------------------------------------------------------------------------------------ the package's calls
def _own_norm_rope(s: dict):
    from scaling_b200.ops import functional as K

    c = s["case"]
    rotary = (c["rot"], c["base"], c["interleaved"]) if c["rot"] else None
    return K.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], q_bias=s["q_bias"], k_bias=s["k_bias"],
                          positions=s["pos"], rotary=rotary, eps=1e-5, rms=c["rms"])


def _own_append(s: dict):
    from scaling_b200.ops.paged_attention import paged_append

    c = s["case"]
    rotary = (c["rot"], c["base"], c["interleaved"]) if c["rot"] else None
    q = paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["cu_seqlens"], s["seq_lens"],
                     q=s["q"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), q_bias=s.get("q_bias"),
                     k_bias=s.get("k_bias"), rotary=rotary, eps=1e-5, rms=c["norm"] == "rms")
    return q, s["k_cache"], s["v_cache"]


def _own_attend(s: dict):
    from scaling_b200.ops.paged_attention import paged_attention

    window = s["case"]["window"]
    return paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["cu_seqlens"], s["seq_lens"],
                           causal=True, window=None if window < 0 else window)


def run(state: dict):
    case = state["case"]
    if case["op"] == "append":
        return _own_append(state) if own else _plain_append(state)
    if case["op"] == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if not case["train"]:
        with torch.no_grad():
            return tuple(_own_norm_rope(state) if own else _plain_norm_rope(state))
    outs = _own_norm_rope(state) if own else _plain_norm_rope(state)
    names = ["q", "k", "q_weight", "k_weight"] + ([] if case["rms"] else ["q_bias", "k_bias"])
    grads = torch.autograd.grad(outs, [state[n] for n in names], [state["dq"], state["dk"]])
    return tuple(o.detach() for o in outs) + grads


# ------------------------------------------------------------------------------------------------ definition, 64 bits
def _exact_head_rows(x, w, b, rms, pos, rot, base, interleaved, dy=None):
    """Rows ``x[t, h, :]`` normalised and rotated as complex numbers; with ``dy`` also (dx, dw, db) from the formulas."""
    x = x.detach().double()
    n = x.shape[-1]
    if w is None:
        xhat = x
        y = x
    else:
        mu = torch.zeros_like(x[..., :1]) if rms else x.sum(-1, keepdim=True) / n
        inv = 1.0 / torch.sqrt(((x - mu) ** 2).sum(-1, keepdim=True) / n + 1e-5)
        xhat = (x - mu) * inv
        y = xhat * w.detach().double()
        if b is not None:
            y = y + b.detach().double()

    def turn(z, sign):
        if rot == 0:
            return z.clone()
        theta = torch.stack([pos.double() * math.exp(-2.0 * i / rot * math.log(base)) for i in range(rot // 2)], 1)
        unit = torch.polar(torch.ones_like(theta), sign * theta)[:, None, :]
        res = z.clone()
        if interleaved:
            c = torch.complex(z[..., 0:rot:2].contiguous(), z[..., 1:rot:2].contiguous()) * unit
            res[..., 0:rot:2], res[..., 1:rot:2] = c.real, c.imag
        else:
            m = rot // 2
            c = torch.complex(z[..., :m].contiguous(), z[..., m:rot].contiguous()) * unit
            res[..., :m], res[..., m:rot] = c.real, c.imag
        return res

    out = turn(y, 1.0)
    if dy is None:
        return out
    d = turn(dy.double(), -1.0)
    dw, db = (d * xhat).sum((0, 1)), d.sum((0, 1))
    dh = d * w.detach().double()
    proj = (dh * xhat).sum(-1, keepdim=True) / n
    mean = torch.zeros_like(proj) if rms else dh.sum(-1, keepdim=True) / n
    return out, inv * (dh - mean - xhat * proj), dw, db


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        res = [_exact_head_rows(s[n], s[f"{n}_weight"], s[f"{n}_bias"], case["rms"], s["pos"], case["rot"], case["base"],
                                case["interleaved"], s.get(f"d{n}")) for n in ("q", "k")]
        if not case["train"]:
            return tuple(res)
        (qo, dq, dwq, dbq), (ko, dk, dwk, dbk) = res
        return (qo, ko, dq, dk, dwq, dwk) + (() if case["rms"] else (dbq, dbk))
    if case["op"] == "append":
        pos = torch.tensor([p for n, t in zip(s["new"], s["total"]) for p in range(t - n, t)], device="cuda")
        rows = [_exact_head_rows(s[n], s.get(f"{n}_weight"), s.get(f"{n}_bias"), case["norm"] == "rms", pos, case["rot"],
                                 case["base"], case["interleaved"]) for n in ("q", "k")]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        flat_k, flat_v = kc.view(-1, *kc.shape[2:]), vc.view(-1, *vc.shape[2:])
        at = 0
        for b, (n, t) in enumerate(zip(s["new"], s["total"])):
            p = pos[at:at + n]
            slot = s["page_table"][b].long()[p // case["page"]] * case["page"] + p % case["page"]
            flat_k[slot], flat_v[slot] = rows[1][at:at + n], s["v"][at:at + n].double()
            at += n
        return rows[0], kc, vc
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    at = 0
    for b, (n, length) in enumerate(zip(s["new"], s["total"])):
        j = torch.arange(length, device="cuda")
        page, row = s["page_table"][b].long()[j // case["page"]], j % case["page"]
        lo = max(0, length - n - case["window"]) if case["window"] >= 0 else 0
        for hk in range(case["kv_heads"]):
            k, v = s["k_cache"][page[lo:], row[lo:], hk].double(), s["v_cache"][page[lo:], row[lo:], hk].double()
            for i0 in range(0, n, 512):
                i = torch.arange(i0, min(n, i0 + 512), device="cuda")
                q = s["q"][at + i, hk * group:(hk + 1) * group].double()
                z = torch.einsum("ihd,jd->ihj", q, k) / math.sqrt(case["dim"])
                own_pos = (length - n + i)[:, None]
                seen = j[None, lo:] <= own_pos
                if case["window"] >= 0:
                    seen &= j[None, lo:] >= own_pos - case["window"]
                z = torch.where(seen[:, None], z, torch.full_like(z, -torch.inf))
                prob = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
                out[at + i, hk * group:(hk + 1) * group] = torch.einsum("ihj,jd->ihd", prob, v)
        at += n
    return out
