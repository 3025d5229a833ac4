"""Cases of the rotary and shared-prefix operators, for timing and comparison.

Three operators of the decode and prefill step of a model with rotary positions:

* ``norm_rope``: RMS norm of every query and key head, then the position rotation;
* ``append``: the same, with the keys and values stored in the paged KV pool;
* ``shared``: paged decode attention of a batch whose sequences share a prefix.

``run`` computes a case in plain torch operations in 32 bits, or, where
``own`` is set, through the package's entry points.  ``exact`` computes it in
64 bits from the operators' definitions.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_DEVICE = "cuda"
_EPS = 1e-6


def listed():
    rope = dict(d=128, rot=128, hq=32, hkv=8, block=16, layers=1, interleaved=False, norm=True,
                dtype="bf16", pool="bf16", views=True, table=40960)
    shared = dict(op="shared", d=128, hq=32, hkv=8, block=16, layers=1, dtype="bf16", pool="bf16")
    return [
        # One decode step of 64 requests, before an attention call that stores k itself.
        dict(rope, name="norm_rope decode 64", op="norm_rope", tokens=64, seqs=64),
        # 16 prefill chunks of 512 tokens: the largest step of the chunked-prefill benchmark.
        dict(rope, name="norm_rope prefill 8192", op="norm_rope", tokens=8192, seqs=16),
        # A small fp32 model with an odd head layout, partly rotated in adjacent pairs.
        dict(rope, name="norm_rope f32 odd", op="norm_rope", tokens=1021, seqs=3, d=80, rot=32, hq=20,
             hkv=4, interleaved=True, dtype="f32", pool="f32", views=False, table=4096),
        # One decode step of 256 requests with far positions; the pool's other layer stays.
        dict(rope, name="append decode 256", op="append", tokens=256, seqs=256, layers=2, table=131072),
        # The prefill step of a model with as many key as query heads and no norms.
        dict(rope, name="append prefill 8192 mha", op="append", tokens=8192, seqs=16, hkv=32,
             norm=False),
        # A ragged chunk of an fp16 model over a bf16 pool, half of each head rotated.
        dict(rope, name="append f16 partial", op="append", tokens=777, seqs=1, d=96, rot=48, hq=16,
             hkv=2, block=32, interleaved=True, dtype="f16", views=False, table=8192),
        # A few requests behind one system prompt: the latency of a small step.
        dict(shared, name="shared 4 x 2k", b=4, prefix=2048, smin=1, smax=64),
        # The long-context benchmark's 64 requests of 32 heads, 4k of the context in common.
        dict(shared, name="shared 64 x 4k mha", b=64, hkv=32, prefix=4096, smin=1, smax=1024),
        # Many questions to one long document.
        dict(shared, name="shared 64 x 32k", b=64, prefix=32768, smin=16, smax=512),
        # A large batch of samples of one prompt: the prefix is bound by arithmetic.
        dict(shared, name="shared 256 x 16k", b=256, prefix=16384, smin=1, smax=512),
        # Odd sizes: five query heads to a key head, heads of 80, a prefix that ends in a page.
        dict(shared, name="shared odd 37 x 3001", b=37, hq=20, hkv=4, d=80, block=32, layers=2,
             prefix=3001, smin=0, smax=333),
        # The end-to-end benchmark's fp32 heads (8 of 32).
        dict(shared, name="shared f32 16 x 4093", b=16, hq=8, hkv=8, d=32, dtype="f32", pool="f32",
             prefix=4093, smin=1, smax=200),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    # fp32 attention has the fp32 units alone: its operations weigh more.
    slow = 20 if case["op"] == "shared" and "f32" in (case["dtype"], case["pool"]) else 1
    slow = max(slow, 20 if case["op"] == "shared" and case["dtype"] == "f16" else 1)
    return max(w["bytes"], slow * w["flops"] / 200)


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        hkv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        hq = hkv * rng.choice([1, 1, 2, 3, 4, 5, 6, 7, 8, 16])
        if hq > 64:
            continue
        d = rng.choice([32, 64, 80, 96, 128, 128, 128])
        dtype, pool = rng.choice([("bf16", "bf16")] * 5 + [("f32", "f32"), ("f16", "bf16"), ("f32", "bf16")])
        case = dict(d=d, hq=hq, hkv=hkv, block=rng.choice([8, 16, 16, 32, 64]),
                    layers=rng.choice([1, 2]), dtype=dtype, pool=pool)
        op = rng.choice(["norm_rope", "append", "shared", "shared"])
        if op == "shared":
            smax = _log_int(rng, 1, 1024)
            case.update(op=op, b=_log_int(rng, 1, 256), prefix=_log_int(rng, 16, 32768),
                        smin=rng.randint(0, smax), smax=smax)
        else:
            tokens = _log_int(rng, 1, 8192)
            case.update(op=op, tokens=tokens, seqs=_log_int(rng, 1, tokens),
                        rot=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3,
                        norm=rng.random() < 0.7, views=rng.random() < 0.6,
                        table=_log_int(rng, 8192, 131072))
        if _cost(case) <= top:
            return case


# ------------------------------------------------------------------ inputs
def _suffix_lengths(case):
    """Own tokens of each sequence, spread evenly over [smin, smax]."""
    b, lo, hi = case["b"], case["smin"], case["smax"]
    return [hi] if b == 1 else [lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _generator(seed):
    return torch.Generator(device=_DEVICE).manual_seed(seed)


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device=_DEVICE, dtype=torch.float32).to(dtype)


def _pool(case, blocks, g):
    shape = (case["layers"], blocks, case["block"], case["hkv"], case["d"])
    dtype = _TYPES[case["pool"]]
    return SimpleNamespace(k=_randn(shape, dtype, g), v=_randn(shape, dtype, g),
                           block_size=case["block"])


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "shared":
        return _prepare_shared(case, g)
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    dtype = _TYPES[case["dtype"]]
    s = SimpleNamespace(case=case)
    if case["views"]:  # q, k and v are views of one projection's rows
        rows = _randn((t, (hq + 2 * hkv) * d), dtype, g)
        q, k, v = rows.split([hq * d, hkv * d, hkv * d], dim=1)
        s.q, s.k, s.v = q.view(t, hq, d), k.view(t, hkv, d), v.view(t, hkv, d)
    else:
        s.q, s.k, s.v = (_randn((t, h, d), dtype, g) for h in (hq, hkv, hkv))
    s.q_weight = s.k_weight = None
    if case["norm"]:
        s.q_weight = (1 + 0.2 * _randn((d,), torch.float32, g)).to(dtype)
        s.k_weight = (1 + 0.2 * _randn((d,), torch.float32, g)).to(dtype)
    # Chunks of nearly equal length, each at an offset of its own.
    seqs = case["seqs"]
    lengths = torch.tensor([t // seqs + (i < t % seqs) for i in range(seqs)], device=_DEVICE)
    longest = t // seqs + 1
    starts = torch.randint(0, case["table"] - longest + 1, (seqs,), generator=g, device=_DEVICE)
    first = torch.cumsum(lengths, 0) - lengths
    s.positions = (torch.repeat_interleave(starts - first, lengths, output_size=t)
                   + torch.arange(t, device=_DEVICE))
    # The rotation's table, kept like a weight: angles in 64 bits, rounded once.
    inv = 10000.0 ** (-torch.arange(0, case["rot"], 2, device=_DEVICE, dtype=torch.float64)
                      / case["rot"])
    angle = torch.arange(case["table"], device=_DEVICE, dtype=torch.float64)[:, None] * inv
    s.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)
    if case["op"] == "append":
        blocks = -(-t // case["block"]) + 8
        s.pool = _pool(case, blocks, g)
        s.layer = case["layers"] - 1
        s.slots = torch.randperm(blocks * case["block"], generator=g, device=_DEVICE)[:t]
    return s


def _prepare_shared(case, g):
    b, block, prefix = case["b"], case["block"], case["prefix"]
    s = SimpleNamespace(case=case)
    s.q = _randn((b, case["hq"], case["d"]), _TYPES[case["dtype"]], g)
    own_tokens = torch.tensor(_suffix_lengths(case), device=_DEVICE)
    own_tokens = own_tokens[torch.randperm(b, generator=g, device=_DEVICE)]
    s.lengths = own_tokens + prefix
    shared_pages = -(-prefix // block)
    first_own = prefix // block  # the page that holds a sequence's first own token
    pages = -(-s.lengths // block)
    width = max(1, -(-(prefix + case["smax"]) // block))
    own_pages = (pages - first_own).clamp(min=0)
    offset = torch.cumsum(own_pages, 0) - own_pages
    total = b * (width - first_own) + shared_pages + 3
    order = torch.randperm(total, generator=g, device=_DEVICE)
    s.prefix_table = order[:shared_pages].contiguous()
    column = torch.arange(width, device=_DEVICE)
    at = shared_pages + offset[:, None] + column - first_own
    table = torch.where((column >= first_own) & (column < pages[:, None]),
                        order[at.clamp(0, total - 1)], torch.full_like(at, -1))
    whole = prefix // block  # pages that the sequences have in common as a whole
    table[:, :whole] = s.prefix_table[:whole]
    s.tables = table.contiguous()
    s.prefix = prefix
    s.pool = _pool(case, total, g)
    s.layer = case["layers"] - 1
    return s


# --------------------------------------------------------------------- run
def run(s):
    op = s.case["op"]
    if own:
        return _run_own(s, op)
    if op == "norm_rope":
        q = _norm_rope(s, s.q, s.q_weight)
        k = _norm_rope(s, s.k, s.k_weight)
        return {"q": q.to(s.q.dtype), "k": k.to(s.k.dtype)}
    if op == "append":
        q = _norm_rope(s, s.q, s.q_weight).to(s.q.dtype)
        k = _norm_rope(s, s.k, s.k_weight)
        rows = lambda p: p[s.layer].view(-1, *p.shape[3:])  # noqa: E731
        rows(s.pool.k)[s.slots] = k.to(s.pool.k.dtype)
        rows(s.pool.v)[s.slots] = s.v.to(s.pool.v.dtype)
        return {"q": q, "k_pool": s.pool.k, "v_pool": s.pool.v}
    return _shared(s)


def _run_own(s, op):
    package = str(Path(__file__).resolve().parents[1] / "mini-gpt-inference_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import b200attn

    if op == "norm_rope":
        q, k = b200attn.qk_norm_rope_b200(s.q, s.k, s.positions, s.cos_sin, q_weight=s.q_weight,
                                          k_weight=s.k_weight, eps=_EPS,
                                          interleaved=s.case["interleaved"])
        return {"q": q, "k": k}
    if op == "append":
        q = b200attn.rope_kv_append_b200(s.q, s.k, s.v, s.pool, s.slots, s.positions, s.cos_sin,
                                         s.layer, q_weight=s.q_weight, k_weight=s.k_weight,
                                         eps=_EPS, interleaved=s.case["interleaved"])
        return {"q": q, "k_pool": s.pool.k, "v_pool": s.pool.v}
    return b200attn.shared_prefix_decode_b200(s.q, s.pool, s.prefix_table, s.prefix, s.tables,
                                              s.lengths, s.layer)


def _norm_rope(s, x, weight):
    """The norm and the rotation of x [tokens, heads, d], in 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.float()
    rot = s.case["rot"]
    half = rot // 2
    row = s.cos_sin[s.positions]
    cos, sin = row[:, None, :half], row[:, None, half:]
    if s.case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _shared(s):
    """Decode attention in 32 bits, the prefix's scores as one product for all sequences."""
    case = s.case
    b, hq, hkv, d, block = case["b"], case["hq"], case["hkv"], case["d"], case["block"]
    rep, prefix = hq // hkv, s.prefix
    k, v = (p[s.layer].view(-1, hkv, d) for p in (s.pool.k, s.pool.v))
    q = s.q.float().view(b, hkv, rep, d) * (1.0 / math.sqrt(d))
    at = torch.arange(prefix, device=q.device)
    row = s.prefix_table[at // block] * block + at % block
    kp, vp = k[row].float(), v[row].float()  # [prefix, hkv, d]
    qh = q.permute(1, 0, 2, 3).reshape(hkv, b * rep, d)
    scores = torch.matmul(qh, kp.permute(1, 2, 0)).view(hkv, b, rep, prefix).permute(1, 0, 2, 3)
    top = scores.amax(-1, keepdim=True)
    # The sequences' own tokens, padded to the longest.
    most = case["smax"]
    at = prefix + torch.arange(most, device=q.device)
    there = at < s.lengths[:, None]
    page = s.tables[:, at // block].clamp(min=0)
    row = page * block + at % block
    ks = torch.where(there[..., None, None], k[row].float(), 0.0)  # [b, most, hkv, d]
    vs = torch.where(there[..., None, None], v[row].float(), 0.0)
    tail = torch.matmul(q, ks.permute(0, 2, 3, 1))  # [b, hkv, rep, most]
    tail = torch.where(there[:, None, None, :], tail, float("-inf"))
    top = torch.maximum(top, tail.amax(-1, keepdim=True))
    p, t = torch.exp(scores - top), torch.exp(tail - top)
    total = p.sum(-1, keepdim=True) + t.sum(-1, keepdim=True)
    out = torch.matmul(p.permute(1, 0, 2, 3).reshape(hkv, b * rep, prefix), vp.permute(1, 0, 2))
    out = out.view(hkv, b, rep, d).permute(1, 0, 2, 3) + torch.matmul(t, vs.permute(0, 2, 1, 3))
    return (out / total).reshape(b, hq, d).to(s.q.dtype)


# -------------------------------------------------------------------- work
def work(case):
    es, ep, d, hq, hkv = _SIZE[case["dtype"]], _SIZE[case["pool"]], case["d"], case["hq"], case["hkv"]
    if case["op"] == "shared":
        own_tokens = sum(_suffix_lengths(case))
        tokens = case["prefix"] + own_tokens
        pages = -(-case["prefix"] // case["block"]) + -(-own_tokens // case["block"])
        return {"bytes": tokens * hkv * d * 2 * ep + case["b"] * hq * d * 2 * es + 8 * (pages + case["b"]),
                "flops": 4 * d * hq * (case["b"] * case["prefix"] + own_tokens)}
    t = case["tokens"]
    moved = t * hq * d * 2 * es + t * hkv * d * 2 * es  # q and k, read and written
    if case["op"] == "append":
        moved = t * hq * d * 2 * es + 2 * t * hkv * d * (es + ep) + 8 * t
    moved += 8 * t + 4 * case["rot"] * min(t, case["table"])
    turned = t * (hq + hkv) * d
    return {"bytes": moved, "flops": turned * (7 if case["norm"] else 3)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "shared":
        return _exact_shared(s)
    q = _exact_norm_rope(s, s.q, s.q_weight)
    k = _exact_norm_rope(s, s.k, s.k_weight)
    if case["op"] == "norm_rope":
        return {"q": q, "k": k}
    pools = {"q": q}
    for name, pool, new in (("k_pool", s.pool.k, k), ("v_pool", s.pool.v, s.v.double())):
        pool = pool.double()
        pool[s.layer, s.slots // case["block"], s.slots % case["block"]] = new
        pools[name] = pool
    return pools


def _exact_norm_rope(s, x, weight):
    """Each pair of elements as a complex number, turned by the table's row."""
    x = x.double()
    if weight is not None:
        x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS)
    rot = s.case["rot"]
    table = s.cos_sin.double()[s.positions].view(-1, 1, 2, rot // 2)
    turn = torch.complex(table[:, :, 0], table[:, :, 1])
    pairs = x[..., :rot].reshape(*x.shape[:-1], *((rot // 2, 2) if s.case["interleaved"] else (2, rot // 2)))
    axis = -1 if s.case["interleaved"] else -2
    z = torch.complex(*pairs.unbind(axis)) * turn
    turned = torch.stack([z.real, z.imag], axis).reshape(*x.shape[:-1], rot)
    return torch.cat([turned, x[..., rot:]], -1)


def _exact_shared(s):
    """Every sequence by itself, over its whole context in order."""
    case = s.case
    block, hkv, d = case["block"], case["hkv"], case["d"]
    rep = case["hq"] // hkv
    out = torch.empty(s.q.shape, dtype=torch.float64, device=s.q.device)
    k, v = s.pool.k[s.layer], s.pool.v[s.layer]
    common = torch.arange(s.prefix, device=s.q.device)
    common = [p[s.prefix_table[common // block], common % block].double() for p in (k, v)]
    for i, n in enumerate(s.lengths.tolist()):
        at = torch.arange(s.prefix, n, device=s.q.device)
        mine = [p[s.tables[i, at // block], at % block].double() for p in (k, v)]
        q = s.q[i].double().view(hkv, rep, d)
        parts = [torch.einsum("grd,ngd->grn", q, x) / math.sqrt(d) for x in (common[0], mine[0])]
        weight = torch.softmax(torch.cat(parts, -1), -1)
        o = torch.einsum("grn,ngd->grd", weight[..., :s.prefix], common[1])
        o = o + torch.einsum("grn,ngd->grd", weight[..., s.prefix:], mine[1])
        out[i] = o.reshape(-1, d)
    return out
