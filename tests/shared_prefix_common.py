"""Inputs and the 64-bit form of the shared-prefix decode, and the tolerances
its kernels are held to."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch


def case(b, hq, hkv, d, block, prefix, own, dtype=torch.bfloat16, pool_dtype=None, *, layers=1,
         layer=0, seed=0, index=torch.int64, poison=True, scale=1.0):
    """CPU inputs: ``own`` lists the sequences' own tokens.  Rows of the pool
    that no sequence owns are NaN, and so are the rows behind each last
    token; table entries that must not be read are out of range."""
    g = torch.Generator().manual_seed(seed)
    assert len(own) == b
    lens = torch.tensor([prefix + n for n in own])
    first = prefix // block
    shared = -(-prefix // block)
    pages = [-(-int(n) // block) for n in lens]
    need = shared + sum(max(0, p - first) for p in pages) + 2
    order = torch.randperm(need, generator=g).tolist()
    shape = (layers, need, block, hkv, d)
    fill = float("nan") if poison else 0.0
    k, v = torch.full(shape, fill), torch.full(shape, fill)
    table = [order.pop() for _ in range(shared)]
    width = max(1, max(pages))
    tables = torch.full((b, width), -7)
    kc, vc = (torch.randn(prefix, hkv, d, generator=g) for _ in range(2))
    at = torch.arange(prefix)
    if prefix:
        rows = torch.tensor(table)[at // block]
        k[layer, rows, at % block], v[layer, rows, at % block] = kc, vc
    for i in range(b):
        for j in range(first, pages[i]):
            tables[i, j] = order.pop()
        at = torch.arange(prefix, int(lens[i]))
        if len(at):
            rows = tables[i][at // block]
            k[layer, rows, at % block] = torch.randn(len(at), hkv, d, generator=g)
            v[layer, rows, at % block] = torch.randn(len(at), hkv, d, generator=g)
    pool_dtype = pool_dtype or dtype
    pool = SimpleNamespace(k=k.to(pool_dtype), v=v.to(pool_dtype), block_size=block)
    q = (scale * torch.randn(b, hq, d, generator=g)).to(dtype)
    return SimpleNamespace(q=q, pool=pool, table=torch.tensor(table, dtype=index), prefix=prefix,
                           tables=tables.to(index), lens=lens.to(index), layer=layer, block=block)


def to_device(c, device="cuda"):
    pool = SimpleNamespace(k=c.pool.k.to(device), v=c.pool.v.to(device), block_size=c.block)
    return SimpleNamespace(q=c.q.to(device), pool=pool, table=c.table.to(device), prefix=c.prefix,
                           tables=c.tables.to(device), lens=c.lens.to(device), layer=c.layer,
                           block=c.block)


def plain(c):
    """(out, spread) in float64, every sequence over its whole context by
    itself; spread [B, Hq, D] is sum_j p_j |v_j|, what the tolerance goes by."""
    b, hq, d = c.q.shape
    hkv = c.pool.k.shape[3]
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    spread = torch.zeros_like(out)
    big = torch.zeros(b, hq, dtype=torch.float64)
    for i in range(b):
        n = int(c.lens[i])
        if n < 1 or n < c.prefix or n > c.tables.shape[1] * c.block:
            continue
        at = torch.arange(n)
        page = c.tables[i].long()[(at // c.block).clamp(max=c.tables.shape[1] - 1)]
        if c.prefix:
            page[: c.prefix] = c.table.long()[at[: c.prefix] // c.block]
        k = c.pool.k[c.layer, page, at % c.block].double()
        v = c.pool.v[c.layer, page, at % c.block].double()
        q = c.q[i].double().view(hkv, hq // hkv, d)
        s = torch.einsum("grd,ngd->grn", q, k) / math.sqrt(d)
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("grn,ngd->grd", p, v).reshape(hq, d)
        spread[i] = torch.einsum("grn,ngd->grd", p, v.abs()).reshape(hq, d)
        mag = torch.einsum("grd,ngd->grn", q.abs(), k.abs()) / math.sqrt(d)
        big[i] = mag.amax(-1).reshape(hq)
    return out, spread, big


def bound(c, want, spread, big, tensor_cores):
    """Largest error of the kernels' arithmetic.

    A probability's relative error comes from its score's: products of a row
    of at most 128 elements summed in float32 in some order, at most 128
    roundings of partial sums of at most ``big`` = max_j sum_d |q_d k_jd| /
    sqrt(D), plus the scale's: 130 * 2^-24 * big; the exponential's argument
    is rounded once more (2^-24 * 2 big) and exp2 is good to 2^-22.  The
    weights, their sum and the outputs are then float32 sums of at most n
    terms: n * 2^-24 each in the worst order; both numerator and denominator
    carry it.  On tensor cores the weights are rounded to bf16 for the product
    with v: half a step, 2^-8 relative (the sum keeps them whole).  "split": what
    that leaves, at most 2^-8, is rounded to bf16 too and takes part: 2^-16."""
    n = float(c.lens.max())
    rel = 2 * (132 * 2.0 ** -24 * big + 2.0 ** -22 + n * 2.0 ** -24)
    rel = rel + {False: 0.0, True: 2.0 ** -8, "split": 2.0 ** -16}[tensor_cores]
    half = torch.finfo(c.q.dtype).eps / 2
    tiny = 2.0 ** -25 if c.q.dtype == torch.float16 else 1e-30
    return rel[..., None] * spread * (1 + half) + half * want.abs() + tiny


def assert_close(c, got, *, tensor_cores):
    want, spread, big = plain(c)
    err = (got.double().cpu() - want).abs()
    lim = bound(c, want, spread, big, tensor_cores)
    bad = ~(err <= lim)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{float((err / lim).nan_to_num(float('inf')).max()):.2f} of it, first at "
                           f"{bad.nonzero()[0].tolist()}")
