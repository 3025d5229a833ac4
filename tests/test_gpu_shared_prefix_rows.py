"""Shared-prefix decode with more than 128 query rows to a key head (two row
tiles on tcgen05): references that move, invalid lengths and pages, outputs in
place, replays; and what every size does with a bad page of the prefix."""
from __future__ import annotations

import pytest
import torch

from shared_prefix_common import assert_close, case, to_device

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
# b, hq, hkv, prefix: 160 and 280 rows to a key head.
MANY = pytest.mark.parametrize("rows", [(40, 16, 4, 2900), (70, 8, 2, 5003)], ids=str)
HEADS = pytest.mark.parametrize("d", [64, 128])


def _run(c, **kw):
    from b200attn import shared_prefix_decode_b200

    return shared_prefix_decode_b200(c.q, c.pool, c.table, c.prefix, c.tables, c.lens, c.layer, **kw)


def _case(rows, d, seed, **kw):
    b, hq, hkv, prefix = rows
    return case(b, hq, hkv, d, 16, prefix, [i % 29 for i in range(b)], BF16, seed=seed, **kw)


def _check(cpu):
    c = to_device(cpu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status)
    assert int(status) == 0
    assert_close(cpu, out, tensor_cores=True)


@HEADS
@MANY
def test_large_scores(rows, d):
    _check(_case(rows, d, 71, scale=30.0))


@HEADS
@MANY
@pytest.mark.parametrize("most", [60.0, 600.0])
def test_scores_that_keep_growing(rows, d, most):
    """Keys along one direction, longer and longer: rows on its side move their
    reference again and again, by more than 2^16 between tiles at the steeper one."""
    cpu = _case(rows, d, 72)
    prefix = rows[3]
    g = torch.Generator().manual_seed(73)
    u = torch.randn(d, generator=g)
    u /= u.norm()
    at = torch.arange(prefix)
    k = cpu.pool.k.float()
    k[0, cpu.table[at // 16], at % 16] = ((at / prefix * most)[:, None] * u)[:, None, :]
    cpu.pool.k = k.to(BF16)
    q = cpu.q.float()
    cpu.q = (q + (2 + torch.arange(rows[0])[:, None, None] % 5) * u).to(BF16)
    _check(cpu)


@HEADS
@MANY
def test_rows_without_a_valid_length(rows, d):
    from b200attn import _lib

    cpu = _case(rows, d, 74)
    bad = [1, 3, 17, 38]
    cpu.lens[1], cpu.lens[3], cpu.lens[38] = rows[3] - 1, 16 * cpu.tables.shape[1] + 1, -5
    cpu.lens[17] = 0
    c = to_device(cpu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status)
    assert int(status) == _lib.DEV_BAD_LENGTH
    assert not out[bad].any()
    assert_close(cpu, out, tensor_cores=True)


@HEADS
@MANY
def test_out_in_place_of_q(rows, d):
    """Also where rows without a valid length get their zeros while others' are
    still to be read."""
    cpu = _case(rows, d, 75)
    cpu.lens[5], cpu.lens[21] = 0, rows[3] - 1
    c = to_device(cpu)
    want = _run(c)
    for _ in range(5):
        c.q.copy_(cpu.q)
        assert _run(c, out=c.q) is c.q
        assert torch.equal(c.q, want)


@HEADS
@MANY
def test_repeats_and_graph_replays(rows, d):
    a, b = to_device(_case(rows, d, 76)), to_device(_case(rows, d, 77))
    want = [_run(a), _run(b)]
    for _ in range(5):
        assert torch.equal(_run(a), want[0]) and torch.equal(_run(b), want[1])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("value", [-1, 1 << 20, -(1 << 40)])
@pytest.mark.parametrize("size", [(5, 8, 2, 700), (5, 64, 16, 2900), (40, 16, 4, 2900)], ids=str)
def test_a_bad_page_of_the_prefix_is_read_as_page_0(size, value):
    from b200attn import _lib

    cpu = _case(size, 64, 78, poison=False)
    cpu.table[7] = 0
    want = _run(to_device(cpu))
    assert_close(cpu, want, tensor_cores=True)
    c = to_device(cpu)
    c.table[7] = value
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(_run(c, status=status), want)
    assert int(status) == _lib.DEV_BAD_BLOCK


@MANY
def test_bad_own_pages_touch_no_other_sequence(rows):
    from b200attn import _lib

    cpu = _case(rows, 128, 79, poison=False)
    want = _run(to_device(cpu))
    c = to_device(cpu)
    c.tables[28, rows[3] // 16] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status)
    assert int(status) == _lib.DEV_BAD_BLOCK
    rest = [i for i in range(rows[0]) if i != 28]
    assert torch.equal(out[rest], want[rest])


@HEADS
@pytest.mark.parametrize("rows", [(40, 16, 4, 2900), (70, 8, 2, 5003), (20, 16, 16, 3001)], ids=str)
def test_out_in_place_of_padding_rows_that_are_no_numbers(rows, d):
    """Rows that hold anything, and get their zeros where their queries stood, leave
    the other rows' results as they are, bit for bit."""
    cpu = _case(rows, d, 80)
    at = torch.arange(rows[3])
    k = cpu.pool.k.float()
    k[0, cpu.table[at // 16], at % 16, :, 0] += (at / rows[3] * 30 * d ** 0.5)[:, None]
    cpu.pool.k = k.to(BF16)
    cpu.q[..., 0] = 1
    bad = torch.arange(0, rows[0], 6)
    cpu.q[bad] = float("nan")
    cpu.lens[bad] = 0
    c = to_device(cpu)
    want = _run(c)
    assert not want[bad].any() and want.isfinite().all()
    for _ in range(30):
        c.q.copy_(cpu.q)
        _run(c, out=c.q)
        assert torch.equal(c.q, want)
