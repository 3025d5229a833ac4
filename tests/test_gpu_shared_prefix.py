"""Shared-prefix decode on the GPU against the 64-bit form of
tests/shared_prefix_common.py, which derives the tolerances."""
from __future__ import annotations

import pytest
import torch

from shared_prefix_common import assert_close, case, to_device

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(c, **kw):
    from b200attn import shared_prefix_decode_b200

    return shared_prefix_decode_b200(c.q, c.pool, c.table, c.prefix, c.tables, c.lens, c.layer, **kw)


def _check(cpu, tensor_cores=None, **kw):
    c = to_device(cpu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status) == 0
    if tensor_cores is None:  # weights in bf16 where everything is, in two pieces for f16
        tensor_cores = cpu.pool.k.dtype == BF16 and {BF16: True, F16: "split", F32: False}[cpu.q.dtype]
    assert_close(cpu, out, tensor_cores=tensor_cores)
    return c, out


# b, hq, hkv, d, block, prefix, own
SIZES = [
    (1, 1, 1, 128, 16, 1, [0]),                     # one key in all
    (1, 1, 1, 128, 16, 0, [1]),                     # no prefix
    (2, 4, 4, 128, 16, 16, [0, 1]),                 # one page
    (3, 8, 2, 128, 16, 100, [5, 0, 40]),            # the prefix ends inside a page
    (5, 32, 8, 128, 16, 2048, [1, 64, 17, 33, 16]), # grouped heads
    (4, 8, 8, 64, 32, 777, [300, 2, 31, 129]),
    (2, 20, 4, 80, 8, 333, [70, 1]),                # five query heads to a key head
    (3, 6, 2, 96, 64, 130, [3, 200, 64]),
    (7, 8, 8, 32, 16, 513, [1, 2, 3, 4, 5, 6, 100]),
    (2, 48, 3, 128, 16, 257, [9, 100]),             # 16 query heads to a key head
    (2, 34, 2, 64, 16, 64, [20, 0]),                # 17: three chunks of rows
    (70, 4, 2, 64, 16, 300, [i % 37 for i in range(70)]),  # more rows than one tile
    (3, 2, 2, 128, 1, 40, [3, 9, 0]),               # one token to a page
    (2, 2, 1, 16, 4, 50, [7, 30]),                  # short heads
    (2, 4, 4, 128, 256, 1500, [600, 3]),            # long pages
    (300, 8, 1, 128, 16, 640, [i % 5 for i in range(300)]),  # many rows to one key head
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F16, BF16), (F32, BF16), (BF16, F32)],
                         ids=str)
def test_shared_prefix(size, types):
    _check(case(*size, *types, seed=size[0] + size[3]))


# Of bf16, with rows and keys enough for the prefix's tensor tiles.
TILES = [
    (20, 16, 16, 64, 16, 3001, [i % 7 for i in range(20)]),     # 20 rows to a key head
    (5, 64, 16, 128, 16, 2801, [1, 64, 17, 33, 0]),             # four heads to each, 20 rows
    (17, 64, 64, 16, 64, 700, [i for i in range(17)]),          # short heads
    (37, 20, 4, 80, 32, 3001, [9 * i for i in range(37)]),      # a second tile, partly full
    (70, 4, 2, 64, 16, 7400, [i % 37 for i in range(70)]),
    (128, 8, 8, 128, 8, 1100, [i % 3 for i in range(128)]),     # one tile, just full
    (129, 8, 8, 32, 16, 1000, [i % 2 for i in range(129)]),     # a row more
    (256, 32, 32, 128, 16, 130, [i % 5 for i in range(256)]),   # two keys in the last key tile
    (257, 32, 32, 64, 16, 128, [1] * 257),                      # one key tile; a row in the third tile
]


@pytest.mark.parametrize("size", TILES, ids=lambda s: str(s[:6]))
def test_shared_prefix_tiles(size):
    _check(case(*size, seed=size[0]))


@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("size", [TILES[1], TILES[3], (33, 64, 4, 128, 16, 9001, [40 * i for i in range(33)]),
                                  (2, 8, 1, 128, 64, 40000, [0, 150])], ids=lambda s: str(s[:6]))
def test_other_queries_of_a_bf16_pool(size, dtype):
    """f16 and f32 queries meet a bf16 pool in exact pieces, whatever the sizes;
    three f32 pieces keep what f32 sums keep."""
    _check(case(*size, dtype, BF16, seed=50))


def test_queries_of_all_their_bits_against_one_key():
    """One key, so that the output is its value whatever the score; and two keys
    whose weights follow from a difference that only the last pieces show."""
    cpu = case(1, 8, 1, 64, 16, 0, [2], F32, BF16, seed=51)
    k = torch.zeros(2, 64)
    k[0, 0], k[1, 0], k[1, 1] = 1.0, 1.0, 1.0
    cpu.pool.k[0, cpu.tables[0, 0], :2, 0] = k.to(BF16)
    cpu.q[..., 1] = torch.tensor([1.0 + 2.0 ** -23 * (2 * i + 1) for i in range(8)]) * 8
    _check(cpu)


# A small and a large size for the tests below.
BOTH = pytest.mark.parametrize("heads", [(8, 2, 700), (64, 16, 2900)], ids=str)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_other_layer_strides_and_index_types(dtype, index):
    cpu = case(3, 8, 4, 64, 16, 90, [10, 0, 55], dtype, layers=3, layer=1, seed=5, index=index)
    c = to_device(cpu)
    wide = torch.zeros(8, 3, 128, dtype=dtype, device="cuda")
    wide[..., ::2] = c.q.transpose(0, 1)
    c.q = wide[..., ::2].transpose(0, 1)
    c.table = torch.stack([c.table, c.table - 100], 1)[:, 0]
    c.lens = torch.stack([c.lens, c.lens + 1], 1)[:, 0]
    c.tables = torch.cat([c.tables, c.tables - 50], 1).t().contiguous().t()[:, : cpu.tables.shape[1]]
    out = torch.zeros(3, 64, 8, dtype=dtype, device="cuda").transpose(1, 2)
    got = _run(c, out=out)
    assert got is out
    assert_close(cpu, got, tensor_cores=dtype == BF16)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@BOTH
def test_large_scores_keep_their_maximum(heads, dtype):
    # Scores of a few hundred: only a running maximum keeps the exponentials finite.
    hq, hkv, prefix = heads
    _check(case(5, hq, hkv, 128, 16, prefix, [3, 90, 0, 41, 7], dtype, seed=9, scale=30.0))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@BOTH
def test_rows_without_a_valid_length_are_zero_and_told(heads, dtype):
    from b200attn import _lib

    hq, hkv, prefix = heads
    cpu = case(5, hq, hkv, 64, 16, prefix, [4, 9, 0, 30, 7], dtype, seed=6)
    cpu.lens[1] = prefix - 1  # shorter than the prefix: a padding row
    cpu.lens[3] = 16 * cpu.tables.shape[1] + 1
    cpu.lens[4] = 0
    c = to_device(cpu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status)
    assert int(status) == _lib.DEV_BAD_LENGTH
    assert not out[[1, 3, 4]].any()
    assert_close(cpu, out, tensor_cores=dtype == BF16)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("where", ["prefix", "own"])
@BOTH
def test_bad_pages_are_told_and_touch_no_other_sequence(heads, dtype, where):
    from b200attn import _lib

    hq, hkv, prefix = heads
    cpu = case(5, hq, hkv, 128, 16, prefix, [20, 33, 5, 0, 1], dtype, seed=7, poison=False)
    c = to_device(cpu)
    if where == "prefix":
        c.table[2] = cpu.pool.k.shape[1]
    else:
        c.tables[1, prefix // 16 + 1] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, status=status)
    assert int(status) == _lib.DEV_BAD_BLOCK
    if where == "own":
        want = _run(to_device(cpu))
        rest = [0, 2, 3, 4]
        assert torch.equal(out[rest], want[rest])


def test_unread_table_entries_and_prefix_table_as_host_list():
    cpu = case(2, 4, 2, 64, 16, 70, [10, 20], BF16, seed=8)
    c = to_device(cpu)
    want = _run(c)
    c.tables[:, :4] = 1 << 40  # before prefix // S: not read
    c.table = cpu.table.tolist() + [1 << 40]
    assert torch.equal(_run(c), want)


@BOTH
def test_results_repeat_bit_for_bit(heads):
    cpu = case(9, *heads[:2], 128, 16, heads[2], [i * 30 for i in range(9)], BF16, seed=10)
    c = to_device(cpu)
    first = _run(c)
    for _ in range(5):
        assert torch.equal(_run(c), first)


@BOTH
def test_graph_replays_and_streams_have_their_own_workspaces(heads):
    hq, hkv, prefix = heads
    a = to_device(case(5, hq, hkv, 128, 16, prefix, [1, 70, 200, 3, 0], BF16, seed=11))
    b = to_device(case(5, hq, hkv, 128, 16, prefix, [9, 0, 10, 300, 2], BF16, seed=12))
    want = [_run(a), _run(b)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    # New inputs in the same buffers, replayed.
    a.q.mul_(-1)
    graphs[0].replay()
    assert torch.equal(outs[0], _run(a))
    # Direct calls side by side on two streams, and a prepared one.
    call = {0: None}
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(10):
        for c, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(_run(c))
    torch.cuda.synchronize()
    ra, rb = _run(a), _run(b)
    assert all(torch.equal(x, ra if i % 2 == 0 else rb) for i, x in enumerate(got))
    call = _run(a, prepare=True)
    assert torch.equal(call(), ra) and torch.equal(call(), ra)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("prefix", [3000, 4200])
def test_calls_back_to_back_in_one_stream(prefix, dtype):
    """Kernels of a call overlap; calls must not: memory that one call has given
    back serves the next, also where no row of a call is valid."""
    a = to_device(case(33, 8, 2, 128, 16, prefix, [i for i in range(33)], dtype, seed=16))
    b = to_device(case(3, 8, 2, 128, 16, 700, [9, 0, 10], dtype, seed=17))
    none = to_device(case(33, 8, 2, 128, 16, prefix, [5] * 33, dtype, seed=18))
    none.lens.fill_(1)
    want_a, want_b = _run(a), _run(b)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((_run(a), _run(none), _run(b)))
    torch.cuda.synchronize()
    for x, z, y in got:
        assert torch.equal(x, want_a) and torch.equal(y, want_b) and not z.any()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@BOTH
def test_scores_that_keep_growing(heads, dtype):
    """Each key's score exceeds the last's: the reference moves again and again."""
    hq, hkv, prefix = heads
    cpu = case(5, hq, hkv, 64, 16, prefix, [3, 0, 40, 100, 7], dtype, seed=19)
    k = cpu.pool.k.float()
    at = torch.arange(prefix)
    rows = cpu.table[at // 16]
    step = (at / prefix * 60)[:, None, None]
    q = cpu.q.float()
    k[0, rows, at % 16] = step * q[0, :hkv][None] / q[0, :hkv].square().sum(-1, keepdim=True) * 8
    cpu.pool.k = k.to(cpu.pool.k.dtype)
    _check(cpu)


@pytest.mark.parametrize("size", [(1, 1, 1, 64, 16, 300, [9]), (4, 32, 8, 128, 16, 2048, [1, 64, 17, 33]),
                                  (64, 4, 2, 80, 32, 500, [i for i in range(64)]),
                                  (3, 40, 4, 96, 16, 1000, [0, 200, 31]), TILES[0], TILES[1],
                                  (128, 8, 8, 128, 8, 1100, [i % 3 for i in range(128)]),
                                  (40, 6, 2, 96, 64, 6000, [i for i in range(40)])], ids=str)
def test_few_rows_differ_by_their_own_rounding_alone(size):
    """At most 128 rows to a key head: what the weights' rounding leaves takes part."""
    _check(case(*size, BF16, seed=22), tensor_cores="split")


def test_a_long_prefix_in_several_runs_to_a_cta():
    """Two row tiles, units that end inside a CTA's run, a prefix that ends
    inside a key tile."""
    _check(case(45, 14, 2, 128, 16, 9001, [i % 20 for i in range(45)], BF16, seed=20))
    _check(case(9, 8, 8, 64, 32, 20011, [i for i in range(9)], BF16, seed=21))


@pytest.mark.parametrize("size", [(2, 4, 1, 128, 64, 66001, [0, 150]), (5, 8, 1, 64, 256, 67000, [1] * 5)], ids=str)
def test_one_key_head_and_the_most_parts(size):
    _check(case(*size, BF16, seed=44), tensor_cores="split")


def test_torch_op_matches_direct_call():
    c = to_device(case(3, 4, 2, 64, 16, 70, [10, 20, 1], BF16, seed=13))
    got = torch.ops.b200attn.shared_prefix_decode(c.q, c.pool.k, c.pool.v, c.table, c.prefix,
                                                  c.tables, c.lens, c.layer)
    assert torch.equal(got, _run(c))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_agrees_with_the_paged_decode_where_heads_are_equal(dtype):
    from b200attn import paged_attention_batch_b200

    cpu = case(6, 8, 8, 128, 16, 320, [1, 50, 7, 16, 200, 31], dtype, seed=14)
    cpu.tables[:, : 320 // 16] = cpu.table[: 320 // 16]
    c = to_device(cpu)
    assert_close(cpu, paged_attention_batch_b200(c.q, c.pool, c.tables, c.lens, 0),
                 tensor_cores=dtype == BF16)
    assert_close(cpu, _run(c), tensor_cores=dtype == BF16)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_decode_steps_of_a_rotary_model_behind_one_prompt(dtype):
    """Append and attention together, step by step, as a serving loop runs them:
    the prompt is appended once, then every sequence appends its own tokens."""
    from types import SimpleNamespace

    from b200attn import rope_kv_append_b200, rope_table, shared_prefix_decode_b200
    from rope_common import norm_rope
    from shared_prefix_common import plain

    hq, hkv, d, block, prompt, b, steps = 8, 2, 64, 16, 40, 3, 20
    g = torch.Generator().manual_seed(15)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    table = rope_table(128, d)
    w = rnd(d)
    pool = SimpleNamespace(k=torch.full((1, 16, block, hkv, d), float("nan"), dtype=dtype),
                           v=torch.full((1, 16, block, hkv, d), float("nan"), dtype=dtype),
                           block_size=block)
    dev = SimpleNamespace(k=pool.k.cuda(), v=pool.v.cuda(), block_size=block)
    shared = [5, 2, 9]  # 40 tokens: the third page is half full
    tables = torch.tensor([[5, 2, 7, 0], [5, 2, 1, 8], [5, 2, 11, 3]])
    gpu_table = table.cuda()

    def append(q, k, v, slots, pos):
        return rope_kv_append_b200(q.cuda(), k.cuda(), v.cuda(), dev, slots.cuda(), pos.cuda(),
                                   gpu_table, 0, q_weight=w.cuda(), k_weight=w.cuda())

    pos = torch.arange(prompt)
    slots = torch.tensor(shared)[pos // block] * block + pos % block
    append(rnd(prompt, hq, d), rnd(prompt, hkv, d), rnd(prompt, hkv, d), slots, pos)
    for step in range(steps):
        pos = torch.full((b,), prompt + step)
        slots = tables[torch.arange(b), pos // block] * block + pos % block
        q, k, v = rnd(b, hq, d), rnd(b, hkv, d), rnd(b, hkv, d)
        qr = append(q, k, v, slots, pos)
        out = shared_prefix_decode_b200(qr, dev, shared, prompt, tables.cuda(), pos.cuda() + 1, 0)
        # The attention, on the pool and the queries as the kernels left them.
        c = SimpleNamespace(q=qr.cpu(), pool=SimpleNamespace(k=dev.k.cpu(), v=dev.v.cpu()),
                            table=torch.tensor(shared), prefix=prompt, tables=tables, lens=pos + 1,
                            layer=0, block=block)
        assert_close(c, out, tensor_cores=dtype == BF16)
        # The whole step against the formulas: q and k as the operators define them.
        half = torch.finfo(dtype).eps
        assert ((qr.double().cpu() - norm_rope(q, pos, table, w)).abs()
                <= half * norm_rope(q, pos, table, w).abs() + 2.0 ** -16).all()
        at = (0, slots // block, slots % block)
        assert torch.equal(dev.v[at].cpu(), v)
    assert torch.isfinite(plain(c)[0]).all()


@pytest.mark.parametrize("size", [(70, 4, 2, 64, 16, 300, [i % 37 for i in range(70)]),
                                  (5, 32, 8, 128, 16, 2048, [1, 64, 170, 33, 0]), TILES[1], TILES[3]],
                         ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_queries_that_are_no_numbers_stay_in_their_rows(size, dtype):
    cpu = case(*size, dtype, seed=41)
    c = to_device(cpu)
    clean = _run(c)
    odd = torch.zeros(size[:2], dtype=torch.bool, device="cuda")
    odd[1, 2] = odd[3, 0] = odd[4, 3] = True
    c.q[1, 2, 5], c.q[3, 0], c.q[4, 3, 7] = float("nan"), float("inf"), float("-inf")
    out = _run(c)
    assert out[odd].isnan().all()
    out[odd] = clean[odd]
    assert_close(cpu, out, tensor_cores=dtype == BF16)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@BOTH
def test_out_may_be_q_itself(heads, dtype):
    hq, hkv, prefix = heads
    cpu = case(6, hq, hkv, 128, 16, prefix, [600, 3, 0, 40, 1300, 77], dtype, seed=42)
    c = to_device(cpu)
    want = _run(c)
    for _ in range(3):
        c.q.copy_(cpu.q)
        assert _run(c, out=c.q).data_ptr() == c.q.data_ptr()
        assert torch.equal(c.q, want)
    wide = torch.empty(6, hq, 128, device="cuda")
    c.q.copy_(cpu.q)
    assert torch.equal(_run(c, out=wide).to(dtype), want)


def test_a_host_list_is_refused_while_a_graph_is_captured():
    c = to_device(case(2, 4, 2, 64, 16, 70, [10, 20], BF16, seed=43))
    want = _run(c)
    tensor, c.table = c.table, c.table.tolist()
    with pytest.raises(ValueError, match="prefix_table must be a CUDA tensor"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            _run(c)
    torch.cuda.synchronize()
    c.table = tensor
    assert torch.equal(_run(c), want)
