"""Head norms, rotation and the rotary KV append on the GPU, against the plain
forms in 64 bits (tests/rope_common.py, which derives the tolerance)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from rope_common import EPS, assert_close, norm_rope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _randn(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _inputs(t, hq, hkv, d, rot, dtype, seed, *, layout="views", rows=64, wdtype=None):
    from b200attn import rope_table

    if layout == "views":  # slices of one projection
        x = _randn((t, (hq + 2 * hkv) * d), dtype, seed)
        q, k, v = x.split([hq * d, hkv * d, hkv * d], 1)
        q, k, v = q.view(t, hq, d), k.view(t, hkv, d), v.view(t, hkv, d)
    elif layout == "heads first":  # [H, T, D] storage
        q, k, v = (_randn((h, t, d), dtype, seed + i).transpose(0, 1)
                   for i, h in enumerate((hq, hkv, hkv)))
    elif layout == "strided":  # every other element
        q, k, v = (_randn((t, h, 2 * d), dtype, seed + i)[..., ::2]
                   for i, h in enumerate((hq, hkv, hkv)))
    else:  # one element off the 16-byte grid
        q, k, v = (_randn((t * h * d + 1,), dtype, seed + i)[1:].view(t, h, d)
                   for i, h in enumerate((hq, hkv, hkv)))
    w = [1 + 0.3 * _randn((d,), F32, seed + 7 + i) for i in range(2)]
    w = [x.to(wdtype or dtype) for x in w]
    g = torch.Generator().manual_seed(seed + 9)
    pos = torch.randint(0, rows, (t,), generator=g).to(DEV)
    return q, k, v, w[0], w[1], pos, rope_table(rows, rot, device=DEV)


SIZES = [  # t, hq, hkv, d, rot
    (1, 1, 1, 128, 128),   # one token, one head
    (5, 32, 8, 128, 128),  # grouped heads, several rows a thread
    (3, 64, 64, 128, 128), # more rows than one round of the CTA
    (7, 5, 1, 128, 64),    # half of each head rotated
    (9, 8, 8, 32, 32),     # lanes of 16 heads in a warp
    (4, 6, 2, 80, 32),     # chunk pairs not a power of two
    (3, 3, 3, 96, 48),
    (2, 4, 2, 256, 256),   # the widest head
    (5, 8, 2, 80, 40),     # 16-bit rows in chunks of 8 bytes
    (4, 33, 1, 72, 24),
    (3, 4, 2, 84, 44),     # fp32 rows in chunks of 8 bytes
    (5, 6, 2, 80, 20),     # and 16-bit rows in chunks of 4
    (4, 3, 2, 120, 12),
    (6, 2, 1, 64, 2),      # one pair: the element path
    (3, 2, 1, 10, 6),      # rows that are not whole chunks
    (2, 3, 1, 254, 100),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_norm_rope(size, interleaved, dtype):
    from b200attn import qk_norm_rope_b200

    t, hq, hkv, d, rot = size
    q, k, _, qw, kw, pos, table = _inputs(*size, dtype, 11)
    for a, b in ((qw, kw), (None, None), (qw, None), (None, kw)):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        qo, ko = qk_norm_rope_b200(q, k, pos, table, q_weight=a, k_weight=b,
                                   interleaved=interleaved, status=status)
        assert int(status) == 0 and qo.dtype == ko.dtype == dtype
        for what, got, x, w in (("q", qo, q, a), ("k", ko, k, b)):
            assert_close(got, norm_rope(x, pos, table, w, EPS, interleaved), dtype, rot,
                         interleaved, what)


@pytest.mark.parametrize("layout", ["views", "heads first", "strided", "off"])
@pytest.mark.parametrize("wdtype", [BF16, F32, F16], ids=str)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_norm_rope_layouts(layout, wdtype, index):
    from b200attn import qk_norm_rope_b200

    q, k, _, qw, kw, pos, table = _inputs(6, 8, 2, 64, 64, BF16, 3, layout=layout, wdtype=wdtype)
    pos2 = torch.stack([pos, pos + 1], 1).to(index)[:, 0]  # stride 2
    out = torch.zeros(8, 6, 64, dtype=BF16, device=DEV).transpose(0, 1)
    qo, ko = qk_norm_rope_b200(q, k, pos2, table, q_weight=qw, k_weight=kw, q_out=out, eps=1e-3)
    assert qo is out
    assert_close(qo, norm_rope(q, pos, table, qw, 1e-3), BF16, 64, False, "q")
    assert_close(ko, norm_rope(k, pos, table, kw, 1e-3), BF16, 64, False, "k")


@pytest.mark.parametrize("size", [(5, 32, 8, 128, 128), (7, 8, 2, 80, 40), (7, 8, 2, 80, 20), (3, 2, 1, 10, 6)], ids=str)
def test_norm_rope_in_place_gives_the_same(size):
    from b200attn import qk_norm_rope_b200

    q, k, v, qw, kw, pos, table = _inputs(*size, BF16, 5)
    v0 = v.clone()
    want = qk_norm_rope_b200(q, k, pos, table, q_weight=qw, k_weight=kw)
    got = qk_norm_rope_b200(q, k, pos, table, q_weight=qw, k_weight=kw, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(v, v0)  # the third view of the same rows


@pytest.mark.parametrize("size,dtype,interleaved", [((1301, 32, 8, 128, 128), BF16, False),
                                                    ((3001, 20, 4, 80, 32), F32, True),
                                                    ((2600, 32, 8, 80, 40), BF16, False),
                                                    ((2700, 12, 4, 80, 20), F32, True),
                                                    ((2500, 14, 4, 80, 20), BF16, True),
                                                    ((2500, 14, 4, 88, 36), F16, False),
                                                    ((2999, 9, 3, 64, 64), F16, False)], ids=str)
def test_many_tokens_equal_few(size, dtype, interleaved):
    """Large calls give a warp more rows; every row comes out the same."""
    from b200attn import qk_norm_rope_b200, rope_kv_append_b200

    t, hq, hkv, d, rot = size
    q, k, v, qw, kw, pos, table = _inputs(*size, dtype, 31)
    qo, ko = qk_norm_rope_b200(q, k, pos, table, q_weight=qw, k_weight=kw, interleaved=interleaved)
    assert_close(qo, norm_rope(q, pos, table, qw, EPS, interleaved), dtype, rot, interleaved, "q")
    assert_close(ko, norm_rope(k, pos, table, kw, EPS, interleaved), dtype, rot, interleaved, "k")
    pool = _pool(1, -(-t // 16), 16, hkv, d, F32, 95)
    slots = torch.randperm(t, generator=torch.Generator().manual_seed(6)).to(DEV)
    qa = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 0, q_weight=qw, k_weight=kw,
                             interleaved=interleaved)
    assert torch.equal(qa, qo)
    at = (0, slots // 16, slots % 16)
    assert torch.equal(pool.k[at].to(dtype), ko) and torch.equal(pool.v[at], v.float())
    for lo in (0, 500, t - 7):
        one = slice(lo, lo + 7)
        q7, k7 = qk_norm_rope_b200(q[one], k[one], pos[one], table, q_weight=qw, k_weight=kw,
                                   interleaved=interleaved)
        assert torch.equal(q7, qo[one]) and torch.equal(k7, ko[one])


def test_zero_rows_infinities_and_far_positions():
    from b200attn import qk_norm_rope_b200, rope_table

    table = rope_table(1 << 20, 128, device=DEV)
    pos = torch.tensor([0, (1 << 20) - 1, 777777], device=DEV)
    q = _randn((3, 4, 128), F32, 1)
    k = _randn((3, 2, 128), F32, 2)
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    k[2, 0, 3] = float("inf")
    w = torch.ones(128, device=DEV)
    qo, ko = qk_norm_rope_b200(q, k, pos, table, q_weight=w, k_weight=None)
    assert torch.equal(qo[0, 1], torch.zeros_like(qo[0, 1]))
    assert qo[1, 2].isnan().all() and not qo[1, 1].isnan().any()  # its own head alone
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 2] = False
    want = norm_rope(q, pos, table, w)
    assert_close(qo[keep], want[keep], F32, 128, False, "q")
    assert not torch.isfinite(ko[2, 0, [3, 67]]).any() and torch.isfinite(ko[2, 1]).all()


def _pool(layers, blocks, block, hkv, d, dtype, seed):
    return SimpleNamespace(k=_randn((layers, blocks, block, hkv, d), dtype, seed),
                           v=_randn((layers, blocks, block, hkv, d), dtype, seed + 1),
                           block_size=block)


def _bits(x):
    return x.view(torch.int16 if x.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F16, BF16), (F32, BF16), (BF16, F32),
                                   (F16, F32)], ids=str)
@pytest.mark.parametrize("size", [s for s in SIZES if s[3] <= 128 and s[3] % 8 == 0], ids=str)
def test_append(size, types):
    from b200attn import rope_kv_append_b200

    dtype, pdtype = types
    t, hq, hkv, d, rot = size
    q, k, v, qw, kw, pos, table = _inputs(*size, dtype, 21)
    pool = _pool(2, 5, 4, hkv, d, pdtype, 40)
    k0, v0 = pool.k.clone(), pool.v.clone()
    slots = torch.randperm(20, generator=torch.Generator().manual_seed(4))[:t].to(DEV)
    interleaved = t % 2 == 0
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 1, q_weight=qw, k_weight=kw,
                              interleaved=interleaved, status=status)
    assert int(status) == 0
    assert_close(out, norm_rope(q, pos, table, qw, EPS, interleaved), dtype, rot, interleaved, "q")
    at = (1, slots // 4, slots % 4)
    assert_close(pool.k[at], norm_rope(k, pos, table, kw, EPS, interleaved), pdtype, rot,
                 interleaved, "k")
    assert torch.equal(pool.v[at], v.to(pdtype))
    # Every other row stays as it was.
    k0[at], v0[at] = pool.k[at], pool.v[at]
    assert torch.equal(_bits(k0), _bits(pool.k)) and torch.equal(_bits(v0), _bits(pool.v))


@pytest.mark.parametrize("d", [128, 24])
def test_bad_slots_and_positions_skip_their_token_alone(d):
    from b200attn import _lib, qk_norm_rope_b200, rope_kv_append_b200

    q, k, v, qw, kw, pos, table = _inputs(6, 4, 2, d, d, BF16, 8)
    pool = _pool(1, 4, 4, 2, d, BF16, 50)
    k0, v0 = pool.k.clone(), pool.v.clone()
    pos[1], pos[2] = -1, 64  # the table has 64 rows
    slots = torch.tensor([3, 4, 5, -1, 16, 9], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 0, q_weight=qw, k_weight=kw,
                              status=status)
    assert int(status) == _lib.DEV_BAD_POSITION | _lib.DEV_BAD_SLOT
    assert_close(out, norm_rope(q, pos, table, qw), BF16, d, False, "q")  # zero rows included
    want = norm_rope(k, pos, table, kw)
    for t, s in ((0, 3), (5, 9)):
        assert_close(pool.k[0, s // 4, s % 4][None], want[t:t + 1], BF16, d, False, "k")
        k0[0, s // 4, s % 4] = pool.k[0, s // 4, s % 4]
        v0[0, s // 4, s % 4] = v[t]
    assert torch.equal(_bits(k0), _bits(pool.k)) and torch.equal(_bits(v0), _bits(pool.v))
    status.zero_()
    qo, ko = qk_norm_rope_b200(q, k, pos, table, status=status)
    assert int(status) == _lib.DEV_BAD_POSITION
    assert not qo[1:3].any() and not ko[1:3].any() and qo[0].any()


def test_no_tokens_and_host_slots():
    from b200attn import qk_norm_rope_b200, rope_kv_append_b200

    q, k, v, qw, kw, pos, table = _inputs(4, 4, 2, 64, 64, BF16, 13)
    pool = _pool(1, 4, 4, 2, 64, BF16, 60)
    k0 = pool.k.clone()
    qo, ko = qk_norm_rope_b200(q[:0], k[:0], pos[:0], table)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    assert rope_kv_append_b200(q[:0], k[:0], v[:0], pool, [], pos[:0], table, 0).shape[0] == 0
    assert torch.equal(k0, pool.k)
    rope_kv_append_b200(q, k, v, pool, [0, 5, 10, 15], pos, table, 0)
    assert torch.equal(pool.v[0, [0, 1, 2, 3], [0, 1, 2, 3]], v)


def test_host_slots_are_refused_while_a_graph_is_captured():
    from b200attn import rope_kv_append_b200

    q, k, v, qw, kw, pos, table = _inputs(4, 4, 2, 64, 64, BF16, 14)
    pool = _pool(1, 4, 4, 2, 64, BF16, 61)
    with pytest.raises(ValueError, match="slot_mapping must be a CUDA tensor"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rope_kv_append_b200(q, k, v, pool, [0, 5, 10, 15], pos, table, 0)
    torch.cuda.synchronize()
    rope_kv_append_b200(q, k, v, pool, [0, 5, 10, 15], pos, table, 0)
    assert torch.equal(pool.v[0, [0, 1, 2, 3], [0, 1, 2, 3]], v)


def test_prepared_call_graph_replay_and_other_stream():
    from b200attn import rope_kv_append_b200

    q, k, v, qw, kw, pos, table = _inputs(16, 32, 8, 128, 128, BF16, 17)
    slots = torch.arange(16, device=DEV)
    direct, pool = _pool(1, 2, 8, 8, 128, BF16, 70), _pool(1, 2, 8, 8, 128, BF16, 70)
    want = rope_kv_append_b200(q, k, v, direct, slots, pos, table, 0, q_weight=qw, k_weight=kw)
    call = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 0, q_weight=qw, k_weight=kw,
                               prepare=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(pool.k, direct.k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 0, q_weight=qw, k_weight=kw)
    q.mul_(2), v.mul_(-1), pos.add_(1).remainder_(64)
    g.replay()
    want = rope_kv_append_b200(q, k, v, direct, slots, pos, table, 0, q_weight=qw, k_weight=kw)
    assert torch.equal(out, want)
    assert torch.equal(pool.k, direct.k) and torch.equal(pool.v, direct.v)


def test_torch_ops_match_direct_calls():
    from b200attn import qk_norm_rope_b200, rope_kv_append_b200

    q, k, v, qw, kw, pos, table = _inputs(5, 8, 2, 64, 32, BF16, 19)
    want = qk_norm_rope_b200(q, k, pos, table, q_weight=qw, eps=1e-5, interleaved=True)
    got = torch.ops.b200attn.qk_norm_rope(q, k, pos, table, qw, None, 1e-5, True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, b = _pool(1, 2, 4, 2, 64, BF16, 80), _pool(1, 2, 4, 2, 64, BF16, 80)
    slots = torch.tensor([7, 0, 3, 5, 2], device=DEV)
    want = rope_kv_append_b200(q, k, v, a, slots, pos, table, 0, k_weight=kw)
    got = torch.ops.b200attn.rope_kv_append(q, k, v, b.k, b.v, slots, pos, table, 0, None, kw)
    assert torch.equal(got, want) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_a_rotary_step_with_the_paged_decode(dtype):
    """Append + decode equals norm + rotation + decode with its own KV write."""
    from b200attn import paged_attention_batch_b200, qk_norm_rope_b200, rope_kv_append_b200

    b, h, d, block = 3, 4, 64, 16
    q, k, v, qw, kw, pos, table = _inputs(b, h, h, d, d, dtype, 23)
    lens = torch.tensor([1, 16, 33], device=DEV)
    tables = torch.tensor([[4, -1, -1], [2, -1, -1], [0, 5, 1]], device=DEV)
    slots = torch.tensor([4 * 16, 2 * 16 + 15, 1 * 16], device=DEV)
    p1, p2 = (_pool(1, 6, block, h, d, dtype, 90) for _ in range(2))
    q1 = rope_kv_append_b200(q, k, v, p1, slots, lens - 1, table, 0, q_weight=qw, k_weight=kw)
    o1 = paged_attention_batch_b200(q1, p1, tables, lens, 0)
    q2, k2 = qk_norm_rope_b200(q, k, lens - 1, table, q_weight=qw, k_weight=kw)
    o2 = paged_attention_batch_b200(q2, p2, tables, lens, 0, k_new=k2, v_new=v, slot_mapping=slots)
    assert torch.equal(q1, q2) and torch.equal(p1.k, p2.k) and torch.equal(p1.v, p2.v)
    assert torch.equal(o1, o2)
