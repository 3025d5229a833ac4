"""The rotary operators' path for any strides and sizes, element by element:
appends from every layout, and bad positions and slots."""
from __future__ import annotations

import pytest
import torch

from rope_common import EPS, assert_close, norm_rope
from test_gpu_rope import _bits, _inputs, _pool

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


@pytest.mark.parametrize("layout", ["heads first", "strided", "off"])
@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F16, BF16), (F32, BF16), (BF16, F32)],
                         ids=str)
@pytest.mark.parametrize("size", [(6, 8, 2, 64, 64), (5, 3, 3, 80, 32), (4, 2, 1, 24, 2)], ids=str)
def test_append_layouts(size, types, layout):
    from b200attn import rope_kv_append_b200

    dtype, pdtype = types
    t, hq, hkv, d, rot = size
    q, k, v, qw, kw, pos, table = _inputs(*size, dtype, 25, layout=layout)
    pool = _pool(2, 5, 4, hkv, d, pdtype, 42)
    k0, v0 = pool.k.clone(), pool.v.clone()
    slots = torch.randperm(20, generator=torch.Generator().manual_seed(5))[:t].to(DEV)
    interleaved = t % 2 == 1
    out = torch.full((hq, t, d), 9.0, dtype=dtype, device=DEV).transpose(0, 1)
    got = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 1, q_weight=qw, k_weight=kw,
                              interleaved=interleaved, q_out=out)
    assert got is out
    assert_close(out, norm_rope(q, pos, table, qw, EPS, interleaved), dtype, rot, interleaved, "q")
    at = (1, slots // 4, slots % 4)
    assert_close(pool.k[at], norm_rope(k, pos, table, kw, EPS, interleaved), pdtype, rot,
                 interleaved, "k")
    assert torch.equal(pool.v[at], v.to(pdtype))
    k0[at], v0[at] = pool.k[at], pool.v[at]
    assert torch.equal(_bits(k0), _bits(pool.k)) and torch.equal(_bits(v0), _bits(pool.v))


@pytest.mark.parametrize("how", [(24, 2, "views"), (24, 24, "strided"), (64, 64, "off")], ids=str)
def test_bad_slots_and_positions_skip_their_token_alone(how):
    from b200attn import _lib, qk_norm_rope_b200, rope_kv_append_b200

    d, rot, layout = how
    q, k, v, qw, kw, pos, table = _inputs(6, 4, 2, d, rot, BF16, 8, layout=layout)
    pool = _pool(1, 4, 4, 2, d, BF16, 50)
    k0, v0 = pool.k.clone(), pool.v.clone()
    pos[1], pos[2] = -1, 64  # the table has 64 rows
    slots = torch.tensor([3, 4, 5, -1, 16, 9], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = rope_kv_append_b200(q, k, v, pool, slots, pos, table, 0, q_weight=qw, k_weight=kw,
                              status=status)
    assert int(status) == _lib.DEV_BAD_POSITION | _lib.DEV_BAD_SLOT
    assert_close(out, norm_rope(q, pos, table, qw), BF16, rot, False, "q")  # zero rows included
    want = norm_rope(k, pos, table, kw)
    for t, s in ((0, 3), (5, 9)):
        assert_close(pool.k[0, s // 4, s % 4][None], want[t:t + 1], BF16, rot, False, "k")
        k0[0, s // 4, s % 4] = pool.k[0, s // 4, s % 4]
        v0[0, s // 4, s % 4] = v[t]
    assert torch.equal(_bits(k0), _bits(pool.k)) and torch.equal(_bits(v0), _bits(pool.v))
    status.zero_()
    qo, ko = qk_norm_rope_b200(q, k, pos, table, status=status)
    assert int(status) == _lib.DEV_BAD_POSITION
    assert not qo[1:3].any() and not ko[1:3].any() and qo[0].any()
