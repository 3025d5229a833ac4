"""Host side of the head norms, rotation and rotary KV append, without a GPU."""
from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from rope_common import norm_rope


def test_rope_table_rows():
    from b200attn import rope_table

    t = rope_table(100001, 8, base=500.0)
    assert t.dtype == torch.float32 and t.shape == (100001, 8)
    for n in (0, 1, 99999, 100000):
        for i in range(4):
            angle = n * 500.0 ** (-2 * i / 8)
            # float64 angles: off by a few units of 2^-53 * 1e5, then one rounding.
            assert abs(float(t[n, i]) - math.cos(angle)) <= 2.0 ** -24
            assert abs(float(t[n, 4 + i]) - math.sin(angle)) <= 2.0 ** -24
    for bad in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError):
            rope_table(*bad)


def test_plain_rotation_depends_on_the_distance_alone():
    from b200attn import rope_table

    t = rope_table(64, 16)
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(1, 1, 16, generator=g), torch.randn(1, 1, 16, generator=g)
    for inter in (False, True):
        dot = [float((norm_rope(x, torch.tensor([a]), t, None, 1e-6, inter)
                      * norm_rope(y, torch.tensor([a + 5]), t, None, 1e-6, inter)).sum())
               for a in (0, 7, 50)]
        # Table entries are off by 2^-25 at most (half a step below 1).
        assert max(dot) - min(dot) < 64 * 2.0 ** -24


def _rope(**kw):
    from b200attn import _lib

    v = dict(num_tokens=5, num_q_heads=8, num_kv_heads=2, head_dim=64, q=1 << 20, q_s0=512, q_s1=64,
             q_s2=1, k=2 << 20, k_s0=128, k_s1=64, k_s2=1, q_out=3 << 20, q_out_s0=512, q_out_s1=64,
             q_out_s2=1, k_out=4 << 20, k_out_s0=128, k_out_s1=64, k_out_s2=1, cos_sin=5 << 20,
             table_rows=16, rotary_dim=64, positions=6 << 20, position_stride=1,
             dtype=_lib.DTYPE_BF16, position_dtype=_lib.INDEX_I64, eps=1e-6)
    v.update(kw)
    return _lib.QkNormRopeArgs(**v)


BAD = {
    "no query heads": dict(num_q_heads=0),
    "no key heads": dict(num_kv_heads=0),
    "head too wide": dict(head_dim=258),
    "odd rotary_dim": dict(rotary_dim=33),
    "rotary_dim above the head": dict(rotary_dim=66),
    "no rotary_dim": dict(rotary_dim=0),
    "null q": dict(q=None),
    "null q_out": dict(q_out=None),
    "null table": dict(cos_sin=None),
    "null positions": dict(positions=None),
    "empty table": dict(table_rows=0),
    "bad dtype": dict(dtype=9),
    "bad weight dtype": dict(q_weight=7 << 20, weight_dtype=9),
    "bad position dtype": dict(position_dtype=4),
    "eps zero": dict(eps=0.0),
    "eps nan": dict(eps=float("nan")),
    "too many tokens": dict(num_tokens=1 << 31),
    "negative tokens": dict(num_tokens=-1),
}


@pytest.mark.parametrize("why", BAD)
def test_c_entry_refuses(why):
    from b200attn import _lib

    lib = _lib.load()
    refused = (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED)
    assert lib.b200_qk_norm_rope(ctypes.byref(_rope(**BAD[why])), None) in refused
    assert _lib.last_error(lib)
    pool = _lib.KVPool(1 << 20, 2 << 20, 2, 8, 16, 2, 64, _lib.DTYPE_BF16)
    a = _lib.RopeKvAppendArgs(rope=_rope(k_out=None, **BAD[why]), pool=pool, v=8 << 20,
                              slot_mapping=9 << 20, slot_stride=1, slot_dtype=_lib.INDEX_I64)
    assert lib.b200_rope_kv_append(ctypes.byref(a), None) in refused


def test_c_entries_refuse_their_own_and_take_no_tokens():
    from b200attn import _lib

    lib = _lib.load()
    assert ctypes.sizeof(_lib.QkNormRopeArgs) == 28 * 8 + 6 * 4
    assert ctypes.sizeof(_lib.RopeKvAppendArgs) == 28 * 8 + 24 + 64 + 7 * 8 + 8
    assert lib.b200_qk_norm_rope(None, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_rope_kv_append(None, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_qk_norm_rope(ctypes.byref(_rope(k_out=None)), None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_qk_norm_rope(ctypes.byref(_rope(num_tokens=0)), None) == _lib.OK

    def append(pool=(1 << 20, 2 << 20, 2, 8, 16, 2, 64, _lib.DTYPE_BF16), rope=None, **kw):
        v = dict(layer_idx=1, v=8 << 20, slot_mapping=9 << 20, slot_stride=1,
                 slot_dtype=_lib.INDEX_I64)
        v.update(kw)
        a = _lib.RopeKvAppendArgs(rope=rope or _rope(k_out=None), pool=_lib.KVPool(*pool), **v)
        return lib.b200_rope_kv_append(ctypes.byref(a), None)

    bad = (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED)
    assert append(layer_idx=2) in bad
    assert append(v=None) in bad
    assert append(slot_mapping=None) in bad
    assert append(slot_dtype=5) in bad
    assert append(rope=_rope()) in bad  # k_out given
    assert append(pool=(1 << 20, 2 << 20, 2, 8, 16, 4, 64, _lib.DTYPE_BF16)) in bad
    assert append(pool=(1 << 20, 2 << 20, 2, 8, 16, 2, 128, _lib.DTYPE_BF16)) in bad
    assert append(pool=(1 << 20, 2 << 20, 2, 8, 16, 2, 64, _lib.DTYPE_F16)) in bad
    assert append(rope=_rope(k_out=None, num_tokens=0)) == _lib.OK


class _Cuda:
    """A CPU tensor that says it is on the GPU: the refusals come before any launch."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return True if name == "is_cuda" else getattr(self.t, name)


def test_python_entries_refuse():
    from b200attn import qk_norm_rope_b200, rope_kv_append_b200, rope_table

    q, k = torch.zeros(3, 4, 32), torch.zeros(3, 2, 32)
    pos, table = torch.zeros(3, dtype=torch.int64), rope_table(8, 32)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope_b200(q, k, pos, table)
    with pytest.raises(RuntimeError, match="inference"):
        qk_norm_rope_b200(q.clone().requires_grad_(), k, pos, table)
    with pytest.raises(RuntimeError, match="inference"):
        qk_norm_rope_b200(q, k, pos, table, q_weight=torch.ones(32, requires_grad=True))

    with pytest.raises(RuntimeError, match="inference"):
        qk_norm_rope_b200(q, k, pos, table.clone().requires_grad_())

    def refuse(match, q=q, k=k, pos=pos, table=table, **kw):
        with pytest.raises(ValueError, match=match):
            qk_norm_rope_b200(_Cuda(q), k, pos, table, **kw)

    refuse("shape", k=k[0])
    refuse("agree", k=k[:2])
    refuse("agree", k=torch.zeros(3, 2, 16))
    refuse("nonzero", k=k[:, :0])
    refuse("dtype", k=k.half())
    refuse("positions", pos=pos.float())
    refuse("positions", pos=pos[:2])
    refuse("cos_sin", table=table.double())
    refuse("cos_sin", table=table[:, ::2])
    refuse("rotary_dim", table=torch.zeros(8, 34))
    refuse("at least one row", table=table[:0])
    refuse("weights", q_weight=torch.ones(16))
    refuse("weights", q_weight=torch.ones(32), k_weight=torch.ones(32).half())
    refuse("eps", eps=0.0)
    refuse("status", status=torch.zeros(1))
    refuse("shape, dtype", q_out=torch.zeros(3, 4, 16))
    refuse("overlap itself", q_out=torch.zeros(1, 1, 32).expand(3, 4, 32))
    both = torch.zeros(3, 6, 32)
    refuse("overlap the inputs", q=both[:, :4], q_out=both[:, 2:])
    refuse("overlap the inputs", q=q, q_out=k.new_zeros(6, 2, 32)[:3].repeat(1, 2, 1), k=k, k_out=q[:, :2])
    pool = SimpleNamespace(k=torch.zeros(1, 4, 4, 2, 32), v=torch.zeros(1, 4, 4, 2, 32), block_size=4)
    with pytest.raises(ValueError, match="matching"):
        rope_kv_append_b200(_Cuda(q), k, k[:, :1], pool, [0, 1, 2], pos, table, 0)
    with pytest.raises(ValueError, match="do not match the KV pool"):
        rope_kv_append_b200(_Cuda(torch.zeros(3, 4, 16)), torch.zeros(3, 2, 16), torch.zeros(3, 2, 16),
                            pool, [0, 1, 2], pos, rope_table(8, 16), 0)
    with pytest.raises(ValueError, match="layer_idx"):
        rope_kv_append_b200(_Cuda(q), k, k, pool, torch.arange(3), pos, table, 1)
    with pytest.raises(ValueError, match="slot_mapping"):
        rope_kv_append_b200(_Cuda(q), k, k, pool, torch.arange(2), pos, table, 0)


def test_torch_ops_have_schemas_and_fake_shapes():
    import b200attn  # noqa: F401

    s = str(torch.ops.b200attn.rope_kv_append.default._schema)
    assert "Tensor(a3!) k_pool, Tensor(a4!) v_pool" in s
    with FakeTensorMode():
        q, k = torch.empty(3, 8, 64, device="cuda"), torch.empty(3, 2, 64, device="cuda")
        pool = torch.empty(1, 2, 16, 2, 64, device="cuda")
        pos, table = torch.empty(3, dtype=torch.int64, device="cuda"), torch.empty(9, 64, device="cuda")
        qo, ko = torch.ops.b200attn.qk_norm_rope(q, k, pos, table)
        assert qo.shape == q.shape and ko.shape == k.shape
        qo = torch.ops.b200attn.rope_kv_append(q, k, k, pool, pool.clone(), pos, pos, table, 0)
        assert qo.shape == q.shape
