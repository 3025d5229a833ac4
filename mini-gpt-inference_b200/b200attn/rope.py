"""Head norms and position rotation of q and k, and the rotary KV append.

The reference model has learned positions (minivllm/model.py:41-44) and needs
neither; models with rotary positions, and those that normalise each query
and key head, need both before the attention ops of :mod:`b200attn.ops`:

* :func:`qk_norm_rope_b200` gives the normed and rotated q and k, ready for
  ``paged_attention_batch_b200(..., k_new=k, v_new=v, slot_mapping=...)``;
* :func:`rope_kv_append_b200` also stores k and v at their slots, like
  ``kv_scatter_b200``, so that the rotated k never goes through memory twice;
* :func:`rope_table` makes the table of cosines and sines that both read.

Query and key heads may differ in number (grouped heads).
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import (_DTYPES, _INDEX, _DeviceCall, _index_arg, _inference_only, _launch,
                  _pool_fields, _status_ptr)

_PACK_ROPE = _lib.packer(_lib.QkNormRopeArgs).pack
_PACK_APPEND = _lib.packer(_lib.RopeKvAppendArgs).pack


def rope_table(max_positions: int, rotary_dim: int, *, base: float = 10000.0,
               device=None) -> torch.Tensor:
    """[max_positions, rotary_dim] float32: cos(n f_i) in the first half of a
    row n, sin(n f_i) in the second, with f_i = base ** (-2 i / rotary_dim).

    Angles are computed in float64 and rounded once, so far positions keep
    their accuracy.  Models with scaled frequencies pass a table of their own.
    """
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rope_table needs max_positions >= 1 and an even rotary_dim >= 2")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    n = torch.arange(max_positions, dtype=torch.float64, device=device)
    angle = n[:, None] * base ** (-i / rotary_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two [T, H, D] tensors certainly share no byte: their spans are
    apart, or they are different columns of rows of one stride (the views of
    a fused projection)."""
    if x.numel() == 0 or y.numel() == 0:
        return True
    ex, ey = x.element_size(), y.element_size()
    row_x, row_y = ((1 + sum((n - 1) * s for n, s in zip(t.shape[1:], t.stride()[1:]))) * e
                    for t, e in ((x, ex), (y, ey)))
    step_x, step_y = x.stride(0) * ex, y.stride(0) * ey
    a, b = x.data_ptr(), y.data_ptr()
    if a + (x.shape[0] - 1) * step_x + row_x <= b or b + (y.shape[0] - 1) * step_y + row_y <= a:
        return True
    if step_x != step_y or step_x == 0:
        return False
    gap = (b - a) % step_x
    return gap >= row_x and gap + row_y <= step_x


def _check_out(out: torch.Tensor, like: torch.Tensor, name: str, others) -> None:
    """An output is ``like``'s shape, dtype and device, and see _check_place."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must have the shape, dtype and device of its input")
    _check_place(out, like, name, others)


def _check_place(out: torch.Tensor, like: torch.Tensor, name: str, others=()) -> None:
    """An output writes no element twice, is either exactly its input ``like``
    or apart from it, and is apart from the others (one tensor given as two
    inputs would be written as the one and read as the other)."""
    if out.numel() == 0:
        return
    # A permutation of contiguous rows, or rows apart: no element twice.
    extent = 0
    for stride, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        if stride <= extent:
            raise ValueError(f"{name} must not overlap itself")
        extent += stride * (n - 1)
    same = (like.dtype == out.dtype and like.data_ptr() == out.data_ptr()
            and like.stride() == out.stride())
    if not (same or _apart(out, like)) or not all(_apart(out, t) for t in others):
        raise ValueError(f"{name} must be its input itself or not overlap the inputs")


def _rope_fields(q, k, v, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, k_out,
                 status):
    """Checks the arguments both ops share (v is None: no append); returns the
    fields of _lib.QkNormRopeArgs, the outputs and the device."""
    if not q.is_cuda:
        raise ValueError("CUDA q required for the b200 backend")
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError("q must have shape [T,Hq,D] and k [T,Hkv,D]")
    t, hq, d = q.shape
    kt, hkv, kd = k.shape
    if kt != t or kd != d:
        raise ValueError("q and k must agree in tokens and head dimension")
    if hq == 0 or hkv == 0 or d == 0:
        raise ValueError("q and k dimensions must be nonzero")
    dtype = q.dtype
    if dtype not in _DTYPES or k.dtype != dtype:
        raise ValueError("q and k must share a dtype: float32, bfloat16 or float16")
    index = q.get_device()
    if positions.dtype not in _INDEX or positions.shape != (t,):
        raise ValueError("positions must be a [T] integer tensor")
    if cos_sin.dtype != torch.float32 or cos_sin.ndim != 2 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous [positions, rotary_dim] float32 tensor")
    rows, rot = cos_sin.shape
    if rot < 2 or rot % 2 or rot > d:
        raise ValueError("rotary_dim must be even and in [2, D]")
    if rows == 0:
        raise ValueError("cos_sin must have at least one row")
    if (k.get_device() != index or positions.get_device() != index
            or cos_sin.get_device() != index):
        raise ValueError("all inputs must reside on same CUDA device")
    wdtype = qw = kw = 0
    weight = k_weight if q_weight is None else q_weight
    if weight is not None:
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (d,) or w.dtype not in _DTYPES
                                  or w.dtype != weight.dtype or not w.is_contiguous()
                                  or w.get_device() != index):
                raise ValueError("norm weights must be contiguous [D] tensors of one float dtype "
                                 "on the q device")
        wdtype = _DTYPES[weight.dtype]
        qw = 0 if q_weight is None else q_weight.data_ptr()
        kw = 0 if k_weight is None else k_weight.data_ptr()
    if not eps > 0:
        raise ValueError("eps must be positive")
    sp = 0 if status is None else _status_ptr(status, index)
    if q_out is not None:
        _check_out(q_out, q, "q_out", (k,) if v is None else (k, v))
        qs = q_out.stride()
    else:
        q_out = q.new_empty((t, hq, d))
        qs = (hq * d, d, 1)
    kp = 0
    ks = (0, 0, 0)
    if v is None:
        if k_out is not None:
            _check_out(k_out, k, "k_out", (q, q_out))
            ks = k_out.stride()
        else:
            k_out = k.new_empty((t, hkv, d))
            ks = (hkv * d, d, 1)
        kp = k_out.data_ptr()
    fields = (t, hq, hkv, d, q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), q_out.data_ptr(),
              *qs, kp, *ks, qw, kw, cos_sin.data_ptr(), rows, rot, positions.data_ptr(),
              *positions.stride(), sp, _DTYPES[dtype], wdtype, _INDEX[positions.dtype],
              1 if interleaved else 0, eps, 0)
    return fields, q_out, k_out, index


def qk_norm_rope_b200(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                      cos_sin: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                      k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                      interleaved: bool = False, q_out: torch.Tensor | None = None,
                      k_out: torch.Tensor | None = None, status: torch.Tensor | None = None,
                      prepare: bool = False):
    """RMS norm of every head of q and k, then the rotation to ``positions``.

    q: [T, Hq, D], k: [T, Hkv, D] (any strides, one float dtype, D <= 256);
    positions: [T] integers, rows of ``cos_sin`` ([positions, R] float32, see
    :func:`rope_table`; the first R elements of a head are rotated).  With
    q_weight / k_weight ([D]) a head x becomes
    ``x * rsqrt(mean(x*x) + eps) * weight`` first; without one it is only
    rotated.  ``interleaved`` rotates the pairs (2i, 2i+1) instead of
    (i, i + R/2).  Computed in float32, rounded once.

    Returns (q_out, k_out), fresh tensors unless given; q_out may be q itself
    and k_out k itself.  A token whose position lies outside the table gets
    zero rows and sets DEV_BAD_POSITION in ``status``.
    """
    _inference_only(q, k, cos_sin, q_weight, k_weight)
    lib = _lib.load()
    fields, q_out, k_out, index = _rope_fields(q, k, None, positions, cos_sin, q_weight, k_weight,
                                               eps, interleaved, q_out, k_out, status)
    args = _PACK_ROPE(*fields)
    if prepare:
        return _DeviceCall(lib.b200_qk_norm_rope, args, index, (q_out, k_out),
                           "head norm and rotation",
                           (q, k, positions, cos_sin, q_weight, k_weight, status))
    _launch(lib.b200_qk_norm_rope, args, index, "head norm and rotation")
    return q_out, k_out


def rope_kv_append_b200(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pool, slot_mapping,
                        positions: torch.Tensor, cos_sin: torch.Tensor, layer_idx: int, *,
                        q_weight: torch.Tensor | None = None,
                        k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        interleaved: bool = False, q_out: torch.Tensor | None = None,
                        status: torch.Tensor | None = None, prepare: bool = False):
    """:func:`qk_norm_rope_b200` with k and v appended to the paged KV pool.

    pool[layer, slot // S, slot % S] = normed and rotated k / v as it is, for
    each of the T tokens, rounded once to the pool's dtype (float32 or
    bfloat16); v: [T, Hkv, D]; slot_mapping: [T] integer CUDA tensor or (not
    while a graph is captured) a host sequence.  Returns the normed and rotated q ([T, Hq, D], in q.dtype).

    A slot outside the pool, or a position outside the table, skips that
    token's k and v and sets DEV_BAD_SLOT / DEV_BAD_POSITION in ``status``.
    Slots of one call are distinct, except those that nothing reads (padding
    rows that share a scratch slot); q, k and v are not views of the pool's
    slots that the call writes.
    """
    _inference_only(q, k, v, cos_sin, q_weight, k_weight)
    lib = _lib.load()
    if v.shape != k.shape or v.dtype != k.dtype or v.get_device() != k.get_device():
        raise ValueError("k and v must have matching shape [T,Hkv,D], dtype and device")
    fields, q_out, _, index = _rope_fields(q, k, v, positions, cos_sin, q_weight, k_weight, eps,
                                           interleaved, q_out, None, status)
    pool_fields = _pool_fields(pool, index, layer_idx)
    if pool_fields[5] != fields[2] or pool_fields[6] != fields[3]:
        raise ValueError("k/v head dimensions do not match the KV pool")
    slots = _index_arg(slot_mapping, q.device, index, "slot_mapping")
    if slots.shape != (fields[0],):
        raise ValueError("slot_mapping must have shape [T]")
    args = _PACK_APPEND(*fields, *pool_fields, layer_idx, v.data_ptr(), *v.stride(),
                        slots.data_ptr(), *slots.stride(), _INDEX[slots.dtype], 0)
    if prepare:
        return _DeviceCall(lib.b200_rope_kv_append, args, index, q_out, "rotary KV append",
                           (q, k, v, pool.k, pool.v, slots, positions, cos_sin, q_weight, k_weight,
                            status))
    _launch(lib.b200_rope_kv_append, args, index, "rotary KV append")
    return q_out
