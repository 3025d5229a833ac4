"""Plain 64-bit forms of the head norms, the rotation and the KV append, and
the tolerance their float32 kernels are held to."""
from __future__ import annotations

import torch

EPS = 1e-6


def norm_rope(x, positions, cos_sin, weight=None, eps=EPS, interleaved=False):
    """[T, H, D] in float64: the norm (with a weight), then the rotation.
    Rows whose position lies outside the table are zero."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    rot = cos_sin.shape[1]
    ok = (positions >= 0) & (positions < cos_sin.shape[0])
    row = cos_sin.double()[positions.clamp(0, cos_sin.shape[0] - 1).long()][:, None]
    c, s = row[..., : rot // 2], row[..., rot // 2:]
    out = x.clone()
    ia, ib = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved
              else (slice(0, rot // 2), slice(rot // 2, rot)))
    out[..., ia] = x[..., ia] * c - x[..., ib] * s
    out[..., ib] = x[..., ia] * s + x[..., ib] * c
    return torch.where(ok[:, None, None], out, 0.0)


def bound(want, dtype, rot, interleaved):
    """Largest error of one rounding to ``dtype`` after float32 arithmetic.

    The rounding: half a step, eps/2 of the value (2^-25 absolute among fp16's
    subnormals).  The arithmetic, relative to |a| + |b| of a rotated pair: the
    sum of at most 256 squares in chains of at most 16 with at most 5
    reduction steps, halved by the root (11 * 2^-24), rsqrtf (2 ulp: 4 * 2^-24),
    mean + eps, inv * w and * x (3), the rotation's products and sum (3), the
    table's own values are inputs: 21 * 2^-24 < 2^-19."""
    half = torch.finfo(dtype).eps / 2
    pair = want.abs().clone()
    ia, ib = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved
              else (slice(0, rot // 2), slice(rot // 2, rot)))
    both = (want[..., ia].square() + want[..., ib].square()).sqrt() * 2 ** 0.5  # >= |a| + |b|
    pair[..., ia] = both
    pair[..., ib] = both
    # The rounding acts on the computed value: (1 + half) covers its own error.
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    return half * want.abs() + (1 + half) * 2.0 ** -19 * pair + tiny


def assert_close(got, want, dtype, rot, interleaved, what):
    err = (got.double().cpu() - want.cpu()).abs()
    lim = bound(want.cpu(), dtype, rot, interleaved)
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {float((err / lim).max()):.2f} of it"
