"""Helpers of the tests of extend and cross attention: 64-bit values and the bound a
bf16 kernel has to keep.

The output is rounded to bf16 once (half a step, 2^-8 of the value). Every weight p is
rounded before it meets V: to 16 bits in groups, to bf16 in tiles (2^-8 of p, so at
most 2^-8 of sum p |v| / sum p). Scores of up to some 30 (log2) with 128 products each,
their sums and the exponential in 32 bits move a weight by less than 2^-13."""
from __future__ import annotations

import torch

import serve_refs as R


def bound(want, size, tiles):
    return 2.0 ** -8 * want.abs() + ((2.0 ** -8 if tiles else 0.0) + 2.0 ** -13) * size


def rows_of(q, k, v, limits, scale):
    """64-bit attention of rows q [n][hq][128] over keys 0..limits[n] - 1 of k and v [keys][hk][128]: (out, sum p |v| / sum p)."""
    n, hq, _ = q.shape
    hk = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(n, hq, 128, dtype=torch.float64)
    size = torch.zeros_like(out)
    for i in range(n):
        lim = max(0, int(limits[i]))
        if lim:
            o, s = R.attend(q[i], k[:lim], v[:lim], scale)
            out[i], size[i] = o, s
    return out, size
