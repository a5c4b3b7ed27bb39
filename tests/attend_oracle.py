"""Attention in 64 bits over given keys and values, and two measures of a result that are tight enough to see one
token too many or too few; with data on which they do.

Data.  Keys, queries and values are standard normal, so that scores (q . k / sqrt(128)) have a standard deviation of
one and no token dominates; one value in a hundred, and those at the masks' and the kernels' borders, are 50 times as large.
A row that sees n tokens then has an output of about 5 / sqrt(n) of a value's size, in which a large value has a part
of 50 / n: a hundredth of the output at n = 10^6, more where n is less.

Measures.  ``by_head``: the 2-norm of the error over all rows and channels of a query head, relative to the output's.  For 16-bit
types half a step of the type, eps / 2: the output's own rounding has 0.42 of that in the mean square (an error even over half a
step, relative to a mantissa even over [1, 2)).  Bfloat16 (2^-8) meets probabilities, values and keys as half-precision numbers
(2^-11 at worst, 0.42 of that in the mean square; a score is off by the root of 128 such products / sqrt(128), that is by as much): three
times 0.42 / 8, added as squares, 0.1 of eps / 2.  Float16 (2^-11) meets keys and values as pairs, and its probabilities are rounded once:
0.6 with the output's.  float32: 2^-20, four pairs of half-precision parts (2^-22 each) at worst.
``by_row``: the same of every row by itself, within eps / 2 + 2^-10: the output's rounding, a probability's and a value's at their worst
and of one sign; float32: 2^-19.
"""

from __future__ import annotations

import math

import torch

LARGE = 50.0


def limits(dtype):
    if dtype == torch.float32:
        return 2.0**-20, 2.0**-19
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).eps / 2 + 2.0**-10


def values(n, heads, gen, device, borders=()):
    """``[n, heads, 128]``, with the large ones."""
    v = torch.randn(n, heads, 128, generator=gen, device=device)
    large = torch.rand(n, generator=gen, device=device) < 0.01
    for at in borders:
        if 0 <= at < n:
            large[at] = True
    return v * torch.where(large, LARGE, 1.0)[:, None, None]


def borders(n, t, window, sinks, blocks):
    """Positions where a mask or a kernel's division may be off by one."""
    at = {0, 1, n - 2, n - 1, sinks - 1, sinks, blocks - 1, blocks}
    for p in (n - t, n - t + 1, n - 1):
        at |= {p, p - 1, p + 1, p - (window or 0), p - (window or 0) + 1, p - (window or 0) - 1}
    for size in (32, 64, 80, 100, 256):
        at |= {size - 1, size, (n // size) * size, (n // size) * size - 1, blocks // size * size}
    return sorted(at)


def attention(k, v, q, q_n, window, sinks, hidden=()):
    """``[T, Hq, 128]`` in 64 bits, for queries that belong to the newest ``q_n`` tokens; tokens of ``hidden`` are left out."""
    n, t = k.shape[1], q.shape[0]
    p = n - q_n + torch.arange(t, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)
    sees = (j <= p) & (torch.arange(t, device=q.device) < q_n)[:, None]
    if window is not None:
        sees &= (j > p - window) | (j < sinks)
    for span in hidden:
        sees[:, span] = False
    g, out = q.shape[1] // k.shape[0], []
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[h // g].double().t() / math.sqrt(q.shape[2])
        pr = torch.softmax(s.masked_fill(~sees, -math.inf), 1).masked_fill(~sees.any(1)[:, None], 0.0)
        out.append(pr @ v[h // g].double())
    return torch.stack(out, 1)


def measures(got, want):
    off = got.double() - want
    head = off.norm(dim=(0, 2)) / want.norm(dim=(0, 2)).clamp_min(1e-300)
    row = off.norm(dim=2) / want.norm(dim=2).clamp_min(1e-300)
    return float(head.max()), float(row.max())


def check(got, want):
    head, row = measures(got, want)
    most_head, most_row = limits(got.dtype)
    assert head <= most_head and row <= most_row, (head / most_head, row / most_row)


# float16 queries with scores of standard deviation four: the output's rounding and, at worst, that of the probabilities
# are 0.42 of eps / 2 each in the mean square, 0.6 together.  Keys of half precision without a low part would move scores by
# 0.42 * 4 = 1.7, less what a row's heaviest tokens, which then have most of its weight, have in common.
PAIRS = 0.75 * torch.finfo(torch.float16).eps / 2
