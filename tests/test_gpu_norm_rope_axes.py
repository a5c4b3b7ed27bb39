"""norm_rope with positions of several axes against the formula in 64 bits, and behind a prefix.

Tolerance: that of one axis.  The result is rounded once, by at most eps/2 of its value; before that 2^-17 of the pair's length
stands for the float32 arithmetic (a sum of 128 squares, a root, sines and cosines, two products and a sum).
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


def _check(torch, got, x, weight, inv_freq, positions, axes, eps=1e-6):
    """``positions`` ``[n_axes, n, T]``."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    h = inv_freq.numel()
    of = torch.stack([positions[min(a, len(positions) - 1)] for a in axes], -1) if h else positions[0][..., None][..., :0]
    a = (of.double() * inv_freq.double())[..., None, :]
    lo, hi, rest = y[..., :h], y[..., h:2 * h], y[..., 2 * h:]
    want = torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), rest), -1)
    size = torch.sqrt(lo * lo + hi * hi)
    size = torch.cat((size, size, rest.abs()), -1)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0**-17 * size + torch.finfo(x.dtype).tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def _freq(torch, rotary_dim, theta=1000000.0):
    h = rotary_dim // 2
    return torch.tensor(theta ** (-np.arange(h) / max(h, 1)), dtype=torch.float32, device="cuda")


def _axes(torch, of):
    return torch.tensor(of, dtype=torch.uint8, device="cuda")


RUNS, TURNS = [0] * 16 + [1] * 24 + [2] * 24, [i % 3 for i in range(64)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, t, hq, hk, axes, start", [
    (1, 1, 28, 4, RUNS, 5000), (3, 37, 5, 1, TURNS, 2**28), (2, 700, 4, 2, [0] * 32 + [1] * 32, -900),
    (1, 5, 3, 3, [1, 0, 1, 0], 7), (2, 3, 2, 1, [], 3), (1, 9, 2, 2, [0] * 48, 10)])
def test_matches_the_formula(torch, dtype, n, t, hq, hk, axes, start):
    from turboquant_pro_b200 import norm_rope

    gen = torch.Generator(device="cuda").manual_seed(n * 100 + t)
    dt = getattr(torch, dtype)
    qkv = torch.randn(n, t, hq + 2 * hk, 128, generator=gen, device="cuda").mul_(3).to(dt)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    f, ax = _freq(torch, 2 * len(axes)), _axes(torch, axes)
    pos = start + torch.randint(0, 90, (max(axes, default=0) + 1, n, t), generator=gen, device="cuda")
    w = torch.rand(128, generator=gen, device="cuda").add_(0.5).to(dt)
    for qw, kw in ((w, w * 0.5), (None, w), (None, None)):
        gq, gk = norm_rope(q, k, f, pos, q_weight=qw, k_weight=kw, axes=ax)
        _check(torch, gq, q, qw, f, pos, axes)
        _check(torch, gk, k, kw, f, pos, axes)


def test_orders_and_types_of_the_positions(torch):
    from turboquant_pro_b200 import norm_rope

    q, k = torch.randn(2, 5, 3, 128, device="cuda"), torch.randn(2, 5, 1, 128, device="cuda")
    f, ax = _freq(torch, 128), _axes(torch, RUNS)
    one = torch.randint(0, 1000, (3, 5), device="cuda")
    each = torch.randint(0, 1000, (3, 2, 5), device="cuda")
    last = each.permute(1, 2, 0).contiguous().permute(2, 0, 1)  # a token's axes side by side
    for p in (one, one.int(), each, each.int(), last, one[:, None].expand(3, 2, 5), each[:, :, ::2].repeat_interleave(2, 2)[:, :, :5]):
        gq, gk = norm_rope(q, k, f, p, axes=ax)
        full = p[:, None].expand(3, 2, 5) if p.dim() == 2 else p
        _check(torch, gq, q, None, f, full, RUNS)
        _check(torch, gk, k, None, f, full, RUNS)


def test_axes_that_are_all_one_are_the_one(torch):
    from turboquant_pro_b200 import norm_rope

    q, k = (torch.randn(2, 40, h, 128, device="cuda").bfloat16() for h in (6, 2))
    f, pos = _freq(torch, 96), torch.randint(0, 10**6, (2, 40), device="cuda")
    want = norm_rope(q, k, f, pos)
    for p, ax in ((pos.expand(3, 2, 40), [2, 1, 0] * 16), (torch.stack((pos + 1, pos)), [1] * 48), (pos[None], [0] * 48)):
        got = norm_rope(q, k, f, p, axes=_axes(torch, ax))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_numbers_beyond_the_axes_count_as_the_last(torch):
    from turboquant_pro_b200 import norm_rope

    q = torch.randn(1, 4, 2, 128, device="cuda")
    f, pos = _freq(torch, 16), torch.randint(0, 10**6, (2, 1, 4), device="cuda")
    gq, _ = norm_rope(q, q, f, pos, axes=_axes(torch, [0, 1, 2, 255, 7, 0, 1, 1]))
    _check(torch, gq, q, None, f, pos, [0, 1, 1, 1, 1, 0, 1, 1])


def test_nothing_to_turn(torch):
    from turboquant_pro_b200 import norm_rope

    f, ax = _freq(torch, 128), _axes(torch, RUNS)
    for n, t in ((0, 3), (2, 0)):
        q, k = torch.empty(n, t, 4, 128, device="cuda"), torch.empty(n, t, 2, 128, device="cuda")
        gq, gk = norm_rope(q, k, f, torch.empty(3, n, t, dtype=torch.long, device="cuda"), axes=ax)
        assert gq.shape == q.shape and gk.shape == k.shape


def test_refusals(torch):
    from turboquant_pro_b200 import norm_rope

    q, k = torch.randn(2, 5, 4, 128, device="cuda"), torch.randn(2, 5, 2, 128, device="cuda")
    f, ax, pos = _freq(torch, 128), _axes(torch, RUNS), torch.zeros(3, 2, 5, dtype=torch.long, device="cuda")
    for bad in (dict(axes=ax[:63]), dict(axes=ax.int()), dict(axes=ax.view(2, 32)), dict(axes=ax.cpu()),
                dict(positions=pos[:, :1]), dict(positions=pos[0, 0]), dict(positions=pos[:0]),
                dict(positions=pos.float()), dict(positions=pos[None])):
        with pytest.raises(ValueError):
            norm_rope(q, k, f, **{"positions": pos, "axes": ax, **bad})


def test_positions_behind_a_prefix(torch):
    from turboquant_pro_b200 import KVContext, norm_rope

    ctx = KVContext(n_layers=2, n_seqs=4, n_kv_heads=2, n_q_heads=4, max_tokens_per_seq=1024, kv_dtype="float16", seed=1)
    for s, n in enumerate((700, 3, 0, 20)):
        if n:
            x = torch.randn(1, n, 2, 128, device="cuda").half()
            ctx.append(1, x, x, seq_begin=s)
    q, k = torch.randn(2, 3, 4, 128, device="cuda").half(), torch.randn(2, 3, 2, 128, device="cuda").half()
    f = _freq(torch, 128)
    got = ctx.norm_rope(1, q, k, f, seq_begin=1, prefix=0)
    at = torch.tensor([[703], [700]], device="cuda") + torch.arange(3, device="cuda")
    want = norm_rope(q, k, f, at)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="prefix"):
        ctx.norm_rope(1, q, k, f, seq_begin=0, prefix=1)
    with pytest.raises(ValueError, match="prefix"):
        ctx.norm_rope(1, q, k, f, seq_begin=0, prefix=4)
    with pytest.raises(ValueError, match="positions"):
        ctx.norm_rope(1, q, k, f, at, seq_begin=1, prefix=0)
    # positions of several axes through the context
    ax, pos = _axes(torch, TURNS), torch.randint(0, 99, (3, 2, 3), device="cuda")
    got, want = ctx.norm_rope(1, q, k, f, pos, axes=ax), norm_rope(q, k, f, pos, axes=ax)
    assert torch.equal(got[0], want[0])
    with pytest.raises(ValueError, match="axes"):
        ctx.norm_rope(1, q, k, f, axes=ax)
