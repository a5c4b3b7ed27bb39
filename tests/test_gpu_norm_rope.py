"""norm_rope against the formula in 64 bits.

Tolerance: the result is rounded once, by at most eps/2 of its value.  Before that the norm (a sum of 128
squares, a root, two products), the sines and cosines and two products and a sum are float32: with u =
2^-24, at most (64 + 8) u of the larger of the pair's values each, for which 2^-17 of the pair's length stands.
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


def _want(torch, x, weight, inv_freq, positions, eps):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    a = positions.double()[..., None, None] * inv_freq.double()
    h = inv_freq.numel()
    lo, hi, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    size = torch.sqrt(lo * lo + hi * hi)
    return (torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), rest), -1),
            torch.cat((size, size, rest.abs()), -1))


def _check(torch, got, x, weight, inv_freq, positions, eps=1e-6):
    want, size = _want(torch, x, weight, inv_freq, positions, eps)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0**-17 * size + torch.finfo(x.dtype).tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def _freq(torch, rotary_dim, theta=10000.0):
    h = rotary_dim // 2
    return torch.tensor(theta ** (-np.arange(h) / max(h, 1)), dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, t, hq, hk, rotary, start", [
    (1, 1, 32, 8, 128, 8191), (3, 7, 5, 1, 64, 0), (2, 33, 28, 4, 96, 2**28), (1, 5, 1, 1, 8, 1000000),
    (1, 2, 70, 3, 0, 3), (2, 1, 64, 64, 128, -17)])
def test_matches_the_formula(torch, dtype, n, t, hq, hk, rotary, start):
    from turboquant_pro_b200 import norm_rope

    gen = torch.Generator(device="cuda").manual_seed(n * 100 + t)
    dt = getattr(torch, dtype)
    # a fused projection's views, rows of other widths between the heads of two tokens
    qkv = torch.randn(n, t, hq + 2 * hk, 128, generator=gen, device="cuda").mul_(3).to(dt)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    f = _freq(torch, rotary)
    pos = start + torch.arange(n * t, device="cuda").view(n, t)
    w = torch.rand(128, generator=gen, device="cuda").add_(0.5).to(dt)
    for qw, kw in ((w, w * 0.5), (None, w), (None, None)):
        gq, gk = norm_rope(q, k, f, pos, q_weight=qw, k_weight=kw)
        _check(torch, gq, q, qw, f, pos)
        _check(torch, gk, k, kw, f, pos)


def test_positions_of_one_row_and_of_32_bits(torch):
    from turboquant_pro_b200 import norm_rope

    q, k = torch.randn(3, 4, 2, 128, device="cuda"), torch.randn(3, 4, 1, 128, device="cuda")
    f = _freq(torch, 128)
    pos = torch.tensor([5, 900000, 2, 77], device="cuda")
    for p in (pos, pos.int(), pos.int().expand(3, 4), pos.repeat(2, 1).t()[:, 0]):
        gq, gk = norm_rope(q, k, f, p)
        _check(torch, gq, q, None, f, pos.expand(3, 4))
        _check(torch, gk, k, None, f, pos.expand(3, 4))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_off_the_vector_grid_and_other_orders(torch, dtype):
    from turboquant_pro_b200 import norm_rope

    dt = getattr(torch, dtype)
    flat = torch.randn(2 * 3 * 5 * 128 + 1, device="cuda").to(dt)
    q = flat[1:].view(2, 3, 5, 128)                                # one element off
    k = torch.randn(2, 4, 3, 128, device="cuda").to(dt).permute(0, 2, 1, 3)  # heads before tokens
    wide = torch.randn(2, 3, 5, 131, device="cuda").to(dt)[..., 2:130]
    turned = torch.randn(2, 3, 128, 5, device="cuda").to(dt).transpose(2, 3)  # channels not contiguous
    f, w = _freq(torch, 64), torch.rand(128, device="cuda").to(dt)
    pos = torch.arange(6, device="cuda").view(2, 3)
    for x in (q, wide, turned):
        gq, gk = norm_rope(x, k, f, pos, q_weight=w, k_weight=w, eps=0.25)
        _check(torch, gq, x, w, f, pos, 0.25)
        _check(torch, gk, k, w, f, pos, 0.25)


def test_zero_rows_and_large_values(torch):
    from turboquant_pro_b200 import norm_rope

    q = torch.randn(1, 3, 2, 128, device="cuda")
    q[0, 0] = 0.0
    q[0, 1] *= 1e15
    q[0, 2] *= 1e-15
    f, w, pos = _freq(torch, 128), torch.ones(128, device="cuda"), torch.arange(3, device="cuda")
    gq, _ = norm_rope(q, q, f, pos, q_weight=w)
    _check(torch, gq, q, w, f, pos)
    assert bool((gq[0, 0] == 0).all())
    q[0, 2, 1, 5] = float("nan")
    gq, gk = norm_rope(q, q, f, pos, q_weight=w)
    assert bool(gq[0, 2, 1].isnan().all()) and not bool(gq[0, 2, 0].isnan().any())
    assert int(gk.isnan().sum()) == 2  # without the norm, the pair it turns with


def test_empty_calls(torch):
    from turboquant_pro_b200 import norm_rope

    f = _freq(torch, 128)
    for n, t in ((0, 3), (2, 0)):
        q, k = (torch.randn(n, t, h, 128, device="cuda") for h in (4, 2))
        gq, gk = norm_rope(q, k, f, torch.zeros(n, t, dtype=torch.long, device="cuda"))
        assert gq.shape == q.shape and gk.shape == k.shape


def test_positions_of_a_cache_follow_its_lengths_under_replay(torch):
    from turboquant_pro_b200 import KVContext

    ctx = KVContext(n_layers=2, n_seqs=3, n_kv_heads=1, n_q_heads=2, hot_window=16, max_tokens_per_seq=64,
                    kv_dtype="bfloat16", seed=0)
    tok = lambda n, t, h: torch.randn(n, t, h, 128, device="cuda").bfloat16()  # noqa: E731
    ctx.append(1, tok(1, 20, 1), tok(1, 20, 1), seq_begin=1)
    ctx.append(1, tok(1, 3, 1), tok(1, 3, 1), seq_begin=2)
    f = _freq(torch, 128)
    q, k = tok(2, 4, 2), tok(2, 4, 1)
    pos = torch.tensor([[20], [3]], device="cuda") + torch.arange(4, device="cuda")
    gq, gk = ctx.norm_rope(1, q, k, f, seq_begin=1)
    _check(torch, gq, q, None, f, pos)
    _check(torch, gk, k, None, f, pos)
    given = ctx.norm_rope(1, q, k, f, pos + 5, seq_begin=1)
    _check(torch, given[0], q, None, f, pos + 5)
    ctx.norm_rope(0, tok(3, 1, 2), tok(3, 1, 1), f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gq, gk = ctx.norm_rope(1, q, k, f, seq_begin=1)
    ctx.append(1, tok(2, 7, 1), tok(2, 7, 1), seq_begin=1)
    graph.replay()
    torch.cuda.synchronize()
    _check(torch, gk, k, None, f, pos + 7)


def test_refusals(torch):
    from turboquant_pro_b200 import KVContext, norm_rope

    q, k = torch.zeros(1, 3, 4, 128, device="cuda"), torch.zeros(1, 3, 2, 128, device="cuda")
    f, p = torch.zeros(64, device="cuda"), torch.arange(3, device="cuda")
    w = torch.ones(128, device="cuda")
    for bad in (dict(k=k.half()), dict(k=k.cpu()), dict(inv_freq=f.double()), dict(inv_freq=f[:, None]),
                dict(positions=p.float()), dict(positions=p[:2]), dict(positions=p.cpu()),
                dict(q_weight=w[:64]), dict(q_weight=w, k_weight=w.half()), dict(eps=-1.0),
                dict(q=q.double(), k=k.double()), dict(q=q.clone().requires_grad_())):
        args = {"q": q, "k": k, "inv_freq": f, "positions": p, **bad}
        with pytest.raises(ValueError):
            norm_rope(args.pop("q"), args.pop("k"), args.pop("inv_freq"), args.pop("positions"), **args)
    with pytest.raises(NotImplementedError):
        norm_rope(q, k, f[:6], p)
    with pytest.raises(NotImplementedError):
        norm_rope(q, k, torch.zeros(68, device="cuda"), p)
    ctx = KVContext(n_seqs=2, n_kv_heads=2, n_q_heads=4, hot_window=16, max_tokens_per_seq=32)
    for bad in (dict(layer=1), dict(seq_begin=2), dict(seq_begin=-1), dict(q=q[:, :, :2])):
        args = {"layer": 0, "q": q, "seq_begin": 0, **bad}
        with pytest.raises(ValueError):
            ctx.norm_rope(args["layer"], args["q"], k, f, seq_begin=args["seq_begin"])
