"""KVContext.attend against attention in 64 bits over the dequantised keys and values (the getters, which
are bit-exact with the reference's decoders).

Tolerance.  With u the relative step of the operands of the kernels' products (float32: 2^-22, a pair of
half-precision parts; 16-bit queries: 2^-11, a half-precision number, twice its rounding) a score is off by
at most u * A, A the largest sum of |q_d k_d| / sqrt(D) of a visible token (keys taken from their mean
over the tokens where that is smaller, or not); a probability by that part of itself, twice (its sum is off, too) and
a rounding u of its own; a value by u.  So an output is off by at most (2 u A + 4 u) * max |v| over the visible
tokens, and by its own rounding, eps / 2.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


def _fill(torch, ctx, lens, gen, layer=0, spread=3.0):
    h = ctx.n_kv_heads
    scale = torch.exp(0.5 * torch.randn(h, 128, generator=gen, device="cuda"))
    scale[:, :2] *= 8.0
    shift = torch.randn(h, 128, generator=gen, device="cuda") * (torch.arange(128, device="cuda") % 8 == 0)
    for s, n in enumerate(lens):
        if n:
            k = torch.randn(1, n, h, 128, generator=gen, device="cuda") * scale + spread * shift
            v = torch.randn(1, n, h, 128, generator=gen, device="cuda")
            ctx.append(layer, k.to(ctx.kv_dtype), v.to(ctx.kv_dtype), seq_begin=s)


def _want(torch, ctx, layer, seq, q, q_n, window, sinks):
    """Output and its bound (without the rounding) for the queries ``[T, Hq, D]`` of one sequence."""
    n = ctx.lengths(layer, seq)[0]
    t, hq, d = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device="cuda")
    bound = torch.zeros(t, hq, 1, dtype=torch.float64, device="cuda")
    if n == 0:
        return out, bound
    u = 2.0**-22 if q.dtype == torch.float32 else 2.0**-11
    k, v = (x.double() for x in ctx.dequant(layer, seq, 0, n))
    p = n - q_n + torch.arange(t, device="cuda")
    j = torch.arange(n, device="cuda")
    sees = (j <= p[:, None]) & (torch.arange(t, device="cuda") < q_n)[:, None]
    if window is not None:
        sees &= (j > p[:, None] - window) | (j < sinks)
    g = hq // ctx.n_kv_heads
    for h in range(hq):
        qk = q[:, h].double()
        s = (qk @ k[h // g].t() / math.sqrt(d)).masked_fill(~sees, -math.inf)
        pr = torch.softmax(s, 1).masked_fill(~sees.any(1)[:, None], 0.0)
        out[:, h] = pr @ v[h // g]
        a = (qk.abs() @ k[h // g].abs().t() / math.sqrt(d)).masked_fill(~sees, 0.0).amax(1)
        top = v[h // g].abs().amax(1)[None].masked_fill(~sees, 0.0).amax(1)
        bound[:, h, 0] = (2 * a + 4) * u * top
    return out, bound


def _check(torch, ctx, got, q, window=None, sinks=0, q_lens=None, seq_begin=0, layer=0):
    assert got.shape == q.shape and got.dtype == q.dtype
    for s in range(q.shape[0]):
        q_n = q.shape[1] if q_lens is None else int(q_lens[s])
        want, bound = _want(torch, ctx, layer, seq_begin + s, q[s], q_n, window, sinks)
        off = (got[s].double() - want).abs()
        limit = bound + torch.finfo(q.dtype).eps / 2 * want.abs()
        bad = ~(off <= limit)
        assert not bool(bad.any()), (s, bad.nonzero()[:4].tolist(), float((off / limit.clamp_min(1e-30)).max()))


def _ctx(**kw):
    from turboquant_pro_b200 import KVContext

    return KVContext(**{"n_layers": 1, "seed": 3, "max_tokens_per_seq": 4096, **kw})


CASES = [
    # lens, T, Hkv, Hq, window, sinks, kv dtype, q dtype, hot, keys, value bits
    ([700], 1, 2, 8, None, 0, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([1500, 3, 0, 800], 1, 2, 8, 300, 4, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([1500, 513, 900], 1, 1, 5, 1, 0, "float16", "float16", 512, "nf4_asym", 4),
    ([2100, 40], 1, 2, 2, 700, 1, "float32", "float32", 512, "nf4_asym", 4),
    ([2100, 515], 4, 2, 14, 600, 300, "float32", "float32", 512, "uniform", 3),
    ([1025, 5, 0], 7, 1, 8, None, 0, "bfloat16", "float16", 512, "nf4", 3),
    ([1300, 2000], 33, 2, 8, None, 0, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([1300, 20], 33, 1, 16, 100, 7, "float16", "float16", 512, "uniform", 4),
    ([1999], 130, 2, 6, 513, 4, "float16", "bfloat16", 512, "nf4_asym", 4),
    ([3500], 301, 1, 4, None, 0, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([3500], 301, 1, 7, 1000, 130, "bfloat16", "float16", 512, "nf4_asym", 3),
    ([600, 601], 600, 1, 3, None, 0, "float16", "float16", 512, "nf4_asym", 3),
    ([100, 333], 400, 2, 2, 64, 2, "bfloat16", "bfloat16", 512, "nf4", 4),
    ([300, 17], 19, 1, 2, 50, 3, "float16", "float16", 33, "nf4_asym", 3),
    ([300, 301], 70, 2, 4, None, 0, "bfloat16", "bfloat16", 33, "uniform", 4),
    ([260], 1, 1, 4, None, 0, "bfloat16", "bfloat16", 2, "nf4_asym", 4),
    ([500], 9, 1, 4, 90, 5, "float32", "float32", 100, "nf4_asym", 3),
    ([700, 130], 21, 1, 4, 200, 5, "float16", "float16", 128, "polar", 4),
    ([700, 130], 1, 2, 4, None, 0, "float32", "float32", 512, "polar", 3),
    ([900], 150, 1, 2, None, 0, "bfloat16", "bfloat16", 256, "nf4_asym", 3),
    ([512, 511, 513], 2, 1, 1, 4096, 4096, "float16", "float16", 512, "nf4_asym", 3),
]


def _build(torch, case, seed):
    lens, t, h, hq, window, sinks, kv, qd, hot, keys, vb = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx = _ctx(n_seqs=len(lens), n_kv_heads=h, n_q_heads=hq, kv_dtype=kv, hot_window=hot, key_mode=keys,
               value_bits=vb, key_bits=vb if keys == "polar" else 4, outlier_frac=0.0 if keys == "polar" else 0.02)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(len(lens), t, hq, 128, generator=gen, device="cuda").to(getattr(torch, qd))
    return ctx, q, gen


@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_attention_in_64_bits(torch, case):
    ctx, q, gen = _build(torch, case, 7)
    window, sinks = case[4], case[5]
    got = ctx.attend(0, q, window=window, sinks=sinks)
    _check(torch, ctx, got, q, window, sinks)
    assert ctx.status() == 0
    # padded: other numbers of query tokens, one of them none
    q_lens = torch.tensor([(i * 7 + 3) % (q.shape[1] + 1) for i in range(q.shape[0])], dtype=torch.int32,
                          device="cuda")
    got = ctx.attend(0, q, window=window, sinks=sinks, q_lens=q_lens)
    _check(torch, ctx, got, q, window, sinks, q_lens)
    for s, r in enumerate(q_lens.tolist()):
        assert not bool(got[s, r:].any())


@pytest.mark.parametrize("case", [CASES[1], CASES[4], CASES[6], CASES[10], CASES[13]], ids=str)
def test_same_bits_again_and_out(torch, case):
    ctx, q, _ = _build(torch, case, 11)
    first = ctx.attend(0, q, case[4], case[5])
    out = torch.full((q.shape[0] + 1, *q.shape[1:]), 7.0, dtype=q.dtype, device="cuda")
    assert ctx.attend(0, q, case[4], case[5], out=out[:-1]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:-1], first) and bool((out[-1] == 7.0).all())


def test_lengths_beyond_the_queries_count_as_the_ends(torch):
    ctx, q, _ = _build(torch, CASES[6], 3)
    lens = torch.tensor([-5, 1000], dtype=torch.int32, device="cuda")
    got = ctx.attend(0, q, q_lens=lens)
    # (not the bits of a call with all queries: what the other sequences see decides at which tokens a sequence's
    # history is divided, and with it the order of the sums)
    assert not bool(got[0].any())
    _check(torch, ctx, got, q, q_lens=[0, q.shape[1]])
    assert torch.equal(got, ctx.attend(0, q, q_lens=torch.tensor([0, q.shape[1]], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_orders_and_alignments_of_the_queries(torch, dtype):
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(5)
    ctx = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=6, kv_dtype=dtype)
    _fill(torch, ctx, [900, 700, 20], gen)
    q = torch.randn(2, 9, 6, 128, generator=gen, device="cuda").to(dt)
    want = ctx.attend(0, q, window=200, sinks=3, seq_begin=1)
    _check(torch, ctx, want, q, 200, 3, seq_begin=1)
    heads_first = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    flat = torch.zeros(q.numel() + 3, dtype=dt, device="cuda")
    flat[3:] = q.flatten()
    wide = torch.zeros(2, 9, 6, 130, dtype=dt, device="cuda")
    wide[..., 1:129] = q
    for x in (heads_first, flat[3:].view_as(q), wide[..., 1:129], q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(ctx.attend(0, x, window=200, sinks=3, seq_begin=1), want)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("hot", [512, 200])
def test_what_is_masked_may_hold_anything(torch, dtype, rows, hot):
    """Infinities and NaN in hidden tokens of the window reach nothing; in visible ones, only those that see them."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(9)
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=4, kv_dtype=dtype, hot_window=hot)
    n = 600
    k = torch.randn(1, n, 1, 128, generator=gen, device="cuda").to(dt)
    v = torch.randn(1, n, 1, 128, generator=gen, device="cuda").to(dt)
    bad = 480  # in the uncompressed window
    k[0, bad, 0, 3] = float("inf")
    v[0, bad, 0, 5] = float("nan")
    v[0, bad, 0, 7] = float("-inf")
    ctx.append(0, k, v)
    q = torch.randn(1, rows, 4, 128, generator=gen, device="cuda").to(dt)
    got = ctx.attend(0, q, window=50, sinks=2)
    p = n - rows + torch.arange(rows, device="cuda")
    sees = (p >= bad) & (p < bad + 50)
    assert bool(got[0, ~sees].isfinite().all())
    if bool(sees.any()):
        assert bool(got[0, sees].isnan().any(-1).all())
    ok = k.clone(), v.clone()
    ok[0][0, bad], ok[1][0, bad] = 0.0, 0.0
    ctx.clear(0)
    ctx.append(0, *ok)
    want = ctx.attend(0, q, window=50, sinks=2)
    _check(torch, ctx, want, q, 50, 2)
    off = (got.double() - want.double())[0, ~sees].abs()
    assert bool((off <= 2.0**-9 * 6 + torch.finfo(dt).eps * want[0, ~sees].double().abs()).all())


@pytest.mark.parametrize("hot, at, many", [(512, 450, 200), (200, 650, 45)])  # (all rows see the token)
def test_value_that_is_no_number_stays_in_its_channels(torch, hot, at, many):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for rows in (1, many):
        ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=2, kv_dtype="bfloat16", hot_window=hot)
        k, v = (torch.randn(1, 700, 1, 128, generator=gen, device="cuda").bfloat16() for _ in range(2))
        v[0, at, 0, 9] = float("nan")
        ctx.append(0, k, v)
        got = ctx.attend(0, torch.randn(1, rows, 2, 128, generator=gen, device="cuda").bfloat16())
        assert bool(got[..., 9].isnan().all()) and int(got.isnan().sum()) == 2 * rows


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 8, 300])
@pytest.mark.parametrize("hot", [512, 300])
def test_a_token_with_a_small_value_may_dominate(torch, dtype, rows, hot):
    """The softmax all on a token whose value is 2^-9 of the others': the output keeps its digits."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(21)
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=1, kv_dtype=dtype, outlier_frac=0.0, hot_window=hot)
    n = 1100
    k = 0.1 * torch.randn(1, n, 1, 128, generator=gen, device="cuda")
    v = torch.randn(1, n, 1, 128, generator=gen, device="cuda")
    q = 0.1 * torch.randn(1, rows, 1, 128, generator=gen, device="cuda")
    k[0, 700, 0, :64] += 6.0
    v[0, 700] *= 2.0**-9
    q[..., :64] += 6.0
    ctx.append(0, k.to(dt), v.to(dt))
    q = q.to(dt)
    got = ctx.attend(0, q)
    want, _ = _want(torch, ctx, 0, 0, q[0], rows, None, 0)
    rel = (got[0].double() - want).norm() / want.norm()
    assert float(rel) < torch.finfo(dt).eps / 2 + 2.0**-9, float(rel)


def test_one_token_is_what_decode_gives(torch):
    gen = torch.Generator(device="cuda").manual_seed(1)
    ctx = _ctx(n_seqs=2, n_kv_heads=2, n_q_heads=8, kv_dtype="float16", n_layers=2)
    _fill(torch, ctx, [1300, 700], gen, layer=1)
    q = torch.randn(2, 8, 128, generator=gen, device="cuda").half()
    a, b = ctx.decode(1, q), ctx.attend(1, q[:, None])[:, 0]
    assert torch.allclose(a, b.float(), rtol=2e-2, atol=2e-3)


def test_captured_calls_are_replayed_on_longer_sequences_and_side_by_side(torch):
    gen = torch.Generator(device="cuda").manual_seed(4)
    ctx = _ctx(n_seqs=2, n_kv_heads=1, n_q_heads=4, kv_dtype="bfloat16")
    _fill(torch, ctx, [40, 300], gen)
    shapes = [(1, None, 0), (1, 100, 4), (9, None, 0), (200, None, 0), (200, 150, 3)]
    qs = [torch.randn(2, t, 4, 128, generator=gen, device="cuda").bfloat16() for t, _, _ in shapes]
    side, graphs, outs = torch.cuda.Stream(), [], []
    side.wait_stream(torch.cuda.current_stream())
    for q, (_, w, s) in zip(qs, shapes):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(ctx.attend(0, q, window=w, sinks=s))
    for more in (0, 700, 1900):
        _fill(torch, ctx, [more, more], gen)
        for o in outs:
            o.fill_(5.0)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, q, (_, w, s) in zip(outs, qs, shapes):
            _check(torch, ctx, o, q, w, s)


def test_an_eager_call_after_replayed_appends(torch):
    """Replays of a captured append lengthen the sequences on the device without the host's knowledge."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=4, kv_dtype="bfloat16")
    ref = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=4, kv_dtype="bfloat16")
    k, v = (torch.randn(1, 100, 1, 128, generator=gen, device="cuda").bfloat16() for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    ctx.append(0, k[:, :1], v[:, :1])
    with torch.cuda.graph(graph, stream=side):
        ctx.append(0, k, v)
    ref.append(0, k[:, :1], v[:, :1])
    for _ in range(4):
        graph.replay()
        ref.append(0, k, v)
    torch.cuda.synchronize()
    for t in (1, 30, 250):
        q = torch.randn(1, t, 4, 128, generator=gen, device="cuda").bfloat16()
        _check(torch, ref, ctx.attend(0, q), q)
        _check(torch, ref, ctx.attend(0, q, window=120, sinks=2), q, 120, 2)


def test_two_streams_and_a_small_workspace(torch):
    import ctypes as C

    from turboquant_pro_b200 import _lib

    ctx, q, _ = _build(torch, CASES[6], 17)
    want = ctx.attend(0, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(ctx.attend(0, q))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    # a workspace for one sequence at a time: in rounds, whose divisions are their own
    out = torch.empty_like(q)
    a = _lib.TqAttendArgs(q=q.data_ptr(), out=out.data_ptr(), q_seq_stride=q.stride(0), q_tok_stride=q.stride(1),
                          q_head_stride=q.stride(2), seq_count=2, n_tokens=q.shape[1], q_dtype=_lib.TQ_BF16)
    size, stream = C.c_size_t(), torch.cuda.current_stream().cuda_stream
    assert ctx._lib.tq_attend_workspace(ctx._h, C.byref(a), stream, C.byref(size)) == 0
    work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    longest = _lib.TqAttendArgs.from_buffer_copy(a)
    longest.seq_begin = longest.seq_count = 1
    assert ctx._lib.tq_attend_workspace(ctx._h, C.byref(longest), stream, C.byref(size)) == 0
    assert size.value < work.numel()
    a.workspace, a.workspace_bytes = work.data_ptr(), size.value
    assert ctx._lib.tq_attend(ctx._h, C.byref(a), stream) == 0
    _check(torch, ctx, out, q)
    for bad, code in ((dict(workspace_bytes=100), -4), (dict(workspace=work.data_ptr() + 16), -1),
                      (dict(q=None), -1), (dict(out=None), -1), (dict(n_tokens=-1), -1), (dict(window=-1), -1),
                      (dict(sinks=-1), -1), (dict(q_dtype=9), -1), (dict(layer=1), -1), (dict(seq_count=3), -1),
                      (dict(seq_begin=1), -1)):
        b = _lib.TqAttendArgs.from_buffer_copy(a)
        for name, value in bad.items():
            setattr(b, name, value)
        assert ctx._lib.tq_attend(ctx._h, C.byref(b), stream) == code, bad


def test_empty_calls_and_refusals(torch):
    ctx, q, _ = _build(torch, CASES[1], 2)
    assert ctx.attend(0, q[:0]).shape == q[:0].shape
    assert ctx.attend(0, q[:, :0]).shape == q[:, :0].shape
    lens = torch.ones(4, dtype=torch.int32, device="cuda")
    for bad in (dict(layer=1), dict(layer=-1), dict(q=q[0]), dict(q=q[:, :, :4]), dict(q=q.cpu()),
                dict(q=q.double()), dict(q=q.clone().requires_grad_()), dict(window=0), dict(window=-3),
                dict(sinks=-1), dict(q_lens=lens[:2]), dict(q_lens=lens.long()), dict(q_lens=lens.cpu()),
                dict(seq_begin=1), dict(seq_begin=-1), dict(out=q.float()), dict(out=q[:2].clone()),
                dict(out=torch.empty(4, 1, 8, 129, dtype=q.dtype, device="cuda")[..., :128])):
        args = {"layer": 0, "q": q, **bad}
        with pytest.raises(ValueError):
            ctx.attend(args.pop("layer"), args.pop("q"), **args)


def test_a_refused_step_appends_nothing(torch):
    ctx = _ctx(n_seqs=1, n_kv_heads=2, n_q_heads=4, kv_dtype="bfloat16")
    q, k, v = (torch.zeros(1, 3, h, 128, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2))
    f = torch.ones(64, device="cuda")
    for bad in (dict(window=0), dict(sinks=-1), dict(eps=-1.0), dict(layer=1), dict(v=v[:, :2]), dict(seq_begin=1)):
        args = {"layer": 0, "q": q, "k": k, "v": v, "inv_freq": f, **bad}
        with pytest.raises(ValueError):
            ctx.step(**args)
    assert ctx.lengths(0, 0)[0] == 0


@pytest.mark.parametrize("dtype, chunks", [("bfloat16", [700, 1, 1, 40, 1, 300]), ("float32", [30, 1, 600, 5])])
def test_a_layer_from_projections_to_output(torch, dtype, chunks):
    """step: norm and rotation, append, attention; the keys that the cache holds are the rotated ones."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(6)
    make = lambda: _ctx(n_seqs=2, n_kv_heads=2, n_q_heads=6, kv_dtype=dtype)  # noqa: E731
    ctx, ref = make(), make()
    from turboquant_pro_b200 import norm_rope

    f = torch.tensor([10000.0 ** (-i / 64) for i in range(64)], device="cuda")
    qw, kw = (torch.rand(128, generator=gen, device="cuda").add_(0.5).to(dt) for _ in range(2))
    at = 0
    for t in chunks:
        qkv = torch.randn(2, t, 10, 128, generator=gen, device="cuda").to(dt)
        q, k, v = qkv[:, :, :6], qkv[:, :, 6:8], qkv[:, :, 8:]
        got = ctx.step(0, q, k, v, f, q_weight=qw, k_weight=kw, window=500, sinks=4)
        rq, rk = norm_rope(q, k, f, at + torch.arange(t, device="cuda"), q_weight=qw, k_weight=kw)
        ref.append(0, rk, v)
        _check(torch, ref, got, rq, 500, 4)
        at += t
    assert ctx.lengths(0, 1)[0] == at


def test_the_classes_above_it_take_a_window(torch):
    import numpy as np

    from turboquant_pro_b200 import TurboQuantKVCache
    from turboquant_pro_b200.connector import DeviceBlockStore
    from turboquant_pro_b200.manager import TurboQuantKVManager

    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((700, 2, 128)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((4, 128)).astype(np.float32)
    cache = TurboQuantKVCache.robust(128, 2, n_q_heads=4, max_tokens=1024, seed=0)
    manager = TurboQuantKVManager(1, 2, n_q_heads=4, value_bits=4, max_tokens=1024, seed=0)
    store = DeviceBlockStore(1, 2, n_q_heads=4, max_requests=2, max_tokens=1024, dtype="float32")
    for i in range(0, 700, 100):
        cache._ctx.append(0, torch.from_numpy(k[None, i:i + 100]).cuda(), torch.from_numpy(v[None, i:i + 100]).cuda())
    manager.store(0, k, v)
    store.save("a", 0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    qt = torch.from_numpy(q)[None, None].cuda()
    outs = [(cache._ctx, cache.fused_decode(q, window=90, sinks=2)),
            (manager.context, manager.attend(0, q, window=90, sinks=2)),
            (store.ctx, store.attend(0, {"a": torch.from_numpy(q)}, window=90, sinks=2)["a"].cpu().numpy())]
    for ctx, out in outs:
        slot = ctx.n_seqs - 1 if ctx is store.ctx and ctx.lengths(0, 0)[0] == 0 else 0
        _check(torch, ctx, torch.from_numpy(out)[None, None].cuda(), qt, 90, 2, seq_begin=slot)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("t", [1, 2, 63, 127, 128, 129, 255, 256, 257, 520])
def test_edges_of_the_tiles(torch, dtype, t):
    """Lengths and rows next to the tiles' sizes (80 tokens, 128 and 256 rows), blocks of 150 tokens; queries before
    the first token, which see nothing."""
    gen = torch.Generator(device="cuda").manual_seed(100 + t)
    lens = [79, 80, 81, 160, 161, 449, 450, 600, 641, 1]
    ctx = _ctx(n_seqs=len(lens), n_kv_heads=1, n_q_heads=1, kv_dtype=dtype, hot_window=300)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(len(lens), t, 1, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    for window, sinks in ((None, 0), (1, 0), (80, 0), (81, 80), (200, 161)):
        got = ctx.attend(0, q, window=window, sinks=sinks)
        _check(torch, ctx, got, q, window, sinks)
    assert ctx.status() == 0


@pytest.mark.parametrize("kv", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 11, 31, 90])
def test_types_of_queries_and_cache(torch, kv, dtype, rows):
    gen = torch.Generator(device="cuda").manual_seed(31)
    ctx = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=6, kv_dtype=kv, outlier_frac=0.12)
    _fill(torch, ctx, [1100, 0, 530], gen)
    q = torch.randn(3, rows, 6, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    for window, sinks in ((None, 0), (300, 5)):
        _check(torch, ctx, ctx.attend(0, q, window=window, sinks=sinks), q, window, sinks)
    assert ctx.status() == 0


@pytest.mark.parametrize("hot", [512, 128])
def test_many_sequences(torch, hot):
    """More of them than one launch of the form for few rows divides."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    lens = [(i * 37) % 700 for i in range(150)]
    ctx = _ctx(n_seqs=150, n_kv_heads=1, n_q_heads=4, kv_dtype="bfloat16", hot_window=hot, max_tokens_per_seq=1024)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(149, 2, 4, 128, generator=gen, device="cuda").bfloat16()
    _check(torch, ctx, ctx.attend(0, q, seq_begin=1), q, seq_begin=1)
    _check(torch, ctx, ctx.attend(0, q, seq_begin=1, window=90, sinks=3), q, 90, 3, seq_begin=1)


@pytest.mark.parametrize("hot", [512, 200])
def test_long_sequence(torch, hot):
    gen = torch.Generator(device="cuda").manual_seed(6)
    n = 70001
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=2, kv_dtype="bfloat16", hot_window=hot, max_tokens_per_seq=n)
    _fill(torch, ctx, [n], gen)
    for t in (1, 3, 150):
        q = torch.randn(1, t, 2, 128, generator=gen, device="cuda").bfloat16()
        for window, sinks in ((None, 0), (60000, 100)):
            _check(torch, ctx, ctx.attend(0, q, window=window, sinks=sinks), q, window, sinks)
    assert ctx.status() == 0


def test_one_unit_of_many_is_left_to_the_general_form(torch):
    """Keys beyond half precision's range in one KV head of one sequence, many rows; the others stay as they are."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    ctx = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=4, kv_dtype="bfloat16", hot_window=200)
    k, v = (torch.randn(3, 900, 2, 128, generator=gen, device="cuda").bfloat16() for _ in range(2))
    k[1, 850, 1, 3] = 2.0**30
    ctx.append(0, k, v)
    q = torch.randn(3, 300, 4, 128, generator=gen, device="cuda").bfloat16()
    q[..., 3] = -q[..., 3].abs()  # (that key gets no weight, so that the bound means something)
    got = ctx.attend(0, q, window=400, sinks=5)
    ctx.clear(0)
    k[1, 850, 1, 3] = 0.0
    ctx.append(0, k, v)
    # token 850 aside, the same attention: 64 bits without it
    for s in range(3):
        n, h = 900, 1
        kk, vv = (x.double() for x in ctx.dequant(0, s, 0, n))
        p = n - 300 + torch.arange(300, device="cuda")
        j = torch.arange(n, device="cuda")
        sees = (j <= p[:, None]) & ((j > p[:, None] - 400) | (j < 5))
        for hq in range(4):
            see = sees & ((j != 850)[None] if s == 1 and hq // 2 == 1 else True)
            qk = q[s, :, hq].double()
            pr = torch.softmax((qk @ kk[hq // 2].t() / math.sqrt(128)).masked_fill(~see, -math.inf), 1)
            want = pr @ vv[hq // 2]
            a = (qk.abs() @ kk[hq // 2].abs().t() / math.sqrt(128)).masked_fill(~see, 0.0).amax(1)
            top = vv[hq // 2].abs().amax(1)[None].masked_fill(~see, 0.0).amax(1)
            limit = ((2 * a + 4) * 2.0**-11 * top)[:, None] + torch.finfo(q.dtype).eps / 2 * want.abs()
            off = (got[s, :, hq].double() - want).abs()
            assert bool((off <= limit).all()), (s, hq, float((off / limit).max()))
    assert ctx.status() == 0


@pytest.mark.parametrize("window", [None, 90])
def test_hf_layers_attend_chunks_and_windows(torch, window):
    """The adapter's attention function on stored history: one and several tokens, with and without a window."""
    from types import SimpleNamespace

    from turboquant_pro_b200 import hf_cache

    gen = torch.Generator(device="cuda").manual_seed(13)
    cache = hf_cache.TurboQuantCache(n_layers=1, n_q_heads=4, max_tokens=2048, attend=True)
    module = SimpleNamespace(layer_idx=0, is_causal=True, sliding_window=window, num_key_value_groups=2, training=False)
    n = 0
    for t in (600, 1, 70, 5, 300):
        q = torch.randn(2, 4, t, 128, generator=gen, device="cuda").bfloat16()
        k, v = (torch.randn(2, 2, t, 128, generator=gen, device="cuda").bfloat16() for _ in range(2))
        kk, vv = cache.layers[0].update(k, v)
        n += t
        if n == t:  # a prompt, on its own keys and values
            got = hf_cache.turboquant_attention_forward(module, q, kk, vv, None, scaling=128**-0.5)[0]
            j = torch.arange(t, device="cuda")
            sees = (j <= j[:, None]) & (j > j[:, None] - (window or t))
            qk = (q.double().view(2, 2, 2, t, 128) @ k.double()[:, :, None].transpose(3, 4)) / math.sqrt(128)
            pr = torch.softmax(qk.masked_fill(~sees, -math.inf), 4)
            want = (pr @ v.double()[:, :, None]).view(2, 4, t, 128).transpose(1, 2)
            # (bfloat16 probabilities and values in that product at worst: a step of each, and the output's)
            top = v.double().abs().amax()
            assert bool(((got.double() - want).abs() <= 2.0**-8 * 2 * top + 2.0**-8 * want.abs()).all())
            continue
        p, j = torch.arange(n - t, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        sees = (j <= p) & (j > p - window) if window else j <= p
        outs = [hf_cache.turboquant_attention_forward(module, q, kk, vv, m, scaling=128**-0.5)[0]
                for m in (None, torch.ones(2, n, dtype=torch.int64, device="cuda"), sees[None, None].expand(2, 1, t, n))]
        if t > 1 or window:  # (a single token without a window is decoded, as without the option)
            _check(torch, cache.context, outs[0], q.transpose(1, 2), window)
            assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    # a mask of another kind is attended densely
    other = sees.clone()
    other[:, 3] = False
    got = hf_cache.turboquant_attention_forward(module, q, kk, vv, other[None, None], scaling=128**-0.5)[0]
    kd, vd = cache.layers[0].full()
    want = torch.nn.functional.scaled_dot_product_attention(q, kd, vd, other[None, None], enable_gqa=True)
    assert torch.allclose(got, want.transpose(1, 2), rtol=2e-2, atol=2e-2)
