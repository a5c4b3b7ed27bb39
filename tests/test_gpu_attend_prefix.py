"""KVContext.attend with a shared beginning against attention in 64 bits over the dequantised keys and values of the prefix and of
each sequence, with the data and the limits of attend_oracle."""

from __future__ import annotations

import pytest

import attend_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


def _ctx(**kw):
    from turboquant_pro_b200 import KVContext

    return KVContext(**{"n_layers": 1, "seed": 3, "max_tokens_per_seq": 4096, **kw})


def _fill(torch, ctx, lens, gen, layer=0):
    h, s = ctx.n_kv_heads, ctx.block_tokens
    for seq, n in enumerate(lens):
        if n:
            cold = ctx.cold_blocks(n) * s
            # tokens at what a tile of a kernel may begin or end with
            borders = {0, n - 1, cold - 1, cold} | {c * b + d for c in (64, 80, 128, 256) for b in range(0, n // c + 1, 5) for d in (-1, 0)}
            k = torch.randn(1, n, h, 128, generator=gen, device="cuda")
            v = oracle.values(n, h, gen, "cuda", borders)
            ctx.append(layer, k.to(ctx.kv_dtype), v[None].to(ctx.kv_dtype), seq_begin=seq)


def _check(torch, ctx, got, q, prefix, q_lens=None, seq_begin=0, layer=0, by_head=1.0):
    assert got.shape == q.shape and got.dtype == q.dtype
    m = ctx.lengths(layer, prefix)[0]
    pk, pv = ctx.dequant(layer, prefix, 0, m)
    t = q.shape[1]
    for s in range(q.shape[0]):
        q_n = t if q_lens is None else min(max(int(q_lens[s]), 0), t)
        n = ctx.lengths(layer, seq_begin + s)[0]
        k, v = ctx.dequant(layer, seq_begin + s, 0, n)
        k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
        # (rows before a sequence's first token see nothing)
        skip = max(q_n - n, 0)
        assert not bool(got[s, :skip].any()) and not bool(got[s, q_n:].any())
        if q_n > skip:
            want = oracle.attention(k, v, q[s, skip:q_n], q_n - skip, None, 0)
            head, row = oracle.measures(got[s, skip:q_n], want)
            most_head, most_row = oracle.limits(got.dtype)
            assert head <= by_head * most_head and row <= most_row, (head / most_head, row / most_row)


CASES = [
    # lens of the sequences, prefix, T, Hkv, Hq, kv dtype, q dtype, hot, keys, value bits
    ([100, 700], 2000, 1, 2, 8, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([5, 1, 600, 1200, 33], 1300, 1, 2, 2, "float16", "float16", 512, "nf4_asym", 4),
    ([900] * 40, 3000, 1, 1, 8, "bfloat16", "bfloat16", 512, "uniform", 3),
    ([20] * 33, 4000, 1, 2, 8, "bfloat16", "bfloat16", 512, "nf4_asym", 4),
    ([3, 800], 513, 5, 1, 7, "bfloat16", "float16", 512, "nf4", 3),
    ([1500, 40], 777, 130, 2, 4, "float16", "bfloat16", 512, "nf4_asym", 3),
    ([700] * 5, 2500, 2, 1, 16, "float32", "float32", 512, "nf4_asym", 4),
    ([90], 500, 1, 1, 4, "bfloat16", "bfloat16", 512, "nf4_asym", 3),     # a prefix without blocks
    ([90, 4], 1, 1, 1, 4, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([300, 20], 1000, 3, 2, 6, "bfloat16", "bfloat16", 33, "nf4_asym", 3),
    ([300] * 20, 900, 4, 1, 4, "float16", "float16", 100, "uniform", 4),
    ([200, 700], 900, 2, 1, 4, "float32", "float32", 128, "polar", 4),
    ([700, 3], 900, 1, 2, 4, "bfloat16", "bfloat16", 512, "polar", 3),
    ([60] * 70, 1800, 1, 1, 2, "bfloat16", "float32", 512, "nf4_asym", 3),
    ([600] * 3, 1111, 300, 1, 2, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    # many tiles a CTA, pages that change within its part
    ([9] * 40, 4096, 1, 16, 128, "bfloat16", "bfloat16", 512, "nf4_asym", 4),
    ([30] * 50, 3900, 1, 32, 192, "bfloat16", "bfloat16", 512, "uniform", 3),
    ([17] * 20, 4000, 1, 16, 128, "float16", "float16", 512, "nf4", 4),
    ([40] * 70, 3333, 2, 8, 64, "float16", "float16", 512, "nf4_asym", 3),
    # drafts on windows and blocks of their own, several tiles of rows
    ([3, 800, 512, 513, 32, 33, 64], 700, 5, 1, 7, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([300, 1, 2000], 300, 4, 2, 32, "float16", "float16", 512, "uniform", 4),
    ([700] * 66, 600, 1, 1, 3, "float16", "float16", 512, "nf4_asym", 3),
]


def _build(torch, case, seed):
    lens, prefix, t, h, hq, kv, qd, hot, keys, vb = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx = _ctx(n_seqs=len(lens) + 1, n_kv_heads=h, n_q_heads=hq, kv_dtype=kv, hot_window=hot, key_mode=keys,
               value_bits=vb, key_bits=vb if keys == "polar" else 4, outlier_frac=0.0 if keys == "polar" else 0.02)
    _fill(torch, ctx, [prefix] + lens, gen)
    q = torch.randn(len(lens), t, hq, 128, generator=gen, device="cuda").to(getattr(torch, qd))
    return ctx, q, gen


@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_attention_in_64_bits(torch, case):
    ctx, q, _ = _build(torch, case, 7)
    b, t = q.shape[:2]
    got = ctx.attend(0, q, prefix=0, seq_begin=1)
    _check(torch, ctx, got, q, 0, seq_begin=1)
    assert torch.equal(got, ctx.attend(0, q, prefix=0, seq_begin=1))
    part = torch.tensor([(i * 7 + 3) % (t + 1) for i in range(b)], dtype=torch.int32, device="cuda")
    got = ctx.attend(0, q, prefix=0, seq_begin=1, q_lens=part)
    _check(torch, ctx, got, q, 0, part, seq_begin=1)
    assert ctx.status() == 0


def test_empty_prefix_and_empty_sequences(torch):
    for hot in (512, 33):
        ctx = _ctx(n_seqs=4, n_kv_heads=2, n_q_heads=4, kv_dtype="bfloat16", hot_window=hot)
        gen = torch.Generator(device="cuda").manual_seed(1)
        _fill(torch, ctx, [0, 600, 0, 9], gen)
        q = torch.randn(3, 2, 4, 128, generator=gen, device="cuda").bfloat16()
        got = ctx.attend(0, q, prefix=0, seq_begin=1)
        oracle.check(got[0], oracle.attention(*ctx.dequant(0, 1, 0, 600), q[0], 2, None, 0))
        assert not bool(got[1].any())
        got = ctx.attend(0, q[:1], prefix=1, seq_begin=0)
        assert not bool(got.any())


def test_padding_that_is_no_number(torch):
    for case in (CASES[0], CASES[5], CASES[9]):
        ctx, q, _ = _build(torch, case, 2)
        t = q.shape[1]
        part = torch.tensor([t, max(t // 2, 0)], dtype=torch.int32, device="cuda")
        q[1, int(part[1]):] = float("nan")
        got = ctx.attend(0, q, prefix=0, seq_begin=1, q_lens=part)
        _check(torch, ctx, got, torch.nan_to_num(q), 0, part, seq_begin=1)


def test_large_and_small_values_in_the_prefix(torch):
    # beyond what half precision holds, and infinities in the prefix's window: some heads go by the general form
    for t in (1, 150):
        gen = torch.Generator(device="cuda").manual_seed(3)
        ctx = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=4, kv_dtype="float32", value_bits=3)
        k, v = (torch.randn(1, 1500, 2, 128, generator=gen, device="cuda") for _ in range(2))
        k[:, :, 1] *= 1e-3
        v[:, 700:, 1] *= 1e9
        ctx.append(0, k, v)
        for s in (1, 2):
            x = torch.randn(1, 200, 2, 128, generator=gen, device="cuda")
            ctx.append(0, x, x, seq_begin=s)
        q = torch.randn(2, t, 4, 128, generator=gen, device="cuda").bfloat16()
        _check(torch, ctx, ctx.attend(0, q, prefix=0, seq_begin=1), q, 0, seq_begin=1)
        w = torch.randn(1, 1, 2, 128, generator=gen, device="cuda")
        ctx.append(0, w, torch.full_like(w, float("inf")))
        got = ctx.attend(0, q, prefix=0, seq_begin=1)
        assert bool(torch.isposinf(got).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("hot, keys, prefix, b, t", [(512, "nf4_asym", 2000, 20, 1), (100, "uniform", 1500, 9, 30),
                                                     (512, "uniform", 2500, 3, 200), (512, "nf4_asym", 300, 2, 120)])
def test_keys_with_a_large_constant_part(torch, dtype, hot, keys, prefix, b, t):
    # other constants in the prefix than in each of the sequences: what a form takes off all scores of a part shows
    gen = torch.Generator(device="cuda").manual_seed(9)
    ctx = _ctx(n_seqs=b + 1, n_kv_heads=2, n_q_heads=4, kv_dtype="float32" if dtype == "float32" else dtype, hot_window=hot,
               key_mode=keys)
    q = torch.randn(b, t, 4, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    for s, n in enumerate([prefix] + [t + 130 * i for i in range(b)]):
        constant = 0.5 * torch.randn(2, 128, generator=gen, device="cuda")
        k = torch.randn(1, n, 2, 128, generator=gen, device="cuda") + constant
        v = torch.randn(1, n, 2, 128, generator=gen, device="cuda")
        ctx.append(0, k.to(ctx.kv_dtype), v.to(ctx.kv_dtype), seq_begin=s)
    _check(torch, ctx, ctx.attend(0, q, prefix=0, seq_begin=1), q, 0, seq_begin=1)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_values_that_are_no_numbers_in_the_sequences_windows(torch, dtype):
    gen = torch.Generator(device="cuda").manual_seed(13)
    ctx = _ctx(n_seqs=4, n_kv_heads=2, n_q_heads=6, kv_dtype=dtype)
    _fill(torch, ctx, [900, 200, 300, 40], gen)
    k, v = (torch.randn(3, 3, 2, 128, generator=gen, device="cuda") for _ in range(2))
    v[0, 1, 0, 5], v[0, 1, 0, 6], v[1, 2, 1] = float("inf"), float("nan"), float("-inf")
    k[2, 1, 0, 7] = float("inf")
    ctx.append(0, k.to(ctx.kv_dtype), v.to(ctx.kv_dtype), seq_begin=1)
    q = torch.randn(3, 3, 6, 128, generator=gen, device="cuda").to(ctx.kv_dtype)
    q[..., 7] = -q[..., 7].abs() - 0.1  # (an infinite key then has a score of -inf, a weight of zero)
    got = ctx.attend(0, q, prefix=0, seq_begin=1)
    pk, pv = ctx.dequant(0, 0, 0, 900)
    for s, n in enumerate((203, 303, 43)):
        sk, sv = ctx.dequant(0, s + 1, 0, n)
        kk, vv = torch.cat((pk, sk), 1), torch.cat((pv, sv), 1)
        want = oracle.attention(torch.nan_to_num(kk, posinf=0.0), torch.nan_to_num(vv, 0.0, 0.0, 0.0), q[s], 3, None, 0)
        spoilt = torch.zeros_like(want, dtype=torch.bool)
        if s == 0:  # from the second token on, of the first KV head
            spoilt[1:, :3, 5:7] = True
            assert bool(torch.isposinf(got[s, 1:, :3, 5]).all()) and bool(torch.isnan(got[s, 1:, :3, 6]).all())
        if s == 1:
            spoilt[2:, 3:] = True
            assert bool(torch.isneginf(got[s, 2, 3:]).all())
        if s == 2:  # (the infinite key's token counts for nothing)
            hidden = [slice(900 + 41, 900 + 42)]
            first = oracle.attention(torch.nan_to_num(kk, posinf=0.0), vv, q[s], 3, None, 0, hidden)
            want[:, :3] = first[:, :3]
        x = torch.where(spoilt, want, got[s].double())
        assert bool(torch.isfinite(x).all())
        keep = ~spoilt.any(-1)
        head, row = oracle.measures(got[s][keep][None], want[keep][None])
        assert row <= oracle.limits(got.dtype)[1], row
        rest = (x - want).norm(dim=-1) / want.norm(dim=-1)
        assert float(rest.max()) <= oracle.limits(got.dtype)[1]


def test_orders_parts_of_the_batch_and_out(torch):
    for case in (CASES[0], CASES[4], CASES[5], CASES[9]):
        ctx, q, _ = _build(torch, case, 4)
        want = ctx.attend(0, q, prefix=0, seq_begin=1)
        b, t, hq, _ = q.shape
        heads_first = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        tokens_first = q.transpose(0, 1).contiguous().transpose(0, 1)
        flat = torch.zeros(q.numel() + 3, dtype=q.dtype, device="cuda")
        flat[3:] = q.flatten()
        fused = torch.zeros(b, t, hq + 3, 128, dtype=q.dtype, device="cuda")
        fused[:, :, 1:hq + 1] = q
        for x in (heads_first, tokens_first, flat[3:].view(q.shape), fused[:, :, 1:hq + 1]):
            assert torch.equal(ctx.attend(0, x, prefix=0, seq_begin=1), want)
        out = torch.full((b + 1, t, hq, 128), 7.0, dtype=q.dtype, device="cuda")
        ctx.attend(0, q, prefix=0, seq_begin=1, out=out[:b])
        assert torch.equal(out[:b], want) and bool((out[b] == 7.0).all())
        _check(torch, ctx, ctx.attend(0, q[1:], prefix=1, seq_begin=2), q[1:], 1, seq_begin=2)
        _check(torch, ctx, ctx.attend(0, q[:1], prefix=2, seq_begin=0), q[:1], 2, seq_begin=0)


# A head of few rows (two a sequence), float16.  The limit by head counts a probability's rounding as 0.42 of eps / 2, its mean square over
# many.  A row's error is e = sum_j d_j p_j v_j with |d_j| <= eps / 2 (half a step, next to a power of two), and its output o = sum_j
# p_j v_j: with v_j independent, of 128 channels and so nearly orthogonal, |e|^2 = sum d_j^2 p_j^2 |v_j|^2 <= (eps / 2)^2 |o|^2,
# which a row comes to whose output is mostly that of one token (50 times as large as the others).  With the output's own rounding,
# 0.42 as ever: sqrt(1 + 0.42^2) = 1.085.
FEW_ROWS = 1.085


@pytest.mark.parametrize("case", [CASES[2], CASES[5], CASES[11], CASES[18]], ids=str)
def test_rounds(torch, case):
    import ctypes as C

    from turboquant_pro_b200._lib import TqAttendArgs

    ctx, q, _ = _build(torch, case, 9)
    b, t = q.shape[:2]
    a, size = TqAttendArgs(), C.c_size_t()
    a.n_tokens, a.q_dtype, a.seq_begin, a.seq_count = t, {"float32": 0, "float16": 1, "bfloat16": 2}[case[6]], 1, b
    a.q_seq_stride, a.q_tok_stride, a.q_head_stride = q.stride()[:3]
    assert ctx._lib.tq_attend_prefix_workspace(ctx._h, C.byref(a), 0, None, C.byref(size)) == 0
    whole, one = size.value, 0
    a.seq_count = 1
    for s in range(b):
        a.seq_begin = 1 + s
        assert ctx._lib.tq_attend_prefix_workspace(ctx._h, C.byref(a), 0, None, C.byref(size)) == 0
        one = max(one, size.value)
    want = ctx.attend(0, q, prefix=0, seq_begin=1)
    assert torch.equal(ctx.attend(0, q, prefix=0, seq_begin=1, max_workspace=whole), want)
    for most in (one, (one + whole) // 2, whole - 1):
        if one <= most < whole:
            got = ctx.attend(0, q, prefix=0, seq_begin=1, max_workspace=most)
            _check(torch, ctx, got, q, 0, seq_begin=1, by_head=FEW_ROWS if case[6] == "float16" else 1.0)
            # the same as calls of so many sequences
            n, same = b, False
            while not same and n > 1:
                n = (n + 1) // 2
                parts = [ctx.attend(0, q[i:i + n], prefix=0, seq_begin=1 + i) for i in range(0, b, n)]
                same = torch.equal(torch.cat(parts), got)
            assert same
    assert ctx.status() == 0


def test_captured_calls_follow_the_lengths(torch):
    for case in (([100, 700, 9], 600, 1, 2, 8, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
                 ([300] * 12, 600, 5, 1, 8, "bfloat16", "bfloat16", 512, "nf4_asym", 3)):
        ctx, q, gen = _build(torch, case, 8)
        ctx.attend(0, q, prefix=0, seq_begin=1)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            got = ctx.attend(0, q, prefix=0, seq_begin=1)
        for n in (900, 1):
            graph.replay()
            _check(torch, ctx, got, q, 0, seq_begin=1)
            for s in (0, 2):
                k = torch.randn(1, n, ctx.n_kv_heads, 128, generator=gen, device="cuda").bfloat16()
                ctx.append(0, k, oracle.values(n, ctx.n_kv_heads, gen, "cuda")[None].bfloat16(), seq_begin=s)
        graph.replay()
        _check(torch, ctx, got, q, 0, seq_begin=1)


def test_two_calls_at_once(torch):
    ctx, q, gen = _build(torch, CASES[3], 6)
    qs = [q, torch.randn_like(q)]
    want = [ctx.attend(0, x, prefix=0, seq_begin=1) for x in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for x, stream in zip(qs, streams):
            with torch.cuda.stream(stream):
                got.append(ctx.attend(0, x, prefix=0, seq_begin=1))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])


def test_refusals(torch):
    from turboquant_pro_b200._lib import TqError

    ctx = _ctx(n_seqs=4, n_kv_heads=2, n_q_heads=4)
    q = torch.zeros(2, 3, 4, 128, device="cuda")
    for bad in (dict(prefix=1), dict(prefix=2), dict(prefix=-1), dict(prefix=4), dict(window=5), dict(sinks=1),
                dict(blocks=torch.zeros(2, 3, 2, 1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.attend(**{"layer": 0, "q": q, "prefix": 0, "seq_begin": 1, **bad})
    with pytest.raises(TypeError):
        ctx.attend(0, q, prefix=0.5, seq_begin=1)
    with pytest.raises(TqError, match="workspace"):
        ctx.attend(0, q, prefix=0, seq_begin=1, max_workspace=1000)
    assert ctx.attend(0, q[:, :0], prefix=0, seq_begin=1).shape == (2, 0, 4, 128)
    assert ctx.attend(0, q[:0], prefix=0, seq_begin=1).shape == (0, 3, 4, 128)


# ---- a layer's step with all of it ----------------------------------------------------------------------------
def _freq(torch):
    import numpy as np

    return torch.tensor(1e6 ** (-np.arange(64) / 64), dtype=torch.float32, device="cuda")


def test_a_step_on_a_shared_beginning(torch):
    from turboquant_pro_b200 import norm_rope

    gen = torch.Generator(device="cuda").manual_seed(11)
    ctx = _ctx(n_layers=2, n_seqs=4, n_kv_heads=2, n_q_heads=8, kv_dtype="bfloat16")
    same = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=8, kv_dtype="bfloat16")
    f = _freq(torch)

    def tokens(b, t):
        q, k, v = (torch.randn(b, t, h, 128, generator=gen, device="cuda").bfloat16() for h in (8, 2, 2))
        return q, k, v

    w = torch.rand(128, generator=gen, device="cuda").add_(0.5).bfloat16()
    q, k, v = tokens(1, 1200)
    ctx.step(1, q, k, v, f, q_weight=w, k_weight=w)
    start = 1200
    for t in (7, 1, 3):
        q, k, v = tokens(3, t)
        got = ctx.step(1, q, k, v, f, q_weight=w, k_weight=w, seq_begin=1, prefix=0)
        at = start + torch.arange(t, device="cuda")
        nq, nk = norm_rope(q, k, f, at, q_weight=w, k_weight=w)
        same.append(0, nk, v)
        start += t
        pk, pv = ctx.dequant(1, 0, 0, 1200)
        n = start - 1200
        for s in range(3):
            sk, sv = same.dequant(0, s, 0, n)
            want = oracle.attention(torch.cat((pk, sk), 1), torch.cat((pv, sv), 1), nq[s], t, None, 0)
            oracle.check(got[s], want)


def test_a_step_on_selected_blocks_with_positions_of_several_axes(torch):
    from turboquant_pro_b200 import norm_rope

    gen = torch.Generator(device="cuda").manual_seed(12)
    a, b = (_ctx(n_seqs=2, n_kv_heads=2, n_q_heads=6, kv_dtype="float16") for _ in range(2))
    f, axes = _freq(torch), torch.tensor([i % 3 for i in range(64)], dtype=torch.uint8, device="cuda")
    start = 0
    for t in (1500, 1, 1, 4):
        q, k, v = (torch.randn(2, t, h, 128, generator=gen, device="cuda").half() for h in (6, 2, 2))
        pos = start + torch.randint(0, 50, (3, 2, t), generator=gen, device="cuda")
        got = a.step(0, q, k, v, f, positions=pos, axes=axes, top_blocks=3, first_blocks=1)
        nq, nk = norm_rope(q, k, f, pos, axes=axes)
        b.append(0, nk, v)
        blocks = b.select_blocks(0, nq, 3, first=1)
        assert torch.equal(got, b.attend(0, nq, blocks=blocks))
        start += t


def test_what_a_step_refuses_is_not_appended(torch):
    ctx = _ctx(n_seqs=3, n_kv_heads=2, n_q_heads=4, kv_dtype="float16")
    q, k = (torch.zeros(2, 1, h, 128, device="cuda").half() for h in (4, 2))
    f = _freq(torch)
    for bad in (dict(prefix=1), dict(prefix=3), dict(prefix=0, top_blocks=2), dict(prefix=0, window=4),
                dict(top_blocks=2, sinks=3), dict(top_blocks=0), dict(top_blocks=2, first_blocks=-1),
                dict(axes=torch.zeros(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.step(0, q, k, k, f, seq_begin=1, **bad)
    assert [ctx.lengths(0, s)[0] for s in range(3)] == [0, 0, 0]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tile", [0, 1, 5])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(torch, dtype, tile):
    """The test hook withholds the keys of a tile of the prefix and shortens the probe limit: the call returns, the status word
    has bit 1, and nothing of it is left."""
    from turboquant_pro_b200._lib import TqError

    gen = torch.Generator(device="cuda").manual_seed(61)
    # (enough heads that a CTA has a dozen tiles)
    ctx = _ctx(n_seqs=21, n_kv_heads=37, n_q_heads=37 * 8, kv_dtype=dtype, hot_window=300, max_tokens_per_seq=4000)
    _fill(torch, ctx, [40] * 20 + [3900], gen)
    q = torch.randn(20, 1, 37 * 8, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    good = ctx.attend(0, q, prefix=20)
    assert ctx.status() == 0
    ctx.debug_wait(wait_limit=64, withhold_tile=tile)
    ctx.attend(0, q, prefix=20)
    with pytest.raises(TqError, match="wait"):
        ctx.raise_on_timeout()
    assert ctx.status() == 0
    ctx.debug_wait()
    assert torch.equal(ctx.attend(0, q, prefix=20), good)
    assert ctx.status() == 0


def test_a_prefix_among_the_callers_own_sequences_is_refused_below_python_too(torch):
    import ctypes as C

    from turboquant_pro_b200._lib import TqRope

    ctx = _ctx(n_seqs=5, n_kv_heads=2, n_q_heads=4, kv_dtype="float16")
    q, k = (torch.randn(2, 3, h, 128, device="cuda").half() for h in (4, 2))
    out = [torch.empty_like(x) for x in (q, k)]
    f = _freq(torch)
    r = TqRope(q.data_ptr(), k.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), None, None, f.data_ptr(), None,
               *q.stride()[:3], *k.stride()[:3], 0, 0, 2, 3, 4, 2, 1, 0, 64, 128, 1e-6)
    stream = torch.cuda.current_stream().cuda_stream
    for prefix, ok in ((-1, True), (0, True), (1, False), (2, False), (3, True), (4, True), (5, False), (-2, False)):
        assert (ctx._lib.tq_ctx_norm_rope_after(ctx._h, 0, 1, prefix, C.byref(r), stream) == 0) == ok, prefix
    assert b"prefix" in ctx._lib.tq_last_error()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_a_token_of_no_value_that_has_most_of_the_weight(torch, dtype):
    """The first token of each window has a score 12 above the others' and a value of zero: the output is what tokens with
    probabilities of some 1e-6 have, whose digits have to be there."""
    b, n = 12, 300
    ctx = _ctx(n_seqs=b + 1, n_kv_heads=2, n_q_heads=8, kv_dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(17)
    k, v = (torch.randn(b + 1, n, 2, 128, generator=gen, device="cuda") for _ in range(2))
    q = torch.randn(b, 1, 8, 128, generator=gen, device="cuda")
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[1:, 0, :, 0], v[1:, 0] = 12.0 * 128**0.5 / 8.0, 0.0
    v *= 2000.0  # (outputs are then some tenths, and keep their digits in float16)
    k, v, q = (x.to(getattr(torch, dtype)) for x in (k, v, q))
    ctx.append(0, k, v)
    got = ctx.attend(0, q, prefix=0, seq_begin=1)
    assert ctx.last_launches() == 3
    assert float(got.abs().mean()) > 0.05
    _check(torch, ctx, got, q, 0, seq_begin=1)
