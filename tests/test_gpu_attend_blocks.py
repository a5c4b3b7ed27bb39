"""KVContext.attend on listed blocks against attention in 64 bits over the dequantised keys and values, with the data and the
limits of attend_oracle: tight enough to see one token too many or too few."""

from __future__ import annotations

import math

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
            borders = {0, n - 1, cold - 1, cold} | {b * s + d for b in range(cold // s + 1) for d in (0, s - 1)}
            k = torch.randn(1, n, h, 128, generator=gen, device="cuda")
            v = oracle.values(n, h, gen, "cuda", borders if s > 16 else ())
            ctx.append(layer, k.to(ctx.kv_dtype), v[None].to(ctx.kv_dtype), seq_begin=seq)


def _want(torch, ctx, layer, seq, q, blocks, q_n):
    """``[T, Hq, 128]``; ``blocks``: lists ``[T][H]``."""
    n, cold, _ = ctx.lengths(layer, seq)
    t, hq, d = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device="cuda")
    if n == 0:
        return out
    s, g, nb = ctx.block_tokens, hq // ctx.n_kv_heads, cold // ctx.block_tokens
    k, v = (x.double() for x in ctx.dequant(layer, seq, 0, n))
    j = torch.arange(n, device="cuda")
    for i in range(min(q_n, t)):
        p = n - q_n + i
        for h in range(ctx.n_kv_heads):
            sees = j >= cold
            before = -1
            for b in blocks[i][h]:
                if not before < b < nb:
                    break
                sees[b * s:(b + 1) * s] = True
                before = b
            sees &= j <= p
            if bool(sees.any()):
                x = q[i, h * g:(h + 1) * g].double() @ k[h, sees].t() / math.sqrt(d)
                out[i, h * g:(h + 1) * g] = torch.softmax(x, 1) @ v[h, sees]
    return out


def _check(torch, ctx, got, q, blocks, q_lens=None, seq_begin=0, layer=0):
    assert got.shape == q.shape and got.dtype == q.dtype
    lists = blocks.tolist()
    for s in range(q.shape[0]):
        q_n = q.shape[1] if q_lens is None else int(q_lens[s])
        want = _want(torch, ctx, layer, seq_begin + s, q[s], lists[s], q_n)
        empty = ~want.any(-1)
        assert not bool(got[s][empty].any())
        if q_n:
            oracle.check(got[s][:q_n], want[:q_n])


CASES = [
    # lens, T, Hkv, Hq, n, kv dtype, q dtype, hot, keys, value bits
    ([4000], 1, 2, 8, 6, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([3000, 512, 0, 513, 4096], 1, 2, 2, 4, "float16", "float16", 512, "nf4_asym", 4),
    ([3000, 700, 5], 5, 1, 7, 3, "bfloat16", "bfloat16", 512, "uniform", 3),
    ([2500, 1000], 3, 2, 24, 5, "float16", "bfloat16", 512, "nf4", 4),
    ([2500, 40], 2, 1, 16, 40, "float32", "float32", 512, "nf4_asym", 3),
    ([2100], 700, 1, 4, 2, "bfloat16", "float16", 512, "nf4_asym", 3),
    ([1000, 999], 2, 2, 8, 9, "bfloat16", "bfloat16", 33, "nf4_asym", 3),
    ([1000], 130, 1, 5, 2, "float16", "float16", 100, "uniform", 4),
    ([700], 1, 1, 4, 300, "float32", "float32", 2, "nf4_asym", 4),
    ([900, 100], 4, 1, 6, 4, "bfloat16", "bfloat16", 128, "polar", 4),
    ([1800], 1, 2, 4, 3, "float32", "float32", 512, "polar", 3),
    ([1300] * 70, 1, 1, 2, 2, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    # many tokens on the same window: a kernel of its own
    ([1700, 300, 600, 5, 0, 2000] * 3, 24, 3, 15, 3, "bfloat16", "bfloat16", 512, "nf4_asym", 3),
    ([1000, 700], 60, 8, 80, 2, "float16", "float16", 512, "uniform", 4),
    ([900], 900, 2, 16, 1, "bfloat16", "bfloat16", 512, "nf4", 3),
]


def _build(torch, case, seed):
    lens, t, h, hq, n, kv, qd, hot, keys, vb = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx = _ctx(n_seqs=len(lens), n_kv_heads=h, n_q_heads=hq, kv_dtype=kv, hot_window=hot, key_mode=keys,
               value_bits=vb, key_bits=vb if keys == "polar" else 4, outlier_frac=0.0 if keys == "polar" else 0.02)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(len(lens), t, hq, 128, generator=gen, device="cuda").to(getattr(torch, qd))
    return ctx, q, gen


def _lists(torch, ctx, lens, t, n, gen, layer=0):
    """Random lists: ascending, of any number of blocks, what is no entry behind them."""
    h = ctx.n_kv_heads
    out = torch.full((len(lens), t, h, n), -1, dtype=torch.int32, device="cuda")
    for s, length in enumerate(lens):
        nb = ctx.cold_blocks(length)
        if nb:
            m = min(n, nb)
            of = torch.rand(t, h, nb, generator=gen, device="cuda").argsort(-1)[..., :m].sort(-1).values.int()
            some = torch.randint(0, m + 1, (t, h, 1), generator=gen, device="cuda")
            out[s, :, :, :m] = torch.where(torch.arange(m, device="cuda") < some, of, -1)
    return out


@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_attention_in_64_bits(torch, case):
    lens, t, n = case[0], case[1], case[4]
    ctx, q, gen = _build(torch, case, 7)
    lists = [_lists(torch, ctx, lens, t, n, gen)]
    if case[8] != "polar":
        lists.append(ctx.select_blocks(0, q, n))
    part = torch.tensor([(i * 7 + 3) % (t + 1) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    for blocks in lists:
        got = ctx.attend(0, q, blocks=blocks)
        _check(torch, ctx, got, q, blocks)
        assert torch.equal(got, ctx.attend(0, q, blocks=blocks))
    got = ctx.attend(0, q, blocks=lists[0], q_lens=part)
    _check(torch, ctx, got, q, lists[0], part)
    for s, r in enumerate(part.tolist()):
        assert not bool(got[s, r:].any())
    assert ctx.status() == 0


@pytest.mark.parametrize("case", [CASES[0], CASES[2], CASES[6], CASES[9]], ids=str)
def test_where_a_list_ends(torch, case):
    ctx, q, _ = _build(torch, case, 5)
    lens, t, h = case[0], case[1], case[2]
    nb = ctx.cold_blocks(lens[0])
    for row in ([2, 1, 0], [1, 1, 2], [0, nb, 1], [-1, 0, 1], [0, 2**31 - 1, 1], [-2**31, 0, 1], [nb - 1, nb, 0], [0, 1, -5]):
        blocks = torch.tensor(row, dtype=torch.int32, device="cuda").expand(len(lens), t, h, 3)
        _check(torch, ctx, ctx.attend(0, q, blocks=blocks), q, blocks)


def test_no_list_at_all_and_every_block(torch):
    for case in (CASES[0], CASES[6]):
        ctx, q, _ = _build(torch, case, 9)
        lens, t, h = case[0], case[1], case[2]
        none = torch.empty(len(lens), t, h, 0, dtype=torch.int32, device="cuda")
        _check(torch, ctx, ctx.attend(0, q, blocks=none), q, none)
        nb = max(ctx.cold_blocks(n) for n in lens)
        every = torch.arange(nb, dtype=torch.int32, device="cuda").expand(len(lens), t, h, nb)
        got = ctx.attend(0, q, blocks=every)
        _check(torch, ctx, got, q, every)
        k, v = ctx.dequant(0, 0, 0, lens[0])
        oracle.check(got[0], oracle.attention(k, v, q[0], t, None, 0))


def test_rows_that_see_nothing(torch):
    # a chunk that is longer than the window: its first tokens see blocks alone, and only up to their own position
    ctx, q, _ = _build(torch, CASES[5], 4)
    blocks = torch.full((1, 700, 1, 2), -1, dtype=torch.int32, device="cuda")
    blocks[:, :, :, 0] = 7  # (1792 .. 2047: not yet there for the rows before)
    got = ctx.attend(0, q, blocks=blocks)
    _check(torch, ctx, got, q, blocks)
    first = 2100 - 700
    cold = ctx.lengths(0, 0)[1]
    assert not bool(got[0, :min(7 * 256, cold) - first].any())


def test_orders_parts_of_the_batch_out_and_rounds(torch):
    case = ([2000, 3000, 900, 1500], 3, 2, 6, 3, "bfloat16", "bfloat16", 512, "nf4_asym", 3)
    for hot in (512, 100):
        case = case[:7] + (hot,) + case[8:]
        ctx, q, gen = _build(torch, case, 3)
        lists = _lists(torch, ctx, case[0], 3, 3, gen)[1:]
        q = q[1:]
        want = ctx.attend(0, q, blocks=lists, seq_begin=1)
        _check(torch, ctx, want, q, lists, seq_begin=1)
        wide = torch.zeros(3, 3, 2, 7, dtype=torch.int32, device="cuda")
        wide[..., 2:5] = lists
        for x, b in ((q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), lists), (q, wide[..., 2:5]),
                     (q, lists.transpose(1, 2).contiguous().transpose(1, 2))):
            assert torch.equal(ctx.attend(0, x, blocks=b, seq_begin=1), want)
        out = torch.full((4, 3, 6, 128), 7.0, dtype=q.dtype, device="cuda")
        ctx.attend(0, q, blocks=lists, seq_begin=1, out=out[:3])
        assert torch.equal(out[:3], want) and bool((out[3] == 7.0).all())
        # in rounds of one sequence
        import ctypes as C

        from turboquant_pro_b200._lib import TqAttendArgs

        one, size = TqAttendArgs(), C.c_size_t()
        one.seq_begin, one.seq_count, one.n_tokens, one.q_dtype = 2, 1, 3, 2
        most = 0
        for s in (1, 2, 3):
            one.seq_begin = s
            assert ctx._lib.tq_attend_blocks_workspace(ctx._h, C.byref(one), 3, None, C.byref(size)) == 0
            most = max(most, size.value)
        _check(torch, ctx, ctx.attend(0, q, blocks=lists, seq_begin=1, max_workspace=most), q, lists, seq_begin=1)


def test_captured_calls_follow_the_lengths(torch):
    case = ([600], 1, 2, 8, 3, "bfloat16", "bfloat16", 512, "nf4_asym", 3)
    ctx, q, gen = _build(torch, case, 8)
    ctx.attend(0, q, blocks=ctx.select_blocks(0, q, 3))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        blocks = ctx.select_blocks(0, q, 3)
        got = ctx.attend(0, q, blocks=blocks)
    for _ in range(3):
        graph.replay()
        _check(torch, ctx, got, q, blocks)
        k = torch.randn(1, 900, 2, 128, generator=gen, device="cuda").bfloat16()
        ctx.append(0, k, oracle.values(900, 2, gen, "cuda")[None].bfloat16())
    graph.replay()
    _check(torch, ctx, got, q, blocks)


def test_two_calls_at_once(torch):
    ctx, q, gen = _build(torch, CASES[1], 6)
    lists = [_lists(torch, ctx, CASES[1][0], 1, 4, gen) for _ in range(2)]
    want = [ctx.attend(0, q, blocks=b) for b in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for b, stream in zip(lists, streams):
            with torch.cuda.stream(stream):
                got.append(ctx.attend(0, q, blocks=b))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])


def test_refusals(torch):
    ctx = _ctx(n_seqs=2, n_kv_heads=2, n_q_heads=4)
    q = torch.zeros(2, 3, 4, 128, device="cuda")
    blocks = torch.zeros(2, 3, 2, 5, dtype=torch.int32, device="cuda")
    for bad in (dict(blocks=blocks.long()), dict(blocks=blocks[:1]), dict(blocks=blocks[:, :2]), dict(blocks=blocks[:, :, :1]),
                dict(blocks=blocks[0]), dict(blocks=blocks.cpu()), dict(window=5), dict(sinks=1), dict(seq_begin=1)):
        with pytest.raises(ValueError):
            ctx.attend(**{"layer": 0, "q": q, "blocks": blocks, **bad})
    assert ctx.attend(0, q[:, :0], blocks=blocks[:, :0]).shape == (2, 0, 4, 128)
    assert ctx.attend(0, q[:0], blocks=blocks[:0]).shape == (0, 3, 4, 128)


def test_workspace_of_calls_whose_window_has_a_kernel_of_its_own(torch):
    # room for the states of the blocks alone: of one block, shared by many rows, at most three a row
    import ctypes as C

    from turboquant_pro_b200._lib import TqAttendArgs

    b, t, h, hq = 64, 10, 8, 64
    ctx, q, gen = _build(torch, ([700] * b, t, h, hq, 1, "bfloat16", "bfloat16", 512, "nf4_asym", 3), 8)
    lists = _lists(torch, ctx, [700] * b, t, 1, gen)
    want = ctx.attend(0, q, blocks=lists)
    assert ctx.last_launches() == 2
    _check(torch, ctx, want[:3], q[:3], lists[:3])
    a, size = TqAttendArgs(), C.c_size_t()
    a.seq_count, a.n_tokens, a.q_dtype = b, t, 2
    assert ctx._lib.tq_attend_blocks_workspace(ctx._h, C.byref(a), 1, None, C.byref(size)) == 0
    most = b * t * hq * 3 * (2 + 128) * 4 + 4096  # (and how the work is divided)
    assert size.value <= most
    assert torch.equal(ctx.attend(0, q, blocks=lists, max_workspace=most), want)
    assert ctx.last_launches() == 2
    ctx.attend(0, q, blocks=lists, max_workspace=most // 2)
    assert ctx.last_launches() > 2
