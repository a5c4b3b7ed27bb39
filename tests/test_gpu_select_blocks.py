"""KVContext.select_blocks against scores in 64 bits of the exported containers, ranked by Python's sort.  What is
selected has to be equal: no tolerance.  (Two blocks whose scores differ by less than their sums' rounding in 64 bits, 2^-44 of them,
would be the same block to this test; blocks that are copies of one another have equal scores on both sides.)"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


def _ctx(**kw):
    from turboquant_pro_b200 import KVContext

    return KVContext(**{"n_layers": 1, "seed": 3, "max_tokens_per_seq": 8192, **kw})


def _fill(torch, ctx, lens, gen, layer=0):
    h, s = ctx.n_kv_heads, ctx.block_tokens
    scale = torch.exp(0.5 * torch.randn(h, 128, generator=gen, device="cuda"))
    for seq, n in enumerate(lens):
        if n:
            common = 0.5 * torch.randn((n + s - 1) // s, h, 128, generator=gen, device="cuda")
            k = (torch.randn(n, h, 128, generator=gen, device="cuda") + common.repeat_interleave(s, 0)[:n]) * scale + 0.3
            v = torch.randn(1, n, h, 128, generator=gen, device="cuda")
            ctx.append(layer, k[None].to(ctx.kv_dtype), v.to(ctx.kv_dtype), seq_begin=seq)


def _want(torch, ctx, layer, seq, q, n, first, q_n):
    """``[T, H, n]`` for the queries ``[T, Hq, D]`` of one sequence."""
    import numpy as np

    total, cold, _ = ctx.lengths(layer, seq)
    s, h, g = ctx.block_tokens, ctx.n_kv_heads, ctx.n_q_heads // ctx.n_kv_heads
    nb = cold // s
    blocks = [ctx.export_block(layer, seq, b) for b in range(nb)]
    low, high = (0.0, 15.0) if ctx.key_mode == "uniform" else (-1.0, 1.0)
    out = np.full((q.shape[0], h, n), -1, np.int32)
    x = q.double().cpu().numpy()
    for i in range(min(q_n, q.shape[0])):
        p = total - q_n + i
        m = min(nb, p // s + 1) if p >= 0 else 0
        for head in range(h):
            keyed = []
            for b in range(m):
                mu, sc = (blocks[b][name].reshape(h, 128)[head].astype(np.float64) for name in ("nf4_mean", "nf4_scale"))
                score = sum(np.maximum(x[i, head * g + j] * (mu + low * sc), x[i, head * g + j] * (mu + high * sc)).sum()
                            for j in range(g))
                keyed.append((0 if b < first or b == p // s else 1, -score if score == score else np.inf, b))
            # (copies of a block: equal up to the sums' rounding)
            keyed = [(a, float(f"{sc:.11e}"), b) for a, sc, b in keyed]
            best = sorted(b for _, _, b in sorted(keyed)[:n])
            out[i, head, :len(best)] = best
    return torch.from_numpy(out)


CASES = [
    # lens, T, Hkv, Hq, n, first, q dtype, hot, keys
    ([8000], 1, 2, 8, 5, 1, "bfloat16", 512, "nf4_asym"),
    ([3000, 512, 0, 513, 8192], 1, 2, 2, 4, 0, "float16", 512, "nf4_asym"),
    ([3000, 700, 5], 5, 1, 7, 3, 2, "float32", 512, "uniform"),
    ([2500, 1000], 19, 2, 4, 2, 1, "bfloat16", 512, "nf4"),
    ([2000, 1999], 1, 4, 16, 9, 1, "bfloat16", 33, "nf4_asym"),
    ([4000], 3, 1, 16, 300, 1, "float32", 2, "nf4_asym"),
    ([1500, 40], 1000, 1, 2, 3, 1, "float16", 100, "uniform"),
    ([1200], 1, 1, 1, 7, 0, "float32", 512, "nf4"),
    ([900], 2, 1, 4, 1, 5, "bfloat16", 100, "nf4_asym"),
    ([6000], 1, 3, 9, 1, 0, "bfloat16", 100, "nf4_asym"),
    # about as many blocks as a CTA has threads to count with, and as many as it has threads
    ([126, 127, 128, 129, 130, 131, 132, 133], 3, 1, 2, 50, 1, "bfloat16", 2, "nf4_asym"),
    ([255, 256, 257, 258, 259, 260], 9, 2, 6, 129, 3, "float16", 2, "uniform"),
    # more scores than a CTA's shared memory holds
    ([2000] + [0] * 73 + [30], 8, 2, 2, 40, 1, "float16", 2, "nf4_asym"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_scores_in_64_bits(torch, case):
    lens, t, h, hq, n, first, dt, hot, keys = case
    gen = torch.Generator(device="cuda").manual_seed(sum(lens))
    ctx = _ctx(n_seqs=len(lens), n_kv_heads=h, n_q_heads=hq, kv_dtype=dt, hot_window=hot, key_mode=keys)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(len(lens), t, hq, 128, generator=gen, device="cuda").to(getattr(torch, dt))
    full = [t] * len(lens)
    part = [(i * 7 + 3) % (t + 1) for i in range(len(lens))]
    for q_lens in (None, torch.tensor(part, dtype=torch.int32, device="cuda")):
        got = ctx.select_blocks(0, q, n, first=first, q_lens=q_lens)
        assert got.dtype == torch.int32 and got.shape == (len(lens), t, h, n)
        for s, r in enumerate(full if q_lens is None else part):
            # (a thousand rows take the oracle long: some of them)
            some = range(t) if t < 50 else [0, 1, 63, 64, r - 2, r - 1, t - 1]
            want = _want(torch, ctx, 0, s, q[s], n, first, r) if t < 50 else None
            if want is None:
                want = torch.stack([_row(torch, ctx, s, q[s], i, n, first, r) for i in some])
            assert torch.equal(got[s, list(some)].cpu(), want), s
    assert ctx.status() == 0


def _row(torch, ctx, seq, q, i, n, first, q_n):
    """Row i of `_want`: that of a call with the queries up to it, of a sequence as long as it is."""
    if not 0 <= i < q_n:
        return torch.full((ctx.n_kv_heads, n), -1, dtype=torch.int32)
    one = torch.zeros_like(q)
    one[i] = q[i]
    return _want(torch, ctx, 0, seq, one[:i + 1], n, first, q_n)[i]


def test_copies_of_a_block_go_by_their_index(torch):
    ctx = _ctx(n_kv_heads=2, n_q_heads=4, kv_dtype="float32", hot_window=100)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(50, 2, 128, generator=gen, device="cuda")
    ctx.append(0, k.repeat(40, 1, 1)[None], k.repeat(40, 1, 1)[None])
    q = torch.randn(1, 1, 4, 128, generator=gen, device="cuda")
    got = ctx.select_blocks(0, q, 7, first=0)
    assert got[0, 0, 0].tolist() == got[0, 0, 1].tolist() == list(range(7))
    # a query of nothing: all scores are zero
    assert ctx.select_blocks(0, q * 0, 5, first=2)[0, 0, 1].tolist() == [0, 1, 2, 3, 4]
    # one block is not a copy, and better
    better = ctx.export_block(0, 0, 20)
    better["nf4_scale"] = better["nf4_scale"] * 4
    state = ctx.export_state(0, 0)
    ctx.clear(0, 0)
    blks = [ctx._from_blob(b, None) for b in state["blocks"]]
    blks[20] = better
    for i, b in enumerate(blks):
        ctx.import_block(0, 0, i, b)
    ctx.restore_hot(0, 0, 2000, *(torch.from_numpy(state[x]).view(torch.float32) for x in ("hot_k", "hot_v")))
    assert ctx.select_blocks(0, q, 4, first=1)[0, 0, 0].tolist() == [0, 1, 2, 20]


def test_queries_that_are_no_numbers(torch):
    ctx = _ctx(n_kv_heads=1, n_q_heads=2, kv_dtype="float32", hot_window=100)
    gen = torch.Generator(device="cuda").manual_seed(2)
    _fill(torch, ctx, [1000], gen)
    q = torch.randn(1, 1, 2, 128, generator=gen, device="cuda")
    q[0, 0, 0, 5] = float("nan")
    assert ctx.select_blocks(0, q, 4, first=0)[0, 0, 0].tolist() == [0, 1, 2, 3]  # (no score: the lowest)
    q[0, 0, 0, 5] = float("inf")
    got = ctx.select_blocks(0, q, 4, first=1)[0, 0, 0].tolist()
    assert got[0] == 0 and len(set(got)) == 4 and got == sorted(got)


def test_orders_of_the_queries_out_and_parts_of_the_batch(torch):
    ctx = _ctx(n_layers=2, n_seqs=3, n_kv_heads=2, n_q_heads=6, kv_dtype="bfloat16")
    gen = torch.Generator(device="cuda").manual_seed(3)
    _fill(torch, ctx, [2000, 3000, 900], gen, layer=1)
    q = torch.randn(2, 4, 6, 128, generator=gen, device="cuda").bfloat16()
    want = ctx.select_blocks(1, q, 3, seq_begin=1)
    assert torch.equal(want[0].cpu(), _want(torch, ctx, 1, 1, q[0], 3, 1, 4))
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")
    flat[1:] = q.flatten()
    for x in (q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), flat[1:].view(q.shape),
              q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(ctx.select_blocks(1, x, 3, seq_begin=1), want)
    out = torch.full((3, 4, 2, 3), 9, dtype=torch.int32, device="cuda")
    assert ctx.select_blocks(1, q, 3, seq_begin=1, out=out[:2]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:2], want) and bool((out[2] == 9).all())
    assert ctx.select_blocks(1, q[:0], 3).shape == (0, 4, 2, 3)
    assert ctx.select_blocks(1, q[:, :0], 3, seq_begin=1).shape == (2, 0, 2, 3)


def test_captured_calls_follow_the_lengths(torch):
    ctx = _ctx(n_kv_heads=2, n_q_heads=4, kv_dtype="bfloat16", max_tokens_per_seq=4096)
    gen = torch.Generator(device="cuda").manual_seed(4)
    _fill(torch, ctx, [600], gen)
    q = torch.randn(1, 1, 4, 128, generator=gen, device="cuda").bfloat16()
    ctx.select_blocks(0, q, 3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = ctx.select_blocks(0, q, 3)
    for _ in range(3):
        graph.replay()
        assert torch.equal(got, ctx.select_blocks(0, q, 3))
        more = torch.randn(1, 1000, 2, 128, generator=gen, device="cuda").bfloat16()
        ctx.append(0, more, more)
    graph.replay()
    assert torch.equal(got[0].cpu(), _want(torch, ctx, 0, 0, q[0], 3, 1, 1))


def test_another_stream(torch):
    ctx = _ctx(n_kv_heads=1, n_q_heads=4, kv_dtype="float16")
    gen = torch.Generator(device="cuda").manual_seed(5)
    _fill(torch, ctx, [4000], gen)
    q = torch.randn(1, 2, 4, 128, generator=gen, device="cuda").half()
    want = ctx.select_blocks(0, q, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ctx.select_blocks(0, q, 4)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(torch):
    ctx = _ctx(n_seqs=2, n_kv_heads=2, n_q_heads=4)
    q = torch.zeros(2, 1, 4, 128, device="cuda")
    for bad in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q.cpu()), dict(q=q.double()), dict(n=0), dict(first=-1),
                dict(q_lens=torch.zeros(1, dtype=torch.int32, device="cuda")), dict(seq_begin=1), dict(layer=1),
                dict(out=torch.zeros(2, 1, 2, 4, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.select_blocks(**{"layer": 0, "q": q, "n": 3, **bad})
    polar = _ctx(n_kv_heads=2, n_q_heads=4, key_mode="polar", key_bits=3, outlier_frac=0.0)
    with pytest.raises(NotImplementedError, match="polar"):
        polar.select_blocks(0, q[:1], 3)
