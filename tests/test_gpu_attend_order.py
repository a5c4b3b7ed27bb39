"""KVContext.attend on listed blocks right behind the append that it has to see: sequences that fit the window, so that the
window's kernel is the call's first, queued behind work that keeps the GPU busy until all of it is in the stream."""

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


def _ctx(torch, b, dtype, start, gen):
    from turboquant_pro_b200 import KVContext

    # (no sequence can have a block: a captured call then begins with the window's kernel too)
    ctx = KVContext(n_layers=1, n_seqs=b, n_kv_heads=8, n_q_heads=64, kv_dtype=dtype, max_tokens_per_seq=512, seed=3)
    k, v = (torch.randn(b, start, 8, 128, generator=gen, device="cuda").to(ctx.kv_dtype) for _ in range(2))
    ctx.append(0, k, v)
    return ctx


def _steps(torch, b, t, dtype, gen, n):
    """Queries, keys and values; those values are large, so that a token that is not seen shows."""
    of = getattr(torch, dtype)
    for _ in range(n):
        q, k = (torch.randn(b, t, h, 128, generator=gen, device="cuda").to(of) for h in (64, 8))
        yield q, k, (oracle.LARGE * torch.randn(b, t, 8, 128, generator=gen, device="cuda")).to(of)


def _check(torch, ctx, got, q, n):
    for s in (0, q.shape[0] // 2, q.shape[0] - 1):
        k, v = ctx.dequant(0, s, 0, n)
        oracle.check(got[s], oracle.attention(k, v, q[s], q.shape[1], None, 0))


# by the rule for listed blocks a kernel of its own takes the window where it is more than 14 us of the rows' form's work
CASES = [("bfloat16", 64, 1, 400), ("bfloat16", 16, 5, 430), ("float16", 40, 1, 380), ("float16", 9, 7, 400)]


def _by_the_window(dtype, b, t, start):
    return (0.165 if dtype == "float16" else 0.085) * start * b * 8 * t / 1000 > 14


@pytest.mark.parametrize("dtype, b, t, start", CASES)
def test_attend_sees_what_was_appended_before_it(torch, dtype, b, t, start):
    assert _by_the_window(dtype, b, t, start)
    gen = torch.Generator(device="cuda").manual_seed(21)
    ctx, other = (_ctx(torch, b, dtype, start, torch.Generator(device="cuda").manual_seed(4)) for _ in range(2))
    lists = torch.full((b, t, 8, 3), -1, dtype=torch.int32, device="cuda")
    steps = list(_steps(torch, b, t, dtype, gen, 12))
    ctx.attend(0, steps[0][0], blocks=lists)
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)  # (some 20 ms: all of the calls are in the stream before the first one runs)
    got = []
    for q, k, v in steps:
        ctx.append(0, k, v)
        got.append(ctx.attend(0, q, blocks=lists))
        assert ctx.last_launches() == 1
    for i, (q, k, v) in enumerate(steps):
        other.append(0, k, v)
        torch.cuda.synchronize()
        want = other.attend(0, q, blocks=lists)
        torch.cuda.synchronize()
        assert torch.equal(got[i], want), i
    _check(torch, ctx, got[-1], steps[-1][0], start + 12 * t)
    assert ctx.status() == 0


@pytest.mark.parametrize("dtype, b, t, start", CASES[:3:2])
def test_captured_append_and_attend(torch, dtype, b, t, start):
    gen = torch.Generator(device="cuda").manual_seed(22)
    ctx, other = (_ctx(torch, b, dtype, start, torch.Generator(device="cuda").manual_seed(4)) for _ in range(2))
    lists = torch.full((b, t, 8, 3), -1, dtype=torch.int32, device="cuda")
    steps = list(_steps(torch, b, t, dtype, gen, 8))
    given = [x.clone() for x in steps[0]]
    other.attend(0, given[0], blocks=lists)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        ctx.append(0, *given[1:])
        out = ctx.attend(0, given[0], blocks=lists)
    got = []
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)
    for step in steps:
        for x, y in zip(given, step):
            x.copy_(y)
        graph.replay()
        got.append(out.clone())
    for i, (q, k, v) in enumerate(steps):
        other.append(0, k, v)
        torch.cuda.synchronize()
        want = other.attend(0, q, blocks=lists)
        torch.cuda.synchronize()
        assert torch.equal(got[i], want), i
    _check(torch, other, got[-1], steps[-1][0], start + 8 * t)
    assert ctx.status() == 0
