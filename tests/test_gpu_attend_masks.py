"""Every form of KVContext.attend by the measures of ``attend_oracle``, which a token too many or too few exceeds
(``test_attend_oracle.py``): windows, first tokens, padded batches, at lengths where worst-case bounds see nothing."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from attend_oracle import attention, borders, check, values  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


def _context(lens, heads, group, kv, hot, keys, bits, t, window, sinks, seed):
    from turboquant_pro_b200 import KVContext

    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx = KVContext(n_layers=1, n_seqs=len(lens), n_kv_heads=heads, n_q_heads=heads * group, kv_dtype=kv, hot_window=hot,
                    key_mode=keys, value_bits=bits, key_bits=bits if keys == "polar" else 4, seed=3,
                    outlier_frac=0.0 if keys == "polar" else 0.02, max_tokens_per_seq=max(lens))
    for s, n in enumerate(lens):
        if n == 0:
            continue
        v = values(n, heads, gen, "cuda", borders(n, t, window, sinks, ctx.cold_blocks(n) * ctx.block_tokens))
        k = torch.randn(n, heads, 128, generator=gen, device="cuda")
        ctx.append(0, k[None].to(ctx.kv_dtype), v[None].to(ctx.kv_dtype), seq_begin=s)
    return ctx, gen


CASES = [
    # lens, T, KV heads, group, window, sinks, hot, keys, value bits
    ([8000, 777, 0, 300], 1, 2, 4, None, 0, 512, "nf4_asym", 3),
    ([8000, 6101, 40], 1, 2, 4, 6000, 100, 512, "nf4_asym", 4),
    ([1500, 513, 512], 1, 1, 8, 300, 4, 512, "uniform", 3),
    ([3000, 2000], 5, 2, 7, 1111, 65, 512, "nf4_asym", 3),
    ([2500, 70, 5], 11, 1, 4, None, 0, 512, "nf4", 4),
    ([3500, 900], 301, 1, 4, None, 0, 512, "nf4_asym", 3),
    ([3500, 2000], 301, 1, 4, 1000, 130, 512, "nf4_asym", 4),
    ([6000], 777, 2, 2, 2000, 16, 512, "uniform", 3),
    ([9000], 64, 2, 4, 7777, 81, 512, "nf4_asym", 3),
    ([1000, 600], 1, 1, 4, 400, 33, 200, "nf4_asym", 3),
    ([1000, 600], 130, 1, 3, 400, 33, 200, "nf4_asym", 4),
    ([700, 333], 9, 2, 2, 111, 7, 33, "nf4_asym", 3),
    ([1200, 500], 40, 1, 4, 300, 5, 512, "polar", 4),
]


@pytest.mark.parametrize("kv", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_no_token_too_many_or_too_few(case, dtype, kv):
    lens, t, heads, group, window, sinks, hot, keys, bits = case
    ctx, gen = _context(lens, heads, group, kv, hot, keys, bits, t, window, sinks, 61)
    q = torch.randn(len(lens), t, heads * group, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    q_lens = torch.tensor([max(t - 2 * i, 0) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    for of in (None, q_lens):
        got = ctx.attend(0, q, window=window, sinks=sinks, q_lens=of)
        for s, n in enumerate(lens):
            if n == 0:
                assert not bool(got[s].any())
                continue
            k, v = ctx.dequant(0, s, 0, n)
            want = attention(k, v, q[s], t if of is None else int(of[s]), window, sinks)
            check(got[s], want)
    assert ctx.status() == 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("t, window, sinks", [(1, None, 0), (1, 60000, 100), (3, 60000, 100), (150, 60000, 100), (150, None, 0)])
@pytest.mark.parametrize("hot", [512, 200])
def test_no_token_too_many_or_too_few_in_a_long_history(dtype, t, window, sinks, hot):
    n = 70001
    ctx, gen = _context([n], 1, 2, dtype, hot, "nf4_asym", 3, t, window, sinks, 62)
    q = torch.randn(1, t, 2, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    k, v = ctx.dequant(0, 0, 0, n)
    check(ctx.attend(0, q, window=window, sinks=sinks)[0], attention(k, v, q[0], t, window, sinks))
    assert ctx.status() == 0


@pytest.mark.parametrize("kv", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("t, hot", [(1, 512), (12, 512), (200, 512), (200, 200), (3, 200)])
def test_float16_queries_meet_keys_and_values_as_pairs(t, hot, kv):
    from attend_oracle import PAIRS, measures
    from turboquant_pro_b200 import KVContext

    gen = torch.Generator(device="cuda").manual_seed(63)
    n = 3000
    ctx = KVContext(n_layers=1, n_seqs=1, n_kv_heads=2, n_q_heads=8, kv_dtype=kv, hot_window=hot, seed=3,
                    max_tokens_per_seq=n)
    ctx.append(0, *(torch.randn(1, n, 2, 128, generator=gen, device="cuda").to(ctx.kv_dtype) for _ in range(2)))
    q = (4.0 * torch.randn(1, t, 8, 128, generator=gen, device="cuda")).half()
    k, v = ctx.dequant(0, 0, 0, n)
    for window, sinks in ((None, 0), (1000, 70)):
        got = ctx.attend(0, q, window=window, sinks=sinks)[0]
        assert measures(got, attention(k, v, q[0], t, window, sinks))[0] <= PAIRS
