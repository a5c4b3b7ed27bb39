"""The measures of ``attend_oracle`` see what they are for: results with a window or first tokens off by one, and with
tokens, tiles or parts of the history left out, are refused; rounded ones are not."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attend_oracle import attention, borders, limits, measures, values  # noqa: E402

CASES = [(1500, 1, 300, 4), (8000, 1, 6000, 100), (3500, 301, 1000, 130), (3500, 301, None, 0), (20000, 5, 15000, 64)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_measures_see_a_token(case):
    n, t, window, sinks = case
    gen = torch.Generator().manual_seed(1)
    v = values(n, 1, gen, "cpu", borders(n, t, window, sinks, n - 300)).transpose(0, 1)
    k = torch.randn(1, n, 128, generator=gen)
    q = torch.randn(t, 2, 128, generator=gen)
    want = attention(k, v, q, t, window, sinks)
    planted = {"a token of the history": dict(hidden=[slice(n - t - 1, n - t)]),
               "the newest token": dict(hidden=[slice(n - 1, n)]),
               "a tile": dict(hidden=[slice((n - t - 100) // 80 * 80, (n - t - 100) // 80 * 80 + 80)]),
               "queries a token too early": dict(q_n=t + 1)}
    if window is not None:
        planted.update({"window + 1": dict(window=window + 1), "window - 1": dict(window=window - 1),
                        "no first tokens": dict(sinks=0), "a first token less": dict(sinks=sinks - 1),
                        "a first token more": dict(sinks=sinks + 1)})
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        head, row = measures(want.to(dtype), want)
        assert head <= 0.6 * limits(dtype)[0] and row <= limits(dtype)[1]
        for name, other in planted.items():
            wrong = attention(k, v, q, **{"q_n": t, "window": window, "sinks": sinks, **other}).to(dtype)
            head, row = measures(wrong, want)
            assert head > 1.5 * limits(dtype)[0] or row > 1.5 * limits(dtype)[1], (dtype, name, head, row)


def test_the_measure_of_pairs_sees_keys_without_low_parts():
    from attend_oracle import PAIRS

    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, 3000, 128, generator=gen) for _ in range(2))
    q = (4.0 * torch.randn(64, 2, 128, generator=gen)).half()
    want = attention(k, v, q, 64, None, 0)
    assert measures(want.half(), want)[0] <= 0.6 * PAIRS
    assert measures(attention(k.half(), v, q, 64, None, 0).half(), want)[0] > 1.25 * PAIRS
