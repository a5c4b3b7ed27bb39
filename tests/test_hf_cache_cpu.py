"""The transformers adapter's choices, without a GPU."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")


def test_masks_that_are_the_causal_one_and_masks_that_are_not():
    from turboquant_pro_b200.hf_cache import _causal, _mask_is_causal, _mask_is_open

    t, n = 3, 7
    for window in (None, 2):
        sees = _causal(t, n, window, "cpu")
        assert sees.tolist() == [[j <= p and (window is None or j > p - window) for j in range(n)] for p in range(n - t, n)]
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            low = torch.finfo(dtype).min
            add = torch.zeros(2, 1, t, n, dtype=dtype).masked_fill(~sees, low)
            assert _mask_is_causal(add, t, n, window) and _mask_is_causal(add.masked_fill(~sees, -math.inf), t, n, window)
            for at, value in (((0, 0, 0, 4), 0.5), ((0, 0, 2, 6), -1.0), ((0, 0, 0, 6), -1.0), ((1, 0, 0, 5), 0.0)):
                other = add.clone()
                other[at] = value
                assert not _mask_is_causal(other, t, n, window), (at, value)
        assert _mask_is_causal(sees[None, None].expand(2, 1, t, n), t, n, window)
        assert not _mask_is_causal(torch.ones(2, 1, t, n, dtype=torch.bool), t, n, window)
        assert not _mask_is_causal(sees[None, None, :, 1:], t, n, window)
    pad = torch.ones(2, n, dtype=torch.int64)
    assert _mask_is_causal(pad, t, n, None) and _mask_is_open(pad)
    pad = pad.clone()
    pad[1, 0] = 0
    assert not _mask_is_causal(pad, t, n, None) and not _mask_is_open(pad)
    assert _mask_is_open(None) and _mask_is_open(torch.zeros(2, 1, 1, n))
    assert not _mask_is_open(torch.full((2, 1, 1, n), 0.25)) and not _mask_is_open(torch.full((2, 1, 1, n), -1.0))


def test_the_device_is_asked_once_per_mask():
    from turboquant_pro_b200 import hf_cache

    asked = []
    masks = [torch.ones(2, 1, 3, 7, dtype=torch.bool) for _ in range(3)]
    for _ in range(5):  # (layers)
        for i, m in enumerate(masks):
            hf_cache._remembered(m, (3, 7, None), lambda i=i: asked.append(i) or torch.tensor(True))
    assert asked == [0, 1, 2]
