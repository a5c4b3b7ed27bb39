"""tq_norm_rope with outputs that are its own inputs, which the header allows for contiguous tensors."""

from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, t, hq, hk, rotary", [(1, 1, 32, 8, 128), (2, 33, 28, 4, 96), (3, 700, 5, 1, 64), (1, 3, 1, 70, 8),
                                                  (2, 2500, 3, 2, 128)])
def test_an_output_may_be_its_own_input(torch, dtype, n, t, hq, hk, rotary):
    from turboquant_pro_b200 import _lib, norm_rope
    from turboquant_pro_b200.context import _dtype_codes

    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(t)
    q, k = (torch.randn(n, t, h, 128, generator=gen, device="cuda").to(dt) for h in (hq, hk))
    w = torch.rand(128, generator=gen, device="cuda").to(dt)
    f = torch.tensor([1e4 ** (-2 * i / rotary) for i in range(rotary // 2)], device="cuda")
    pos = torch.arange(n * t, device="cuda").view(n, t)
    for weights in ((w, w), (None, w), (None, None)):
        want = norm_rope(q, k, f, pos, q_weight=weights[0], k_weight=weights[1])
        x, y = q.clone(), k.clone()
        ptr = [None if u is None else u.data_ptr() for u in weights]
        r = _lib.TqRope(x.data_ptr(), y.data_ptr(), x.data_ptr(), y.data_ptr(), ptr[0], ptr[1], f.data_ptr(), pos.data_ptr(),
                        *x.stride()[:3], *y.stride()[:3], *pos.stride(), n, t, hq, hk, _dtype_codes()[dt],
                        _dtype_codes()[dt], 64, rotary, 1e-6)
        assert _lib.load().tq_norm_rope(C.byref(r), 0, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])
