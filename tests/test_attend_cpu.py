"""Refusals of the attention and rotation entry points that need no device: the checks that stand before
any launch."""

from __future__ import annotations

import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge

    ge._load_build_module().build()
    from turboquant_pro_b200 import _lib

    return _lib.load()


def _rope(**kw):
    from turboquant_pro_b200._lib import TqRope

    r = TqRope()
    values = dict(q=256, k=256, q_out=256, k_out=256, inv_freq=256, positions=256, n_seqs=1, n_tokens=1,
                  n_q_heads=2, n_kv_heads=1, dtype=0, pos_bits=64, rotary_dim=128, eps=1e-6)
    for name, v in {**values, **kw}.items():
        setattr(r, name, v)
    return r


@pytest.mark.parametrize("bad, code", [
    (dict(n_seqs=-1), -1), (dict(n_tokens=-1), -1), (dict(n_q_heads=-1), -1), (dict(dtype=3), -1),
    (dict(weight_dtype=7), -1), (dict(rotary_dim=12), -2), (dict(rotary_dim=136), -2),
    (dict(rotary_dim=-8), -2), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(q=None), -1),
    (dict(k_out=None), -1), (dict(inv_freq=None), -1), (dict(positions=None), -1), (dict(pos_bits=16), -1),
    (dict(q_out=264), -1), (dict(n_seqs=1 << 20, n_tokens=1 << 20), -2),
])
def test_norm_rope_refuses(lib, bad, code):
    assert lib.tq_norm_rope(C.byref(_rope(**bad)), 0, None) == code
    assert lib.tq_last_error()


def test_null_arguments(lib):
    from turboquant_pro_b200._lib import TqAttendArgs

    size = C.c_size_t()
    assert lib.tq_norm_rope(None, 0, None) == -1
    assert lib.tq_ctx_norm_rope(None, 0, 0, C.byref(_rope()), None) == -1
    assert lib.tq_attend(None, C.byref(TqAttendArgs()), None) == -1
    assert lib.tq_attend_workspace(None, C.byref(TqAttendArgs()), None, C.byref(size)) == -1


def test_norm_rope_of_host_tensors_is_refused():
    import torch

    from turboquant_pro_b200 import norm_rope

    q, k = torch.zeros(1, 3, 4, 128), torch.zeros(1, 3, 2, 128)
    f, p = torch.zeros(64), torch.arange(3)
    with pytest.raises(ValueError, match="CUDA"):
        norm_rope(q, k, f, p)
    with pytest.raises(ValueError, match="positions"):
        norm_rope(q, k, f, None)
    with pytest.raises(ValueError, match="shape"):
        norm_rope(q[0], k, f, p)
    with pytest.raises(ValueError, match="shape"):
        norm_rope(q, k[:, :2], f, p)
    with pytest.raises(NotImplementedError, match="head_dim"):
        norm_rope(q[..., :64], k[..., :64], f, p)


def test_struct_layouts():
    """The ctypes mirrors are as long as the header's structs (no padding but what both have)."""
    from turboquant_pro_b200._lib import TqAttendArgs, TqRope

    assert C.sizeof(TqAttendArgs) == 5 * 8 + 3 * 8 + 8 * 4
    assert C.sizeof(TqRope) == 8 * 8 + 8 * 8 + 8 * 4 + 8
