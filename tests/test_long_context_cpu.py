"""Refusals of the entry points for selected blocks and positions of several axes that need no device, and the layouts of
their arguments."""

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


@pytest.mark.parametrize("rope, axes", [
    ({}, dict(axes=None)), ({}, dict(n_axes=0)), ({}, dict(n_axes=-1)), (dict(positions=None), {}),
    (dict(rotary_dim=12), {}), (dict(q=None), {})])
def test_norm_rope_axes_refuses(lib, rope, axes):
    from turboquant_pro_b200._lib import TqRopeAxes

    x = TqRopeAxes(256, 1, 3)
    for name, v in axes.items():
        setattr(x, name, v)
    assert lib.tq_norm_rope_axes(C.byref(_rope(**rope)), C.byref(x), 0, None) < 0
    assert lib.tq_last_error()


def test_null_arguments(lib):
    from turboquant_pro_b200._lib import TqAttendArgs, TqSelectArgs

    size = C.c_size_t()
    assert lib.tq_norm_rope_axes(None, None, 0, None) == -1
    assert lib.tq_ctx_norm_rope_after(None, 0, 0, -1, C.byref(_rope()), None) == -1
    assert lib.tq_select_blocks(None, C.byref(TqSelectArgs()), None) == -1
    assert lib.tq_attend_blocks(None, C.byref(TqAttendArgs()), None, 1, None) == -1
    assert lib.tq_attend_blocks_workspace(None, C.byref(TqAttendArgs()), 1, None, C.byref(size)) == -1
    assert lib.tq_attend_prefix(None, C.byref(TqAttendArgs()), 0, None) == -1
    assert lib.tq_attend_prefix_workspace(None, C.byref(TqAttendArgs()), 0, None, C.byref(size)) == -1
    assert lib.tq_select_blocks_workspace(None, C.byref(TqSelectArgs()), None, C.byref(size)) == -1


def test_norm_rope_axes_of_host_tensors_is_refused():
    import torch

    from turboquant_pro_b200 import norm_rope

    q, k = torch.zeros(1, 3, 4, 128), torch.zeros(1, 3, 2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        norm_rope(q, k, torch.zeros(64), torch.zeros(3, 1, 3, dtype=torch.long), axes=torch.zeros(64, dtype=torch.uint8))


def test_struct_layouts():
    from turboquant_pro_b200._lib import TqRopeAxes, TqSelectArgs

    assert C.sizeof(TqRopeAxes) == 8 + 8 + 2 * 4
    assert C.sizeof(TqSelectArgs) == 5 * 8 + 3 * 8 + 8 * 4
