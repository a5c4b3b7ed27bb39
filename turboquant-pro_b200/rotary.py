"""Norm and rotation of queries and keys, as they go into :meth:`KVContext.append` and
:meth:`KVContext.attend`.

The cache stores keys after their rotation (the reference's post-RoPE keys,
``turboquant_pro/per_channel_kv.py:243-267`` for the layout of a rotation's channels); this is the
pass that makes them, one kernel for both tensors.
"""

from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import TqRope, TqRopeAxes, check
from .context import _NO_GUARD, _dtype_codes, _raw_stream, _torch

__all__ = ["norm_rope"]

HEAD_DIM = 128


def norm_rope(q, k, inv_freq, positions, *, q_weight=None, k_weight=None, eps: float = 1e-6, axes=None):
    """Root-mean-square norm of every query and key head and their rotation by position, in one pass.

    ``q`` ``[n_seqs, T, n_q_heads, 128]``, ``k`` ``[n_seqs, T, n_kv_heads, 128]``: CUDA tensors of one
    type (float32 / float16 / bfloat16), any strides with contiguous channels (views of a fused
    projection are read where they are).  ``q_weight`` / ``k_weight`` ``[128]``: weights of the norm;
    ``None`` leaves that tensor as it is.  ``inv_freq``: float32 ``[rotary_dim / 2]``, angular
    frequency of channels ``i`` and ``i + rotary_dim / 2`` (``rotary_dim`` a multiple of 8; the channels
    after it are not turned).  ``positions``: int32 or int64, ``[n_seqs, T]`` or ``[T]``; angles
    are reduced in 64 bits, so far positions keep their precision.

    ``axes``: positions with several axes, as the time, height and width of images and video have them.  A uint8 CUDA tensor
    ``[rotary_dim / 2]`` with the axis that each frequency goes by (one after the other, or in turn);
    ``positions`` is then ``[n_axes, n_seqs, T]`` or ``[n_axes, T]``.  Numbers beyond the axes count as the last one.

    Returns new contiguous tensors ``(q, k)``, float32 arithmetic rounded once.  Inference only: no
    gradients.
    """
    if positions is None:
        raise ValueError("positions are needed (KVContext.norm_rope knows those of a cache)")
    return _norm_rope(q, k, inv_freq, positions, q_weight, k_weight, eps, axes, None)


def _weight(w, codes, other):
    if w.shape != (HEAD_DIM,) or w.dtype not in codes or (other is not None and w.dtype != other):
        raise ValueError(f"norm weights must be [{HEAD_DIM}] and of one floating type")
    return w.contiguous(), codes[w.dtype]


def _norm_rope(q, k, inv_freq, positions, q_weight, k_weight, eps, axes, cache):
    # (a decode step's call is a few microseconds on the GPU: the checks are kept short)
    torch = _torch()
    q_shape, k_shape, dev, dtype = q.shape, k.shape, q.device, q.dtype
    if len(q_shape) != 4 or len(k_shape) != 4 or q_shape[:2] != k_shape[:2]:
        raise ValueError(f"expected q, k of shape [n_seqs, T, heads, {HEAD_DIM}], got {tuple(q_shape)} "
                         f"and {tuple(k_shape)}")
    if q_shape[3] != HEAD_DIM or k_shape[3] != HEAD_DIM:
        raise NotImplementedError(f"only head_dim {HEAD_DIM} is implemented")
    if dev.type != "cuda":
        raise ValueError(f"q must be a CUDA tensor, it lives on {dev}")
    codes = _dtype_codes()
    if dtype not in codes or k.dtype != dtype:
        raise ValueError(f"q and k must share float32, float16 or bfloat16, got {dtype} and {k.dtype}")
    if k.device != dev or inv_freq.device != dev or (positions is not None and positions.device != dev) \
            or (q_weight is not None and q_weight.device != dev) \
            or (k_weight is not None and k_weight.device != dev) or (axes is not None and axes.device != dev):
        raise ValueError(f"k, inv_freq, positions, axes and weights must live where q does, on {dev}")
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or inv_freq.requires_grad
            or (q_weight is not None and q_weight.requires_grad)
            or (k_weight is not None and k_weight.requires_grad)):
        raise ValueError("norm_rope has no backward pass: call it under torch.no_grad()")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("inv_freq must be a float32 vector")
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    weight_type, qw, kw = 0, None, None
    if q_weight is not None:
        q_weight, weight_type = _weight(q_weight, codes, None if k_weight is None else k_weight.dtype)
        qw = q_weight.data_ptr()
    if k_weight is not None:
        k_weight, weight_type = _weight(k_weight, codes, None)
        kw = k_weight.data_ptr()
    n, t = q_shape[0], q_shape[1]
    pos, pos_bits, ps, pt, several = None, 0, 0, 0, None
    if axes is not None:
        if positions is None:
            raise ValueError("axes need positions")
        if axes.dtype != torch.uint8 or axes.shape != inv_freq.shape:
            raise ValueError(f"axes must be uint8, one for each of the {inv_freq.shape[0]} frequencies, got {axes.dtype} "
                             f"{tuple(axes.shape)}")
        if positions.dim() < 2 or positions.shape[0] < 1 or positions.shape[1:] not in ((n, t), (t,)):
            raise ValueError(f"positions must be [n_axes, {n}, {t}] or [n_axes, {t}], got {tuple(positions.shape)}")
        axes = axes.contiguous()
        several = TqRopeAxes(axes.data_ptr(), positions.stride(0), positions.shape[0])
        positions = positions[0]
    if positions is not None:
        if positions.dtype == torch.int64:
            pos_bits = 64
        elif positions.dtype == torch.int32:
            pos_bits = 32
        else:
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape == (n, t):
            ps, pt = positions.stride()
        elif positions.shape == (t,):
            pt = positions.stride(0)
        else:
            raise ValueError(f"positions must be [{n}, {t}] or [{t}], got {tuple(positions.shape)}")
        pos = positions.data_ptr()
    qs, ks = q.stride(), k.stride()
    if qs[3] != 1:
        q = q.contiguous()
        qs = q.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    inv_freq = inv_freq.contiguous()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    r = TqRope(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), qw, kw, inv_freq.data_ptr(), pos,
               qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], ps, pt,
               n, t, q_shape[2], k_shape[2], codes[dtype], weight_type, pos_bits,
               2 * inv_freq.shape[0], eps)
    lib, index = _lib.load(), dev.index
    with _NO_GUARD if torch.cuda.current_device() == index else torch.cuda.device(dev):
        stream = _raw_stream()(index)
        if cache is not None and positions is None:
            ctx, layer, seq_begin, prefix = cache
            check(lib.tq_ctx_norm_rope_after(ctx._h, layer, seq_begin, prefix, C.byref(r), stream))
        elif several is not None:
            check(lib.tq_norm_rope_axes(C.byref(r), C.byref(several), index, stream))
        else:
            check(lib.tq_norm_rope(C.byref(r), index, stream))
    return q_out, k_out
