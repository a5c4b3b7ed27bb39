"""Norm and rotation of queries and keys, as they go into :meth:`KVContext.append` and
:meth:`KVContext.attend`.

The cache stores keys after their rotation (the reference's post-RoPE keys,
``turboquant_pro/per_channel_kv.py:243-267`` for the layout of a rotation's channels); this is the
pass that makes them, one kernel for both tensors.
"""

from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import TqRope, check
from .context import _dtype_code, _dtype_codes, _raw_stream, _torch

__all__ = ["norm_rope"]

HEAD_DIM = 128


def norm_rope(q, k, inv_freq, positions, *, q_weight=None, k_weight=None, eps: float = 1e-6):
    """Root-mean-square norm of every query and key head and their rotation by position, in one pass.

    ``q`` ``[n_seqs, T, n_q_heads, 128]``, ``k`` ``[n_seqs, T, n_kv_heads, 128]``: CUDA tensors of one
    type (float32 / float16 / bfloat16), any strides with contiguous channels (views of a fused
    projection are read where they are).  ``q_weight`` / ``k_weight`` ``[128]``: weights of the norm;
    ``None`` leaves that tensor as it is.  ``inv_freq``: float32 ``[rotary_dim / 2]``, angular
    frequency of channels ``i`` and ``i + rotary_dim / 2`` (``rotary_dim`` a multiple of 8; the channels
    after it are not turned).  ``positions``: int32 or int64, ``[n_seqs, T]`` or ``[T]``; angles
    are reduced in 64 bits, so far positions keep their precision.

    Returns new contiguous tensors ``(q, k)``, float32 arithmetic rounded once.  Inference only: no
    gradients.
    """
    if positions is None:
        raise ValueError("positions are needed (KVContext.norm_rope knows those of a cache)")
    return _norm_rope(q, k, inv_freq, positions, q_weight, k_weight, eps, None)


def _readable(t):
    """``t`` with contiguous channels."""
    return t if t.numel() == 0 or t.stride(-1) == 1 else t.contiguous()


def _norm_rope(q, k, inv_freq, positions, q_weight, k_weight, eps, cache):
    torch = _torch()
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2]:
        raise ValueError(f"expected q, k of shape [n_seqs, T, heads, {HEAD_DIM}], got {tuple(q.shape)} "
                         f"and {tuple(k.shape)}")
    if q.shape[3] != HEAD_DIM or k.shape[3] != HEAD_DIM:
        raise NotImplementedError(f"only head_dim {HEAD_DIM} is implemented")
    if q.device.type != "cuda":
        raise ValueError(f"q must be a CUDA tensor, it lives on {q.device}")
    if q.dtype not in _dtype_codes() or k.dtype != q.dtype:
        raise ValueError(f"q and k must share float32, float16 or bfloat16, got {q.dtype} and {k.dtype}")
    dev = q.device
    inputs = {"k": k, "inv_freq": inv_freq, "positions": positions, "q_weight": q_weight,
              "k_weight": k_weight}
    for name, t in inputs.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} lives on {t.device}, q on {dev}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (q, k, inv_freq, q_weight, k_weight)):
        raise ValueError("norm_rope has no backward pass: call it under torch.no_grad()")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("inv_freq must be a float32 vector")
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if tuple(w.shape) != (HEAD_DIM,) or w.dtype not in _dtype_codes() or w.dtype != weights[0].dtype:
            raise ValueError(f"norm weights must be [{HEAD_DIM}] and of one floating type")
    n, t = q.shape[:2]
    r = TqRope()
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((n, t), (t,)):
            raise ValueError(f"positions must be [{n}, {t}] or [{t}], got {tuple(positions.shape)}")
        positions = positions.expand(n, t)
        r.positions, r.pos_bits = positions.data_ptr(), 8 * positions.element_size()
        r.pos_seq_stride, r.pos_tok_stride = positions.stride()
    q, k, inv_freq = _readable(q), _readable(k), inv_freq.contiguous()
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    r.q, r.k, r.q_out, r.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    r.q_weight = q_weight.data_ptr() if q_weight is not None else None
    r.k_weight = k_weight.data_ptr() if k_weight is not None else None
    r.inv_freq = inv_freq.data_ptr()
    r.q_seq_stride, r.q_tok_stride, r.q_head_stride = q.stride()[:3]
    r.k_seq_stride, r.k_tok_stride, r.k_head_stride = k.stride()[:3]
    r.n_seqs, r.n_tokens, r.n_q_heads, r.n_kv_heads = n, t, q.shape[2], k.shape[2]
    r.dtype = _dtype_code(q.dtype)
    r.weight_dtype = _dtype_code(weights[0].dtype) if weights else 0
    r.rotary_dim, r.eps = 2 * inv_freq.numel(), eps
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _raw_stream()(dev.index)
        if cache is not None and positions is None:
            ctx, layer, seq_begin = cache
            check(lib.tq_ctx_norm_rope(ctx._h, layer, seq_begin, C.byref(r), stream))
        else:
            check(lib.tq_norm_rope(C.byref(r), dev.index, stream))
    return q_out, k_out
