"""KVContext.import_blocks: containers that are tensors on the device, bit for bit what import_block writes."""

from __future__ import annotations

import numpy as np
import pytest
from test_gpu_readback import H, _context

pytestmark = pytest.mark.gpu

NAMES = ("key_indices", "nf4_scale", "nf4_mean", "value_indices", "value_norms", "outlier_idx", "outlier_val")


def _stack(torch, blocks, device):
    out = {}
    for name in NAMES:
        parts = [None if b.get(name) is None else torch.from_numpy(np.array(b[name])).to(device) for b in blocks]
        same = parts[0] is not None and len({p.shape for p in parts}) == 1
        out[name] = torch.stack(parts) if same else None if parts[0] is None else parts
    return out


@pytest.mark.parametrize("mode,frac,vb,dt,w,n", [
    ("nf4_asym", 0.02, 3, "float16", 512, 1500), ("nf4", 0.036, 4, "bfloat16", 512, 1100),
    ("uniform", 0.0, 3, "float32", 512, 800), ("nf4_asym", 0.1, 4, "float16", 100, 500),
    ("nf4_asym", 0.5, 3, "float32", 2, 40)])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_tensors_give_the_pages_of_the_one_block_form(mode, frac, vb, dt, w, n, device):
    import torch

    from turboquant_pro_b200 import KVContext

    src, _, _, kw = _context(torch, w, vb, dt, n, mode=mode, frac=frac)
    nb = src.cold_blocks(n)
    one = [src.export_block(1, 1, b) for b in range(nb)]
    a, b = KVContext(**kw), KVContext(**kw)
    for blk in range(nb):
        a.import_block(1, 1, blk, one[blk])
    b.import_blocks(1, 1, 0, _stack(torch, one[:2], device))
    b.import_blocks(1, 1, 2, _stack(torch, one[2:], device)) if nb > 2 else None
    b.import_blocks(1, 1, 0, {name: x if x is None else x[:0] for name, x in _stack(torch, one[:1], device).items()})
    for name in ("pages", "pool_dec", "pool_val", "page_meta", "state"):
        assert torch.equal(a._regions[name], b._regions[name]), name
    hot = [torch.randn(n - nb * src.block_tokens, H, 128, device="cuda").to(src.kv_dtype) for _ in range(2)]
    for c in (a, b):
        c.restore_hot(1, 1, n, *hot)
    for x, y in zip(a.dequant(1, 1, 0, n), b.dequant(1, 1, 0, n)):
        assert torch.equal(x, y)


def test_containers_that_do_not_fit_are_refused():
    import torch

    from turboquant_pro_b200 import KVContext

    src, _, _, kw = _context(torch, 512, 3, "float16", 1500)
    nb = src.cold_blocks(1500)
    good = _stack(torch, [src.export_block(1, 1, b) for b in range(nb)], "cuda")
    ctx = KVContext(**kw)
    idx, val = good["outlier_idx"], good["outlier_val"]
    bad = [dict(good, **{name: good[name][:, :-1]}) for name in ("key_indices", "value_indices")]
    bad += [dict(good, nf4_scale=good["nf4_scale"][:-1]), dict(good, value_norms=good["value_norms"][:, :, :-1])]
    bad += [dict(good, outlier_idx=i) for i in (
        [i.flip(0) for i in idx], [i - i[0] - 1 for i in idx], [i + 10**6 for i in idx], [i.long() + 2**32 for i in idx],
        [i.float() for i in idx], [i[:1].expand_as(i) for i in idx], [i[:-1] for i in idx], idx[:-1],
        [idx[0], *[i[:-1] for i in idx[1:]]])]
    bad += [dict(good, outlier_val=[v.float() for v in val]), dict(good, outlier_val=[v.bfloat16() for v in val])]
    for containers in bad:
        with pytest.raises(ValueError):
            ctx.import_blocks(1, 1, 0, containers)
    for args in ((0, 9, 0), (9, 0, 0), (-1, 0, 0)):
        with pytest.raises(ValueError):
            ctx.import_blocks(*args, good)
    with pytest.raises(RuntimeError):
        ctx.import_blocks(1, 1, ctx.geom.max_blocks, good)
    ctx.import_blocks(1, 1, 0, good)
    ctx.restore_hot(1, 1, 1500, *(torch.zeros(1500 - nb * ctx.block_tokens, H, 128, device="cuda") for _ in range(2)))
    with pytest.raises(ValueError):  # (not a cleared cache any more)
        ctx.import_blocks(1, 1, 0, good)
