"""What a layer does on long, shared and many-axis contexts of the compressed cache, as cases that can be timed.

``select``  for every query token and KV head the blocks of the cache that it attends, by a cheap score from what a
            block stores per channel anyway, its zero-points and scales (``KVContext.select_blocks``).
``sparse``  attention on the codes of the blocks so chosen and on the uncompressed window
            (``KVContext.attend`` with ``blocks``).
``prefix``  attention of sequences that share a long beginning, which is stored and read once
            (``KVContext.attend`` with ``prefix``).
``axes``    norm and rotation of queries and keys whose positions have several axes, time, height and width of images
            and video (``norm_rope`` with ``axes``).

A cache is given as what an engine stores of it: the containers of its compressed blocks (packed codes, scales, zero-points,
outliers, norms) and the tokens of the uncompressed window.  Keys and values are standard normal times a per-channel
log-normal scale, with 3 of 128 key channels per head a further x20, a constant part in every eighth, and a part that
all tokens of a block have in common, as neighbouring tokens do; queries are standard normal.
"""

import math

import numpy as np
import torch

own = False

D = 128
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}

# (KV heads, query heads, value bits) of the geometries the configurations and the model table name
SHAPES = {"mha": (32, 32, 4), "8b": (8, 32, 3), "70b": (8, 64, 4), "27b": (16, 32, 3), "7b": (4, 28, 3)}

NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
       -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
       0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941,
       0.7229568362236023, 1.0)
LLOYD = {3: (-1.748, -1.050, -0.500, -0.069, 0.069, 0.500, 1.050, 1.748),
         4: (-2.401, -1.844, -1.437, -1.099, -0.800, -0.524, -0.262, -0.066,
             0.066, 0.262, 0.524, 0.800, 1.099, 1.437, 1.844, 2.401)}
OUTLIER_FRAC = 0.02
# frequencies of each axis (time, height, width), one after the other or in turn
SECTIONS = {"runs": (16, 24, 24), "turns": (22, 21, 21), "two": (32, 32)}


def _cached(kind, shape, tokens, rows, top, *, name=None, batch=1, low=0, rows_low=0, dtype="bfloat16", bits=None,
            hot=512, keys="nf4_asym", first=1):
    h, hq, vb = SHAPES[shape]
    c = {"kind": kind, "heads": h, "q_heads": hq, "value_bits": bits or vb, "tokens": tokens, "low": low or tokens,
         "batch": batch, "rows": rows, "rows_low": rows_low or rows, "dtype": dtype, "hot": hot, "keys": keys,
         "top": top, "first": first}
    return c if name is None else dict(c, name=name)


def _prefix(shape, prefix, tokens, rows, *, name=None, batch=1, low=0, dtype="bfloat16", bits=None, hot=512,
            keys="nf4_asym"):
    h, hq, vb = SHAPES[shape]
    c = {"kind": "prefix", "heads": h, "q_heads": hq, "value_bits": bits or vb, "prefix": prefix, "tokens": tokens,
         "low": low or tokens, "batch": batch, "rows": rows, "rows_low": rows, "dtype": dtype, "hot": hot,
         "keys": keys}
    return c if name is None else dict(c, name=name)


def _axes(shape, batch, tokens, *, name=None, dtype="bfloat16", axes="runs", start=0, theta=1000000.0, normed="qk"):
    h, hq, _ = SHAPES[shape]
    c = {"kind": "axes", "heads": h, "q_heads": hq, "batch": batch, "tokens": tokens, "dtype": dtype, "axes": axes,
         "start": start, "theta": theta, "normed": normed}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a single user's decode step in a layer of the 8B model: the smallest choice, latency
        _cached("select", "8b", 8191, 1, 8, name="select_b1_8k"),
        # a serving batch of requests of every length, eight query heads per KV head
        _cached("select", "70b", 32768, 1, 32, name="select_b16_ragged", batch=16, low=500, dtype="float16"),
        # drafts of five tokens to verify on long documents
        _cached("select", "8b", 131072, 5, 64, name="select_b2_128k_t5", batch=2, dtype="float32", keys="uniform"),
        # the same user's attention on a long document
        _cached("sparse", "8b", 32768, 1, 16, name="sparse_b1_32k"),
        # the serving batch's, on 32 blocks of up to 128
        _cached("sparse", "70b", 32768, 1, 32, name="sparse_b16_ragged", batch=16, low=500, dtype="float16"),
        # drafts of one to five tokens, seven query heads per KV head, each token with its own blocks
        _cached("sparse", "7b", 20001, 5, 24, name="sparse_b8_t5", batch=8, rows_low=1),
        # a few requests behind one instruction: the smallest shared beginning
        _prefix("8b", 2000, 100, 1, name="prefix_b4_2k", batch=4, low=10),
        # a serving batch behind a long instruction
        _prefix("8b", 8192, 600, 1, name="prefix_b32_8k", batch=32, low=50),
        # samples of one long document, eight query heads per KV head
        _prefix("70b", 32768, 500, 1, name="prefix_b64_32k", batch=64, low=1),
        # drafts of three tokens on a shared beginning of odd length
        _prefix("7b", 12345, 333, 3, name="prefix_f16_t3", batch=11, low=40, dtype="float16"),
        # a token that is decoded after a picture: the smallest rotation
        _axes("7b", 1, 1, name="axes_b1_t1", start=5000),
        # prompts with pictures
        _axes("8b", 4, 4001, name="axes_b4_t4001"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    shape = rng.choice(list(SHAPES))
    h, hq, _ = SHAPES[shape]
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    kind = rng.choice(["select", "sparse", "sparse", "prefix", "prefix", "axes"])
    if kind == "axes":
        total = _spread(rng, 1, 16000 * 40 // (h + hq))
        batch = min(total, _spread(rng, 1, 32))
        return _axes(shape, batch, max(1, total // batch), dtype=dtype, axes=rng.choice(list(SECTIONS)),
                     start=_spread(rng, 1, 1000000), theta=rng.choice([10000.0, 1000000.0]),
                     normed=rng.choice(["qk", "qk", "k", ""]))
    hot = rng.choice([512, 512, 512, 512, 100, 33])
    keys = rng.choice(["nf4_asym", "nf4_asym", "nf4", "uniform"])
    bits = rng.choice([3, 4])
    if kind == "prefix":
        prefix, rows = _spread(rng, 64, 32768 if hot == 512 else 4000), rng.choice([1, 1, 2, 5, 17])
        most = min(64, max(1, 64 * 32768 * 64 // (prefix * rows * hq)))
        if dtype == "float32":
            most = min(most, max(1, 40_000_000 // (prefix * rows * hq)))
        batch, tokens = _spread(rng, 1, most), _spread(rng, rows, 1000)
        return _prefix(shape, prefix, tokens, rows, batch=batch, low=max(rows, tokens // rng.choice([1, 3, 20])),
                       dtype=dtype, bits=bits, hot=hot, keys=keys)
    tokens = _spread(rng, 300, 131072 if hot == 512 else 8000)
    blocks = max(1, tokens // ((hot + 1) // 2))
    batch = _spread(rng, 1, max(1, min(32, 2_000_000 // (tokens * h))))
    rows = rng.choice([1, 1, 1, 2, 5, 16])
    top = _spread(rng, 1, min(blocks, 64) if kind == "select" else min(blocks, 40))
    if kind == "sparse":  # (no more than the largest listed case attends)
        rows = max(1, min(rows, 16 * 8 * 32 * 256 * 8 // (batch * hq * top * ((hot + 1) // 2))))
        batch = max(1, min(batch, 16 * 8 * 32 * 256 * 8 // (rows * hq * top * ((hot + 1) // 2))))
    return _cached(kind, shape, tokens, rows, top, batch=batch, low=max(1, tokens // rng.choice([1, 2, 20])),
                   rows_low=max(1, rows // rng.choice([1, 3])), dtype=dtype, bits=bits, hot=hot, keys=keys,
                   first=rng.choice([0, 1, 1, 2]))


# ---- what a case holds -----------------------------------------------------------------------
def _even(low, high, n):
    """n whole numbers spread evenly over [low, high], in a scattered order."""
    order = np.argsort((np.arange(n) * 0.6180339887) % 1.0)
    return [int(low + (high - low) * (i + 0.5) / n) if low < high else int(high) for i in order]


def _cold(case, n):
    """Blocks of a sequence of n tokens, and the tokens of one."""
    s = (case["hot"] + 1) // 2
    return (0 if n <= case["hot"] else 1 + (n - case["hot"] - 1) // s), s


def _geometry(case):
    """Tokens and query tokens of every sequence, tokens of a block, compressed blocks of every sequence."""
    lens = _even(case["low"], case["tokens"], case["batch"])
    rows = [min(r, case["rows"]) for r in _even(case["rows_low"], case["rows"], case["batch"])]
    if case["batch"] == 1:
        lens, rows = [case["tokens"]], [case["rows"]]
    return lens, rows, _cold(case, 1)[1], [_cold(case, n)[0] for n in lens]


def _token_bytes(case):
    """Bytes of a compressed token of a KV head."""
    s = (case["hot"] + 1) // 2
    return D // 2 + D * case["value_bits"] // 8 + 4 + (8 * D + 4 * max(1, round(s * OUTLIER_FRAC)) * D) / s


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    h, hq = case["heads"], case["q_heads"]
    if case["kind"] == "axes":
        n = case["batch"] * case["tokens"] * (h + hq)
        return {"bytes": 2 * n * D * size, "flops": 8 * n * D}
    lens, rows, s, blocks = _geometry(case)
    q = sum(rows) * hq * D
    if case["kind"] == "select":
        each = (4 if case["keys"] == "nf4" else 8) * D  # symmetric keys have no zero-points
        return {"bytes": h * sum(blocks) * each + q * size + sum(rows) * h * case["top"] * 4,
                "flops": 4 * D * h * sum(r * b for r, b in zip(rows, blocks))}
    if case["kind"] == "sparse":
        chosen = [min(b, case["top"]) for b in blocks]
        hot = [n - b * s for n, b in zip(lens, blocks)]
        return {"bytes": int(h * (sum(chosen) * s * _token_bytes(case) + sum(hot) * 2 * D * size) + 2 * q * size
                             + sum(rows) * h * case["top"] * 4),
                "flops": 4 * D * hq * sum(r * (c * s + w) for r, c, w in zip(rows, chosen, hot)) + 2 * D * q}
    nb, _ = _cold(case, case["prefix"])
    cold = nb * s + s * sum(blocks)
    hot = case["prefix"] - nb * s + sum(n - b * s for n, b in zip(lens, blocks))
    return {"bytes": int(h * (cold * _token_bytes(case) + hot * 2 * D * size) + 2 * q * size),
            "flops": 4 * D * hq * sum(r * (case["prefix"] + n) for r, n in zip(rows, lens)) + 2 * D * q}


# ---- inputs ------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    return gen


def _normal(gen, shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _axis_of(case):
    """The axis of every frequency."""
    sizes = SECTIONS[case["axes"]]
    if case["axes"] != "turns":
        return [a for a, n in enumerate(sizes) for _ in range(n)]
    return [i % len(sizes) for i in range(sum(sizes))]


def _prepare_axes(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    b, t, h, hq = case["batch"], case["tokens"], case["heads"], case["q_heads"]
    # what a fused projection hands over: q, k and v of a token next to each other
    qkv = (_normal(gen, (b, t, hq + 2 * h, D)) * torch.exp(0.5 * _normal(gen, (hq + 2 * h, D)))).to(dtype)
    half = D // 2
    inv_freq = torch.tensor(case["theta"] ** (-np.arange(half) / half), dtype=torch.float32, device="cuda")
    # text, then a picture of some width in patches, whose tokens share their time, then text again
    at = torch.arange(t, device="cuda")
    begin = torch.randint(0, t // 4 + 1, (b, 1), generator=gen, device="cuda")
    wide = torch.randint(8, 65, (b, 1), generator=gen, device="cuda")
    n = t // 2
    within = (at >= begin) & (at < begin + n)
    i = at - begin
    behind = torch.where(at >= begin + n, i - n + begin + torch.maximum((n + wide - 1) // wide, wide), at)
    axes = [torch.where(within, begin, behind), torch.where(within, begin + i // wide, behind),
            torch.where(within, begin + i % wide, behind)]
    positions = torch.stack(axes[-len(SECTIONS[case["axes"]]):]) + case["start"]
    weight = [torch.exp(0.3 * _normal(gen, (D,))).to(dtype) if which in case["normed"] else None for which in "qk"]
    return {"case": case, "q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + h], "positions": positions, "inv_freq": inv_freq,
            "axes": torch.tensor(_axis_of(case), dtype=torch.uint8, device="cuda"), "q_weight": weight[0],
            "k_weight": weight[1]}


def _pack_keys(codes):
    """Two codes a byte, the first in the high half, the bits of each reversed."""
    turn = torch.tensor([int(f"{i:04b}"[::-1], 2) for i in range(16)], dtype=torch.uint8, device="cuda")
    c = turn[codes.long()]
    return (c[..., 0::2] << 4) | c[..., 1::2]


def _pack_values(codes, bits):
    """A stream of codes, lowest bit first."""
    c = codes.reshape(*codes.shape[:-1], D // 8, 8).long()
    word = (c << (bits * torch.arange(8, device="cuda"))).sum(-1)
    return ((word[..., None] >> (8 * torch.arange(bits, device="cuda"))) & 255).to(torch.uint8).flatten(-2)


def _centroids(case):
    return torch.tensor(np.asarray(LLOYD[case["value_bits"]]) / math.sqrt(D), dtype=torch.float32, device="cuda")


def _grid(case):
    return torch.tensor(NF4 if case["keys"] != "uniform" else tuple(range(16)), dtype=torch.float32, device="cuda")


def _some_blocks(gen, case, n_blocks, scale, shift, pi_t, sv):
    h, s = case["heads"], (case["hot"] + 1) // 2
    grid = _grid(case)
    common = 0.5 * _normal(gen, (n_blocks, h, 1, D))  # what the tokens of a block have in common
    x = (_normal(gen, (n_blocks, h, s, D)) + common) * scale[:, None] + shift[:, None]
    mean = x.mean(2) if case["keys"] == "nf4_asym" else torch.zeros_like(x[:, :, 0])
    k = max(1, round(s * OUTLIER_FRAC))
    far = (x - mean[:, :, None]).abs()
    at = far.topk(k, dim=2).indices
    idx = ((torch.arange(h, device="cuda")[:, None, None] * s + at) * D
           + torch.arange(D, device="cuda")).flatten(1).sort(1).values
    val = x.flatten(1).gather(1, idx).to(torch.float16)
    if case["keys"] == "uniform":
        inner = x.scatter(2, at, x.median(2, keepdim=True).values.expand_as(at))
        mean = inner.amin(2)
        step = (inner.amax(2) - mean) / 15.0
        codes = ((x - mean[:, :, None]) / step[:, :, None].clamp_min(1e-20)).round().clamp(0, 15).to(torch.uint8)
    else:
        far.scatter_(2, at, 0.0)
        step = far.amax(2)
        codes = torch.bucketize((x - mean[:, :, None]) / step[:, :, None].clamp_min(1e-20),
                                (grid[1:] + grid[:-1]) / 2).to(torch.uint8)
    v = _normal(gen, (n_blocks, h, s, D)) * sv[:, None]
    norms = v.norm(dim=-1)
    cent = _centroids(case)
    vc = torch.bucketize((v / norms[..., None]) @ pi_t, (cent[1:] + cent[:-1]) / 2).to(torch.uint8)
    return {"key_indices": _pack_keys(codes), "nf4_scale": step, "nf4_mean": mean,
            "outlier_idx": idx.to(torch.int32), "outlier_val": val,
            "value_indices": _pack_values(vc, case["value_bits"]), "value_norms": norms}


def _blocks(gen, case, n_blocks, *of):
    """Containers of `n_blocks` blocks: the keys' grid codes, scale, zero-point and outliers, the values' codes and
    norms; 128 at a time."""
    parts = [_some_blocks(gen, case, min(128, n_blocks - i), *of) for i in range(0, n_blocks, 128)]
    parts = parts or [_some_blocks(gen, case, 0, *of)]
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _inputs(case, seed):
    """The stored cache and the queries of a case, on the GPU, without this package."""
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    h, hq = case["heads"], case["q_heads"]
    lens, rows, s, blocks = _geometry(case)
    scale = torch.exp(0.5 * _normal(gen, (h, D)))
    sv = torch.exp(0.5 * _normal(gen, (h, D)))
    wide = torch.rand((h, D), generator=gen, device="cuda").argsort(1)[:, :3]
    scale.scatter_(1, wide, 20.0 * scale.gather(1, wide))
    shift = torch.where(torch.arange(D, device="cuda") % 8 == 0, 2.0, 0.0) * _normal(gen, (h, D))
    pi = torch.linalg.qr(_normal(gen, (D, D)))[0].contiguous()
    of = (scale, shift, pi.t(), sv)

    def stored(n_blocks, n_hot, n_seqs):
        parts = [_blocks(gen, case, n_blocks, *of) for _ in range(n_seqs)]
        st = {name: torch.stack([p[name] for p in parts]) for name in parts[0]}
        st["hot_k"] = (_normal(gen, (n_seqs, n_hot, h, D)) * scale + shift).to(dtype)
        st["hot_v"] = (_normal(gen, (n_seqs, n_hot, h, D)) * sv).to(dtype)
        return st

    state = stored(max(blocks), max(n - b * s for n, b in zip(lens, blocks)), len(lens))
    state["q"] = _normal(gen, (len(lens), case["rows"], hq, D)).to(dtype)
    state["pi"] = pi
    for name, values in (("lens", lens), ("q_lens", rows), ("blocks", blocks)):
        state[name] = torch.tensor(values, dtype=torch.int32, device="cuda")
    state["case"] = case
    if case["kind"] == "prefix":
        nb, _ = _cold(case, case["prefix"])
        state["shared"] = stored(nb, case["prefix"] - nb * s, 1)
    if case["kind"] == "sparse":  # what the choice before the attention has given
        state["chosen"] = _plain_select(state)
    return state


CONTAINERS = ("key_indices", "nf4_scale", "nf4_mean", "outlier_idx", "outlier_val", "value_indices", "value_norms")


def prepare(case, seed):
    if case["kind"] == "axes":
        return _prepare_axes(case, seed)
    state = _inputs(case, seed)
    if own:  # the cache that a user's program has filled: the same containers in a context
        from turboquant_pro_b200 import KVContext

        lens, _, s, blocks = _geometry(case)
        shared = case["kind"] == "prefix"
        # (the shared beginning is a sequence of its own, behind the others)
        ctx = state["ctx"] = KVContext(
            n_layers=1, n_seqs=case["batch"] + shared, n_kv_heads=case["heads"], n_q_heads=case["q_heads"],
            value_bits=case["value_bits"], hot_window=case["hot"], outlier_frac=OUTLIER_FRAC,
            max_tokens_per_seq=max(lens + [case.get("prefix", 0)]), kv_dtype=case["dtype"],
            pi=state["pi"].cpu().numpy(), key_mode=case["keys"])
        every = [(state, seq, n, b) for seq, (n, b) in enumerate(zip(lens, blocks))]
        if shared:
            every.append((state["shared"], 0, case["prefix"], _cold(case, case["prefix"])[0]))
        for seq, (of, at, n, b) in enumerate(every):
            ctx.import_blocks(0, seq, 0, {name: of[name][at, :b] for name in CONTAINERS})
            ctx.restore_hot(0, seq, n, of["hot_k"][at, :n - b * s], of["hot_v"][at, :n - b * s])
    return state


# ---- the plain forms -----------------------------------------------------------------------------
def _normed(x, weight, eps=1e-6):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _turned(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _plain_axes(state):
    of = state["positions"][state["axes"].long()].movedim(0, -1)  # the position that a frequency goes by
    angle = (of.double() * state["inv_freq"].double())[..., None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    return tuple(_turned(_normed(state[n], state[n + "_weight"]), cos, sin).to(state[n].dtype) for n in "qk")


def _positions(state):
    """``[batch, rows]``: where a query token stands, and -1 where there is none."""
    i = torch.arange(state["case"]["rows"], device="cuda")
    p = (state["lens"] - state["q_lens"])[:, None] + i
    return torch.where(i < state["q_lens"][:, None], p, -1).clamp_min(-1)


def _plain_select(state):
    """The highest sums over a group's query heads of the largest q . k that the block's grid allows."""
    case, q = state["case"], state["q"]
    h, s, nb = case["heads"], (case["hot"] + 1) // 2, state["nf4_scale"].shape[1]
    b, t = q.shape[:2]
    out = torch.full((b, t, h, case["top"]), -1, dtype=torch.int32, device="cuda")
    if nb == 0:
        return out
    # (in 64 bits: two blocks may be as good as each other but for the last of 24)
    x = q.double().view(b, t, h, -1, D)
    low, high = (0.0, 15.0) if case["keys"] == "uniform" else (-1.0, 1.0)
    up, down = x.clamp_min(0.0).sum(3), x.clamp_max(0.0).sum(3)
    score = torch.einsum("bthd,bnhd->bthn", up + down, state["nf4_mean"].double()) \
        + torch.einsum("bthd,bnhd->bthn", high * up + low * down, state["nf4_scale"].double())
    p, at = _positions(state)[:, :, None, None], torch.arange(nb, device="cuda")
    score = score.masked_fill((at < case["first"]) | (at == p // s), math.inf)
    there = (at < state["blocks"][:, None, None, None]) & (at * s <= p)
    score = score.masked_fill(~there, -math.inf)
    best = score.argsort(dim=-1, descending=True, stable=True)[..., :case["top"]]
    best = torch.where(there.expand_as(score).gather(-1, best), best, nb).sort(-1).values
    n = best.shape[-1]
    out[..., :n] = torch.where(best < nb, best, -1)
    return out


def _keys_of(case, c):
    """Dequantised keys of containers ``[..., heads, block tokens, D]``, without their outliers."""
    turn = torch.tensor([int(f"{i:04b}"[::-1], 2) for i in range(16)], dtype=torch.uint8, device="cuda")
    codes = torch.stack((turn[(c["key_indices"] >> 4).long()], turn[(c["key_indices"] & 15).long()]), -1).flatten(-2)
    return c["nf4_mean"][..., None, :] + c["nf4_scale"][..., None, :] * _grid(case)[codes.long()]


def _values_of(case, c, pi):
    vb = case["value_bits"]
    p = c["value_indices"]
    p = p.reshape(*p.shape[:-1], D // 8, vb).long()
    word = (p << (8 * torch.arange(vb, device="cuda"))).sum(-1)
    codes = ((word[..., None] >> (vb * torch.arange(8, device="cuda"))) & ((1 << vb) - 1)).flatten(-2)
    return (_centroids(case)[codes] @ pi) * c["value_norms"][..., None]


def _dense(case, c, pi):
    """Keys and values ``[sequences, heads, tokens of blocks, then of the window, D]``."""
    k = _keys_of(case, c)
    k = k.flatten(2).scatter(2, c["outlier_idx"].long(), c["outlier_val"].float()).view_as(k)
    v = _values_of(case, c, pi)
    return tuple(torch.cat((x.transpose(1, 2).flatten(2, 3), hot.float().transpose(1, 2)), 2)
                 for x, hot in ((k, c["hot_k"]), (v, c["hot_v"])))


def _softmax(scores):
    """Over the last dimension, in place; zeros where there is nothing."""
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(total.masked_fill(total == 0.0, 1.0))


def _plain_sparse(state):
    case, q = state["case"], state["q"]
    b, t, h, g = q.shape[0], case["rows"], case["heads"], case["q_heads"] // case["heads"]
    s, nb = (case["hot"] + 1) // 2, state["nf4_scale"].shape[1]
    p = _positions(state)
    x = q.float().view(b, t, h, g, D) * (1.0 / math.sqrt(D))
    # the window: token j of it is token blocks * s + j of the sequence
    j = (state["blocks"] * s)[:, None] + torch.arange(state["hot_k"].shape[1], device="cuda")
    seen = ((j < state["lens"][:, None])[:, None] & (j[:, None] <= p[..., None]))[:, :, None, None]
    near = torch.einsum("bthgd,bjhd->bthgj", x, state["hot_k"].float()).masked_fill(~seen, -math.inf)
    hot_v = state["hot_v"].float()
    if nb == 0:
        return torch.einsum("bthgj,bjhd->bthgd", _softmax(near), hot_v).reshape(q.shape).to(q.dtype)
    # the blocks that a query token's KV head has chosen: their containers, dequantised
    at = state["chosen"].long()
    there = (at >= 0) & (at < state["blocks"][:, None, None, None])
    at = at.clamp(0, nb - 1)
    seq, head = torch.arange(b, device="cuda")[:, None, None, None], torch.arange(h, device="cuda")[:, None]
    c = {name: state[name].view(b, nb, h, s, -1)[seq, at, head] for name in ("key_indices", "value_indices")}
    for name in ("nf4_scale", "nf4_mean", "value_norms"):
        c[name] = state[name][seq, at, head]
    k = _keys_of(case, c).flatten(-2)
    # outliers: as many in every block and channel, so that a head has its part of the block's list
    each = state["outlier_idx"].shape[2] // h
    idx = state["outlier_idx"].view(b, nb, h, each)[seq, at, head].long() - head[..., None] * (s * D)
    k.scatter_(-1, idx, state["outlier_val"].view(b, nb, h, each)[seq, at, head].float())
    k = k.view(b, t, h, -1, D)
    far = (x @ k.transpose(-1, -2)).view(b, t, h, g, -1, s)
    token = at[..., None] * s + torch.arange(s, device="cuda")
    seen = there[..., None] & (token <= p[:, :, None, None, None])
    far = far.masked_fill_(~seen[:, :, :, None], -math.inf).flatten(-2)
    w = _softmax(torch.cat((far, near), -1))
    out = w[..., :far.shape[-1]] @ _values_of(case, c, state["pi"]).flatten(-3, -2)
    out = out + torch.einsum("bthgj,bjhd->bthgd", w[..., far.shape[-1]:], hot_v)
    return out.reshape(q.shape).to(q.dtype)


def _plain_prefix(state):
    case, q = state["case"], state["q"]
    b, t, h, g = q.shape[0], case["rows"], case["heads"], case["q_heads"] // case["heads"]
    s, nb = (case["hot"] + 1) // 2, state["nf4_scale"].shape[1]
    p = _positions(state)
    x = q.float().view(b, t, h, g, D).permute(2, 0, 1, 3, 4) * (1.0 / math.sqrt(D))  # [heads, batch, t, g, D]
    k, v = (y[0] for y in _dense(case, state["shared"], state["pi"]))
    far = (x.reshape(h, -1, D) @ k.transpose(1, 2)).view(h, b, t, g, -1)
    there = (p >= 0)[:, :, None, None]
    far.masked_fill_(~there, -math.inf)
    ko, vo = _dense(case, state, state["pi"])  # [batch, heads, tokens, D]: blocks, then the window
    first_hot = (state["blocks"] * s)[:, None]
    cold, hot = torch.arange(nb * s, device="cuda")[None], first_hot + torch.arange(state["hot_k"].shape[1], device="cuda")
    j = torch.cat((cold.expand(b, -1), hot), 1)
    stored = torch.cat((cold < first_hot, hot < state["lens"][:, None]), 1)
    seen = (stored[:, None] & (j[:, None] <= p[..., None]))[:, :, None]
    near = torch.einsum("hbtgd,bhjd->hbtgj", x, ko).masked_fill(~seen, -math.inf)
    w = _softmax(torch.cat((far, near), -1))
    n = far.shape[-1]
    out = (w[..., :n].reshape(h, b * t * g, n) @ v).view(h, b, t, g, D)
    out = out + torch.einsum("hbtgj,bhjd->hbtgd", w[..., n:], vo)
    return out.permute(1, 2, 0, 3, 4).reshape(q.shape).to(q.dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"axes": _plain_axes, "select": _plain_select, "sparse": _plain_sparse,
                "prefix": _plain_prefix}[case["kind"]](state)
    if case["kind"] == "axes":
        from turboquant_pro_b200 import norm_rope

        return norm_rope(state["q"], state["k"], state["inv_freq"], state["positions"], q_weight=state["q_weight"],
                         k_weight=state["k_weight"], axes=state["axes"])
    ctx = state["ctx"]
    if case["kind"] == "select":
        return ctx.select_blocks(0, state["q"], case["top"], first=case["first"], q_lens=state["q_lens"])
    if case["kind"] == "sparse":
        return ctx.attend(0, state["q"], blocks=state["chosen"], q_lens=state["q_lens"])
    return ctx.attend(0, state["q"], prefix=case["batch"], q_lens=state["q_lens"])


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_axes(state):
    out = []
    axis = state["axes"].tolist()
    for name in ("q", "k"):
        x, w = state[name].double(), state[name + "_weight"]
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
        y = x.clone()
        for i, a in enumerate(axis):
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               state["positions"][a].double() * state["inv_freq"][i].double())[..., None]
            z = torch.complex(x[..., i], x[..., i + len(axis)]) * turn
            y[..., i], y[..., i + len(axis)] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_select(state):
    case = state["case"]
    lens, rows, s, blocks = _geometry(case)
    h, g = case["heads"], case["q_heads"] // case["heads"]
    out = torch.full((case["batch"], case["rows"], h, case["top"]), -1, dtype=torch.int32)
    low, high = (0, 15) if case["keys"] == "uniform" else (-1, 1)
    for seq, (n, r, nb) in enumerate(zip(lens, rows, blocks)):
        for i in range(r):
            p = n - r + i
            m = min(nb, p // s + 1) if p >= 0 else 0
            if m == 0:
                continue
            for head in range(h):
                mu, sc = state["nf4_mean"][seq, :m, head].double(), state["nf4_scale"][seq, :m, head].double()
                score = torch.zeros(m, dtype=torch.float64, device="cuda")
                for x in state["q"][seq, i, head * g:(head + 1) * g].double():
                    score += torch.maximum(x * (mu + low * sc), x * (mu + high * sc)).sum(-1)
                order = sorted(range(m), key=lambda b, of=score.tolist():
                               (0 if b < case["first"] or b == p // s else 1, -of[b], b))
                best = sorted(order[:case["top"]])
                out[seq, i, head, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out.cuda()


def _exact_block(case, of, seq, b, head, pi):
    """Keys and values of a block of a head."""
    s, vb = (case["hot"] + 1) // 2, case["value_bits"]
    flip = [int(f"{i:04b}"[::-1], 2) for i in range(16)]
    turn = torch.tensor([(flip[i >> 4], flip[i & 15]) for i in range(256)], device="cuda")
    codes = turn[of["key_indices"][seq, b, head].long()].flatten(1)
    key = of["nf4_mean"][seq, b, head].double() + of["nf4_scale"][seq, b, head].double() * _grid(case).double()[codes]
    idx = of["outlier_idx"][seq, b].long() - head * s * D
    mine = (idx >= 0) & (idx < s * D)
    key.view(-1)[idx[mine]] = of["outlier_val"][seq, b][mine].double()
    bits = (of["value_indices"][seq, b, head].long()[..., None] >> torch.arange(8, device="cuda")) & 1
    codes = (bits.reshape(s, D, vb) << torch.arange(vb, device="cuda")).sum(-1)
    return key, (_centroids(case).double()[codes] @ pi) * of["value_norms"][seq, b, head].double()[:, None]


def _exact_head(case, of, seq, n, head, pi):
    """Keys and values of all tokens of a sequence, of a head."""
    nb, s = _cold(case, n)
    parts = [_exact_block(case, of, seq, b, head, pi) for b in range(nb)]
    parts.append(tuple(of[name][seq, :n - nb * s, head].double() for name in ("hot_k", "hot_v")))
    return tuple(torch.cat([x[i] for x in parts]) for i in (0, 1))


def _exact_rows(q, key, value, sees):
    """Query heads ``[g, D]`` of one token on the keys that it sees."""
    if not bool(sees.any()):
        return torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    return torch.softmax(q.double() @ key[sees].t() / math.sqrt(D), -1) @ value[sees]


def _exact_sparse(state):
    case, pi = state["case"], state["pi"].double()
    lens, rows, s, blocks = _geometry(case)
    g = case["q_heads"] // case["heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    chosen = state["chosen"].cpu()
    for seq, (n, r, nb) in enumerate(zip(lens, rows, blocks)):
        for head in range(case["heads"]):
            made = {}
            window = tuple(state[name][seq, :n - nb * s, head].double() for name in ("hot_k", "hot_v"))
            for i in range(r):
                p = n - r + i
                of = [b for b in chosen[seq, i, head].tolist() if 0 <= b < nb]
                for b in of:
                    if b not in made:
                        made[b] = _exact_block(case, state, seq, b, head, pi)
                key, value = (torch.cat([made[b][x] for b in of] + [window[x]]) for x in (0, 1))
                j = torch.tensor([b * s for b in of], device="cuda")[:, None] + torch.arange(s, device="cuda")
                j = torch.cat((j.flatten().long(), torch.arange(nb * s, n, device="cuda")))
                out[seq, i, head * g:(head + 1) * g] = _exact_rows(
                    state["q"][seq, i, head * g:(head + 1) * g], key, value, j <= p)
    return out


def _exact_prefix(state):
    case, pi = state["case"], state["pi"].double()
    lens, rows, _, _ = _geometry(case)
    g = case["q_heads"] // case["heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for head in range(case["heads"]):
        pk, pv = _exact_head(case, state["shared"], 0, case["prefix"], head, pi)
        for seq, (n, r) in enumerate(zip(lens, rows)):
            key, value = (torch.cat(x) for x in zip((pk, pv), _exact_head(case, state, seq, n, head, pi)))
            for i in range(r):
                sees = torch.arange(len(key), device="cuda") <= len(pk) + n - r + i
                out[seq, i, head * g:(head + 1) * g] = _exact_rows(
                    state["q"][seq, i, head * g:(head + 1) * g], key, value, sees)
    return out


def exact(case, seed):
    if case["kind"] == "axes":
        return _exact_axes(_prepare_axes(case, seed))
    _, rows, _, blocks = _geometry(case)
    h = case["heads"]
    if case["kind"] == "select":
        return None if sum(rows) * h > 4000 else _exact_select(_inputs(case, seed))
    if case["kind"] == "sparse":
        few = sum(min(b, r * case["top"]) for b, r in zip(blocks, rows))
        return None if few * h > 12000 or sum(rows) * h > 6000 else _exact_sparse(_inputs(case, seed))
    few = sum(blocks) + _cold(case, case["prefix"])[0]
    return None if few * h > 12000 or sum(rows) * h > 12000 else _exact_prefix(_inputs(case, seed))
