"""What stands around a decode step on the compressed cache, as cases that can be timed.

``rope``    queries and keys of a layer, normed head by head and turned by their positions, as they go
            into ``KVContext.append`` and ``KVContext.attend`` (``norm_rope``).
``attend``  queries of one token or of many per sequence, attended on the codes of a filled cache
            (``KVContext.attend``): every token sees the tokens before it, those of a sliding window and
            a few first ones where the layer has such a window.

A cache is given as what an engine stores of it: the containers of its compressed blocks (packed codes,
scales, zero-points, outliers, norms) and the tokens of the uncompressed window.  Keys and values are
standard normal times a per-channel log-normal scale, with 3 of 128 key channels per head a further x20
and a constant part in every eighth; queries are standard normal.
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


def _rope(shape, batch, tokens, *, name=None, dtype="bfloat16", turned=D, start=0, theta=500000.0,
          normed="qk"):
    h, hq, _ = SHAPES[shape]
    c = {"kind": "rope", "heads": h, "q_heads": hq, "batch": batch, "tokens": tokens, "dtype": dtype,
         "turned": turned, "start": start, "theta": theta, "normed": normed}
    return c if name is None else dict(c, name=name)


def _attend(shape, tokens, rows, *, name=None, batch=1, low=0, rows_low=0, dtype="bfloat16", window=0,
            sinks=0, bits=None, hot=512, keys="nf4_asym"):
    h, hq, vb = SHAPES[shape]
    c = {"kind": "attend", "heads": h, "q_heads": hq, "value_bits": bits or vb, "tokens": tokens,
         "low": low or tokens, "batch": batch, "rows": rows, "rows_low": rows_low or rows, "dtype": dtype,
         "window": window, "sinks": sinks, "hot": hot, "keys": keys}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the token a single user decodes: the smallest call, launch and latency
        _rope("8b", 1, 1, name="rope_b1_t1", start=8191),
        # a batch of long prompts
        _rope("8b", 8, 2048, name="rope_b8_t2048", start=4096),
        # odd chunk of a few requests, half of the channels turned, only the keys normed, far positions
        _rope("70b", 7, 333, name="rope_b7_t333_half", dtype="float16", turned=64, start=900001,
              normed="k"),
        # a float32 multi-head model, as the cache class defaults to
        _rope("mha", 3, 1001, name="rope_f32_mha", dtype="float32", theta=10000.0),
        # a single user's decode step in a layer with a small window: latency
        _attend("8b", 3000, 1, name="window_b1_1k", window=1024, sinks=4),
        # a serving batch at the 8B model's full context, a layer with a 4k window
        _attend("8b", 8192, 1, name="window_b16_8k", batch=16, window=4096, sinks=4),
        # requests of every length, eight query heads per KV head, a window that is mostly hot
        _attend("70b", 5000, 1, name="window_b24_ragged", batch=24, low=100, dtype="float16",
                window=1000, sinks=64),
        # float32 queries through a multi-head cache
        _attend("mha", 2500, 1, name="window_f32_mha", dtype="float32", window=2000, sinks=1),
        # a batch whose drafts of one to five tokens are verified, whole history
        _attend("8b", 8000, 5, name="verify_b8_t5", batch=8, rows_low=1),
        # an odd chunk of a prompt in a windowed layer, seven query heads per KV head
        _attend("7b", 9001, 777, name="chunk_777_window", dtype="float16", window=2000, sinks=16),
        # chunks of long prompts, whole history
        _attend("8b", 16384, 512, name="chunk_512_16k"),
        _attend("8b", 32768, 2048, name="chunk_2048_32k"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    shape = rng.choice(list(SHAPES))
    h, hq, _ = SHAPES[shape]
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if rng.random() < 0.25:
        total = _spread(rng, 1, 16384 * 40 // (h + hq))
        batch = min(total, _spread(rng, 1, 32))
        return _rope(shape, batch, max(1, total // batch), dtype=dtype, turned=rng.choice([128, 128, 96, 64]),
                     start=_spread(rng, 1, 1000000), theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                     normed=rng.choice(["qk", "qk", "k", ""]))
    tokens = _spread(rng, 20, 32768)
    if rng.random() < 0.5:
        rows, batch = 1, _spread(rng, 1, max(1, min(32, 1_000_000 // (tokens * h))))
    else:
        rows = _spread(rng, 2, min(tokens, 2048))
        batch = _spread(rng, 1, max(1, min(8, 500_000 // (tokens * h), 65_000_000 * 32 // (tokens * rows * hq))))
        if tokens * rows * hq * batch > 65_000_000 * 32:
            rows = max(2, 65_000_000 * 32 // (tokens * hq * batch))
    if dtype == "float32":
        rows = min(rows, 200)
    windowed = rng.random() < 0.6
    return _attend(shape, tokens, rows, batch=batch, low=max(1, tokens // rng.choice([1, 2, 20])),
                   rows_low=max(1, rows // rng.choice([1, 1, 3])), dtype=dtype,
                   window=_spread(rng, 1, tokens) if windowed else 0,
                   sinks=_spread(rng, 1, 200) - 1 if windowed else 0, bits=rng.choice([3, 4]),
                   hot=rng.choice([512, 512, 512, 100, 33]),
                   keys=rng.choice(["nf4_asym", "nf4_asym", "nf4", "uniform"]))


# ---- what a case holds -----------------------------------------------------------------------
def _even(low, high, n):
    """n whole numbers spread evenly over [low, high], in a scattered order."""
    order = np.argsort((np.arange(n) * 0.6180339887) % 1.0)
    return [int(low + (high - low) * (i + 0.5) / n) if low < high else int(high) for i in order]


def _geometry(case):
    """Tokens and query tokens of every sequence, tokens of a block, compressed blocks of every sequence."""
    lens = _even(case["low"], case["tokens"], case["batch"])
    rows = [min(r, case["rows"]) for r in _even(case["rows_low"], case["rows"], case["batch"])]
    if case["batch"] == 1:
        lens, rows = [case["tokens"]], [case["rows"]]
    s, hot = (case["hot"] + 1) // 2, case["hot"]
    blocks = [0 if n <= hot else 1 + (n - hot - 1) // s for n in lens]
    return lens, rows, s, blocks


def _visible(case):
    """(visible (row, token) pairs of a query head, tokens that any row sees) over all sequences."""
    lens, rows, _, _ = _geometry(case)
    pairs = seen = 0
    for n, r in zip(lens, rows):
        p = np.arange(n - r, n)
        p = p[p >= 0]
        w = case["window"] or n + r
        near = np.minimum(p + 1, w)
        pairs += int((near + np.minimum(np.maximum(p + 1 - near, 0), case["sinks"])).sum())
        first = max(int(p[0]) + 1 - w, 0) if p.size else n
        seen += n - first + min(first, case["sinks"])
    return pairs, seen


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "rope":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["q_heads"])
        return {"bytes": 2 * n * D * size, "flops": 8 * n * D}
    lens, rows, s, blocks = _geometry(case)
    pairs, seen = _visible(case)
    hot = sum(n - b * s for n, b in zip(lens, blocks))
    cold = max(seen - hot, 0)
    k = max(1, round(s * OUTLIER_FRAC))
    per_token = D // 2 + D * case["value_bits"] // 8 + 4 + (8 * D + 4 * k * D) / s
    q = sum(rows) * case["q_heads"] * D
    return {"bytes": int(case["heads"] * (cold * per_token + min(seen, hot) * 2 * D * size) + 2 * q * size),
            "flops": 4 * D * case["q_heads"] * pairs + 2 * D * q}


# ---- inputs ------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    return gen


def _normal(gen, shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _prepare_rope(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    b, t, h, hq = case["batch"], case["tokens"], case["heads"], case["q_heads"]
    # what a fused projection hands over: q, k and v of a token next to each other
    qkv = (_normal(gen, (b, t, hq + 2 * h, D)) * torch.exp(0.5 * _normal(gen, (hq + 2 * h, D)))).to(dtype)
    half = case["turned"] // 2
    inv_freq = torch.tensor(case["theta"] ** (-np.arange(half) / half), dtype=torch.float32, device="cuda")
    starts = case["start"] + torch.randint(0, 1000, (b, 1), generator=gen, device="cuda")
    weight = [torch.exp(0.3 * _normal(gen, (D,))).to(dtype) if which in case["normed"] else None
              for which in "qk"]
    return {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + h], "positions": starts + torch.arange(t, device="cuda"),
            "inv_freq": inv_freq, "q_weight": weight[0], "k_weight": weight[1]}


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


def _blocks(gen, case, n_blocks, scale, shift, pi_t, sv):
    """Containers of `n_blocks` blocks: the keys' grid codes, scale, zero-point and outliers, the values' codes
    and norms."""
    h, s = case["heads"], (case["hot"] + 1) // 2
    grid = torch.tensor(NF4 if case["keys"] != "uniform" else tuple(range(16)), device="cuda")
    x = _normal(gen, (n_blocks, h, s, D)) * scale[:, None] + shift[:, None]
    mean = x.mean(2) if case["keys"] == "nf4_asym" else torch.zeros_like(x[:, :, 0])
    k = max(1, round(s * OUTLIER_FRAC))
    far = (x - mean[:, :, None]).abs()
    at = far.topk(k, dim=2).indices
    idx = ((torch.arange(h, device="cuda")[:, None, None] * s + at) * D
           + torch.arange(D, device="cuda")).flatten(1).sort(1).values
    val = x.flatten(1).gather(1, idx).to(torch.float16)
    if case["keys"] == "uniform":
        middle = x.median(2, keepdim=True).values
        inner = x.scatter(2, at, middle.expand_as(at))
        mean = inner.amin(2)
        step = (inner.amax(2) - mean) / 15.0
        codes = ((x - mean[:, :, None]) / step[:, :, None]).round().clamp(0, 15).to(torch.uint8)
    else:
        far.scatter_(2, at, 0.0)
        step = far.amax(2)
        edges = (grid[1:] + grid[:-1]) / 2
        codes = torch.bucketize((x - mean[:, :, None]) / step[:, :, None], edges).to(torch.uint8)
    v = _normal(gen, (n_blocks, h, s, D)) * sv[:, None]
    norms = v.norm(dim=-1)
    cent = _centroids(case)
    vc = torch.bucketize((v / norms[..., None]) @ pi_t, (cent[1:] + cent[:-1]) / 2).to(torch.uint8)
    return {"key_indices": _pack_keys(codes), "nf4_scale": step, "nf4_mean": mean,
            "outlier_idx": idx.to(torch.int32), "outlier_val": val,
            "value_indices": _pack_values(vc, case["value_bits"]), "value_norms": norms}


def _centroids(case):
    return torch.tensor(np.asarray(LLOYD[case["value_bits"]]) / math.sqrt(D), dtype=torch.float32, device="cuda")


def _inputs_attend(case, seed):
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
    nb, nh = max(blocks), max(n - b * s for n, b in zip(lens, blocks))
    parts = [_blocks(gen, case, nb, scale, shift, pi.t(), sv) for _ in lens]
    state = {name: torch.stack([p[name] for p in parts]) for name in parts[0]}
    state["hot_k"] = (_normal(gen, (len(lens), nh, h, D)) * scale + shift).to(dtype)
    state["hot_v"] = (_normal(gen, (len(lens), nh, h, D)) * sv).to(dtype)
    state["q"] = _normal(gen, (len(lens), case["rows"], hq, D)).to(dtype)
    state["pi"] = pi
    for name, values in (("lens", lens), ("q_lens", rows), ("blocks", blocks)):
        state[name] = torch.tensor(values, dtype=torch.int32, device="cuda")
    state["case"] = case
    return state


def prepare(case, seed):
    if case["kind"] == "rope":
        return dict(_prepare_rope(case, seed), case=case)
    state = _inputs_attend(case, seed)
    if own:  # the cache that a user's program has filled: the same containers in a context
        from turboquant_pro_b200 import KVContext

        lens, _, s, blocks = _geometry(case)
        state["ctx"] = KVContext(
            n_layers=1, n_seqs=case["batch"], n_kv_heads=case["heads"], n_q_heads=case["q_heads"],
            value_bits=case["value_bits"], hot_window=case["hot"], outlier_frac=OUTLIER_FRAC,
            max_tokens_per_seq=max(lens), kv_dtype=case["dtype"], pi=state["pi"].cpu().numpy(),
            key_mode=case["keys"])
        names = ("key_indices", "nf4_scale", "nf4_mean", "outlier_idx", "outlier_val", "value_indices", "value_norms")
        for seq, (n, b) in enumerate(zip(lens, blocks)):
            state["ctx"].import_blocks(0, seq, 0, {name: state[name][seq, :b] for name in names})
            state["ctx"].restore_hot(0, seq, n, state["hot_k"][seq, :n - b * s], state["hot_v"][seq, :n - b * s])
    return state


# ---- the plain form ----------------------------------------------------------------------------
def _normed(x, weight, eps=1e-6):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _turned(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _plain_rope(state):
    angle = state["positions"].double()[..., None, None] * state["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    return tuple(_turned(_normed(state[n], state[n + "_weight"]), cos, sin).to(state[n].dtype) for n in "qk")


def _dense_keys(state):
    """Keys ``[batch, heads, blocks * block tokens + window tokens, D]``, dequantised."""
    case = state["case"]
    s, h = (case["hot"] + 1) // 2, case["heads"]
    turn = torch.tensor([int(f"{i:04b}"[::-1], 2) for i in range(16)], dtype=torch.uint8, device="cuda")
    p = state["key_indices"]
    codes = torch.stack((turn[(p >> 4).long()], turn[(p & 15).long()]), -1).flatten(-2).long()
    grid = torch.tensor(NF4 if case["keys"] != "uniform" else tuple(range(16)), dtype=torch.float32, device="cuda")
    k = state["nf4_mean"][:, :, :, None] + state["nf4_scale"][:, :, :, None] * grid[codes]
    k = k.flatten(2).scatter(2, state["outlier_idx"].long(), state["outlier_val"].float()).view_as(k)
    b, nb = k.shape[:2]
    cold = k.permute(0, 2, 1, 3, 4).reshape(b, h, nb * s, D)
    return torch.cat((cold, state["hot_k"].float().transpose(1, 2)), 2)


def _dense_values(state):
    case = state["case"]
    s, h, vb = (case["hot"] + 1) // 2, case["heads"], case["value_bits"]
    p = state["value_indices"]
    p = p.reshape(*p.shape[:-1], D // 8, vb).long()
    word = (p << (8 * torch.arange(vb, device="cuda"))).sum(-1)
    codes = ((word[..., None] >> (vb * torch.arange(8, device="cuda"))) & ((1 << vb) - 1)).flatten(-2)
    v = (_centroids(case)[codes] @ state["pi"]) * state["value_norms"][..., None]
    b, nb = v.shape[:2]
    cold = v.permute(0, 2, 1, 3, 4).reshape(b, h, nb * s, D)
    return torch.cat((cold, state["hot_v"].float().transpose(1, 2)), 2)


def _hidden(state):
    """``[batch, rows, tokens]``: what a query token does not see."""
    case = state["case"]
    s, nb, nh = (case["hot"] + 1) // 2, state["key_indices"].shape[1], state["hot_k"].shape[1]
    first_hot = (state["blocks"] * s)[:, None]
    cold, hot = torch.arange(nb * s, device="cuda")[None], first_hot + torch.arange(nh, device="cuda")
    j = torch.cat((cold.expand(len(first_hot), -1), hot), 1)[:, None]
    stored = torch.cat(((cold < first_hot), (hot < state["lens"][:, None])), 1)[:, None]
    i = torch.arange(case["rows"], device="cuda")
    p = ((state["lens"] - state["q_lens"])[:, None] + i)[..., None]
    near = (j > p - case["window"]) | (j < case["sinks"]) if case["window"] else torch.ones_like(stored)
    return ~(stored & (j <= p) & near & (i < state["q_lens"][:, None])[..., None])


def _plain_attend(state):
    case, q = state["case"], state["q"]
    b, t, h, g = q.shape[0], case["rows"], case["heads"], case["q_heads"] // case["heads"]
    rows = q.float().view(b, t, h, g, D).permute(0, 2, 3, 1, 4).reshape(b, h, g * t, D)
    scores = rows @ (_dense_keys(state) * (1.0 / math.sqrt(D))).transpose(2, 3)
    hidden = _hidden(state)
    scores.view(b, h, g, t, -1).masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores @ _dense_values(state)) / total.masked_fill(total == 0.0, 1.0)
    return out.view(b, h, g, t, D).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)


def run(state):
    if state["case"]["kind"] == "rope":
        if own:
            from turboquant_pro_b200 import norm_rope

            return norm_rope(state["q"], state["k"], state["inv_freq"], state["positions"],
                             q_weight=state["q_weight"], k_weight=state["k_weight"])
        return _plain_rope(state)
    if own:
        case = state["case"]
        return state["ctx"].attend(0, state["q"], window=case["window"] or None, sinks=case["sinks"],
                                   q_lens=state["q_lens"])
    return _plain_attend(state)


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_rope(state):
    out = []
    for name in ("q", "k"):
        x, w = state[name].double(), state[name + "_weight"]
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
        half = state["inv_freq"].numel()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           state["positions"].double()[..., None] * state["inv_freq"].double())[..., None, :]
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        out.append(torch.cat((z.real, z.imag, x[..., 2 * half:]), -1))
    return tuple(out)


def _exact_attend(state):
    """Sequence by sequence and head by head, over the tokens it has; rows in pieces."""
    case = state["case"]
    s, vb, g = (case["hot"] + 1) // 2, case["value_bits"], case["q_heads"] // case["heads"]
    grid = torch.tensor(NF4 if case["keys"] != "uniform" else tuple(range(16)), dtype=torch.float32, device="cuda").double()
    cent, pi = _centroids(case).double(), state["pi"].double()
    flip = [int(f"{i:04b}"[::-1], 2) for i in range(16)]
    turn = torch.tensor([(flip[b >> 4], flip[b & 15]) for b in range(256)], device="cuda")
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lens, rows, _, blocks = _geometry(case)
    for seq, (n, r, nb) in enumerate(zip(lens, rows, blocks)):
        for h in range(case["heads"]):
            key = torch.empty((nb * s, D), dtype=torch.float64, device="cuda")
            value = torch.empty_like(key)
            for b in range(nb):
                codes = turn[state["key_indices"][seq, b, h].long()].flatten(1)
                dense = state["nf4_mean"][seq, b, h].double() + state["nf4_scale"][seq, b, h].double() * grid[codes]
                idx = state["outlier_idx"][seq, b].long() - h * s * D
                mine = (idx >= 0) & (idx < s * D)
                dense.view(-1)[idx[mine]] = state["outlier_val"][seq, b][mine].double()
                key[b * s:(b + 1) * s] = dense
                bits = (state["value_indices"][seq, b, h].long()[..., None] >> torch.arange(8, device="cuda")) & 1
                codes = (bits.reshape(s, D, vb) << torch.arange(vb, device="cuda")).sum(-1)
                value[b * s:(b + 1) * s] = (cent[codes] @ pi) * state["value_norms"][seq, b, h].double()[:, None]
            key = torch.cat((key, state["hot_k"][seq, :n - nb * s, h].double()))
            value = torch.cat((value, state["hot_v"][seq, :n - nb * s, h].double()))
            j = torch.arange(n, device="cuda")
            for i0 in range(0, r, 256):
                i = torch.arange(i0, min(i0 + 256, r), device="cuda")
                p = (n - r + i)[:, None]
                sees = j <= p
                if case["window"]:
                    sees &= (j > p - case["window"]) | (j < case["sinks"])
                x = state["q"][seq, i0:i0 + 256, h * g:(h + 1) * g][:len(i)].double() @ key.t() / math.sqrt(D)
                x = x.masked_fill(~sees[:, None], -math.inf)
                x = torch.softmax(x, -1).masked_fill(~sees.any(1)[:, None, None], 0.0)
                out[seq, i0:i0 + len(i), h * g:(h + 1) * g] = x @ value
    return out


def exact(case, seed):
    if case["kind"] == "rope":
        return _exact_rope(_prepare_rope(case, seed))
    if sum(_geometry(case)[3]) * case["heads"] > 60000:
        return None
    return _exact_attend(_inputs_attend(case, seed))
