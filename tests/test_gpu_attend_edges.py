"""KVContext.attend at the ends of its arguments' ranges, in all of its forms: against attention in 64 bits over
the dequantised keys and values, within the bounds that ``test_gpu_attend.py`` derives."""

from __future__ import annotations

import pytest

from test_gpu_attend import _check, _ctx, _fill

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    return torch


# rows of one KV head and tokens of the window that take each form: few rows, many, general
FORMS = [(2, 512), (300, 512), (300, 200), (2, 200)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, hot", FORMS)
def test_largest_windows_and_sinks(torch, dtype, rows, hot):
    gen = torch.Generator(device="cuda").manual_seed(51)
    ctx = _ctx(n_seqs=2, n_kv_heads=1, n_q_heads=2, kv_dtype=dtype, hot_window=hot)
    _fill(torch, ctx, [1300, 600], gen)
    q = torch.randn(2, rows, 2, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    for window, sinks in ((7, 2**31 - 1), (2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (2**40, 2**40), (1, 2**31 - 80)):
        got = ctx.attend(0, q, window=window, sinks=sinks)
        _check(torch, ctx, got, q, window, sinks)
    assert ctx.status() == 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [60, 129, 700])
@pytest.mark.parametrize("image", [0, 1, 5, 24])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(torch, dtype, rows, image):
    """Many rows: the test hook withholds the copy of one operand image (keys or values, of the first tile or a
    later one) and shortens the probe limit; the call returns, the status word has bit 1, and nothing of it is left."""
    from turboquant_pro_b200._lib import TqError

    gen = torch.Generator(device="cuda").manual_seed(52)
    # (enough units that a CTA has a dozen tiles)
    ctx = _ctx(n_seqs=2, n_kv_heads=37, n_q_heads=74, kv_dtype=dtype, hot_window=300)
    _fill(torch, ctx, [2500, 2500], gen)
    q = torch.randn(2, rows, 74, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    good = ctx.attend(0, q, window=2200)
    assert ctx.status() == 0 and ctx.last_launches() == 4
    ctx.debug_wait(wait_limit=64, withhold_tile=image)
    ctx.attend(0, q, window=2200)
    with pytest.raises(TqError, match="wait"):
        ctx.raise_on_timeout()
    assert ctx.status() == 0
    ctx.debug_wait()
    assert torch.equal(ctx.attend(0, q, window=2200), good)
    assert ctx.status() == 0


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, t, heads", [(1, 1, 4), (2, 1, 4), (1, 3, 4), (1, 1, 1), (3, 1, 1), (1, 5, 1), (2, 6, 1)])
def test_views_of_odd_rows_with_sizes_of_one(torch, dtype, n, t, heads):
    """Any strides: views of rows that are no multiple of 16 bytes, begun on and off a 16-byte boundary, where torch
    takes tensors with sizes of one for contiguous whatever their strides."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(53)
    ctx = _ctx(n_seqs=n, n_kv_heads=1, n_q_heads=heads, kv_dtype=dtype)
    _fill(torch, ctx, [700] * n, gen)
    q = torch.randn(n, t, heads, 128, generator=gen, device="cuda").to(dt)
    want = ctx.attend(0, q, window=90, sinks=2)
    _check(torch, ctx, want, q, 90, 2)
    for off in (0, 3, 8):
        for row in (heads * 128 + 1, heads * 128 + 24):
            flat = torch.zeros(n * t * row + 16, dtype=dt, device="cuda")
            for strides in ((t * row, row, 128, 1), (row, n * row, 128, 1)):
                view = flat.as_strided(q.shape, strides, off)
                view.copy_(q)
                assert torch.equal(ctx.attend(0, view, window=90, sinks=2), want), (off, strides)
        wide = torch.zeros(n, t, heads, 131, dtype=dt, device="cuda")
        wide[..., off // 3:off // 3 + 128] = q
        assert torch.equal(ctx.attend(0, wide[..., off // 3:off // 3 + 128], window=90, sinks=2), want)


def _scaled(torch, n, heads, gen, k_by, v_by=1.0):
    k = k_by * torch.randn(1, n, heads, 128, generator=gen, device="cuda")
    v = v_by * torch.randn(1, n, heads, 128, generator=gen, device="cuda")
    return k, v


@pytest.mark.parametrize("t", [1, 9])
@pytest.mark.parametrize("by", [2.0**-20, 2.0**-13, 2.0**-6, 2.0**8, 2.0**20])
def test_float32_digits_do_not_depend_on_the_size_of_keys_and_values(torch, t, by):
    """Few rows: small (large) keys against large (small) queries are the same scores."""
    gen = torch.Generator(device="cuda").manual_seed(54)
    # (outliers are stored in half precision, which ends at 65504: keys of 2^20 have none)
    ctx = _ctx(n_seqs=1, n_kv_heads=2, n_q_heads=4, kv_dtype="float32", outlier_frac=0.02 if by < 2.0**10 else 0.0)
    ctx.append(0, *_scaled(torch, 1200, 2, gen, by, 1.0 / by))
    q = torch.randn(1, t, 4, 128, generator=gen, device="cuda") / by
    for window, sinks in ((None, 0), (300, 3)):
        _check(torch, ctx, ctx.attend(0, q, window=window, sinks=sinks), q, window, sinks)


@pytest.mark.parametrize("t", [1, 9])
@pytest.mark.parametrize("by", [2.0**30, 2.0**-30])
def test_float32_digits_do_not_depend_on_the_neighbours(torch, t, by):
    """Few rows: every third token's keys and values are 2^30 times (a 2^30th of) the others'; where they are larger
    a window hides them, so that the others are all there is."""
    gen = torch.Generator(device="cuda").manual_seed(55)
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=4, kv_dtype="float32", outlier_frac=0.0)
    k, v = _scaled(torch, 512, 1, gen, 1.0)
    if by > 1.0:
        k[0, :500:3] *= by
        v[0, :500:3] *= by
    else:
        k[0, ::3] *= by
        v[0, ::3] *= by
    ctx.append(0, k, v)
    q = torch.randn(1, t, 4, 128, generator=gen, device="cuda")
    window = 14 - t if by > 1.0 else None  # (of the newest twelve and fewer, none is a larger one)
    _check(torch, ctx, ctx.attend(0, q, window=window), q, window)


@pytest.mark.parametrize("kv", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, hot", [(1, 512), (9, 512), (300, 512), (5, 200), (300, 200)])
def test_an_infinite_key_may_take_all_weight_from_its_token(torch, kv, dtype, rows, hot):
    """A visible key of -inf where the queries are positive: its score is -inf, its weight zero, and the output that
    of the other tokens."""
    gen = torch.Generator(device="cuda").manual_seed(56)
    ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=2, kv_dtype=kv, hot_window=hot)
    k, v = (x.to(ctx.kv_dtype) for x in _scaled(torch, 700, 1, gen, 1.0))
    q = torch.randn(1, rows, 2, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    q[..., 17] = q[..., 17].abs() + 1.0
    k[0, 640, 0, 17] = -float("inf")  # in the uncompressed window
    ctx.append(0, k, v)
    kk, vv = (x[0].double() for x in ctx.dequant(0, 0, 0, 700))
    u = 2.0**-22 if dtype == "float32" else 2.0**-11
    p, j = torch.arange(700 - rows, 700, device="cuda")[:, None], torch.arange(700, device="cuda")
    for window, sinks in ((None, 0), (100, 2)):
        got = ctx.attend(0, q, window=window, sinks=sinks)[0].double()
        sees = (j <= p) & (j != 640)  # (without the token)
        if window is not None:
            sees &= (j > p - window) | (j < sinks)
        for h in range(2):
            x = q[0, :, h].double()
            kf = kk.masked_fill(kk.isinf(), 0.0)
            want = torch.softmax((x @ kf.t() / 128**0.5).masked_fill(~sees, -float("inf")), 1) @ vv
            a = (x.abs() @ kf.abs().t() / 128**0.5).masked_fill(~sees, 0.0).amax(1, keepdim=True)
            limit = (2 * a + 4) * u * vv.abs().max() + torch.finfo(q.dtype).eps / 2 * want.abs()
            assert bool(((got[:, h] - want).abs() <= limit).all()), (window, h)


def test_padding_that_is_no_number_slows_nothing_down_and_stays_out(torch):
    """Rows of a padded batch hold NaN: zeros for them, the others as without."""
    gen = torch.Generator(device="cuda").manual_seed(57)
    for dtype in ("float16", "bfloat16", "float32"):
        ctx = _ctx(n_seqs=2, n_kv_heads=1, n_q_heads=2, kv_dtype=dtype)
        _fill(torch, ctx, [900, 700], gen)
        for rows in (9, 300):
            q = torch.randn(2, rows, 2, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
            lens = torch.tensor([rows // 2, rows], dtype=torch.int32, device="cuda")
            want = ctx.attend(0, q, q_lens=lens)
            _check(torch, ctx, want, q, q_lens=lens)
            q[0, rows // 2:] = float("nan")
            assert torch.equal(ctx.attend(0, q, q_lens=lens), want)


def _relative(torch, ctx, got, q, window=None, sinks=0, q_lens=None, seq_begin=0):
    """The largest relative error (2-norms over a query head's rows) against 64 bits."""
    from test_gpu_attend import _want

    worst = 0.0
    for s in range(q.shape[0]):
        q_n = q.shape[1] if q_lens is None else int(q_lens[s])
        want, _ = _want(torch, ctx, 0, seq_begin + s, q[s], q_n, window, sinks)
        off = (got[s].double() - want).norm(dim=(0, 2)) / want.norm(dim=(0, 2)).clamp_min(1e-300)
        worst = max(worst, float(off.max()))
    return worst


def _step(torch, dtype):
    """What ``_relative`` may give for scores of standard deviation one.  16-bit queries: half a step of the output's
    type; its rounding alone is 0.42 of that in the mean square, and half-precision probabilities, values and keys (2^-11 at worst) add
    less than 0.6 in all (``attend_oracle.py``).  float32: 2^-20, four parts of 2^-22 (the pairs of queries, keys,
    probabilities and values); float32 sums of 128 products are below that."""
    return 2.0**-20 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("kv", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, hot", FORMS)
def test_digits_do_not_depend_on_the_size_of_the_keys(torch, kv, dtype, rows, hot):
    """Small (large) keys against large (small) queries are the same scores."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(58)
    for by in (2.0**-8, 1.0, 2.0**8) if "float16" in (kv, dtype) else \
            (2.0**-28, 2.0**-20, 2.0**-13, 2.0**-6, 2.0**9):
        # (Outliers are stored in half precision, and beside it as their distance from the grid, in half precision too:
        # below 2^-14 both have a step of 2^-24, so that of keys of 2^-28, step 2^-24 / 2^-28 = 16, nothing is left of them
        # in the cache itself.  Such keys have none here.)
        ctx = _ctx(n_seqs=1, n_kv_heads=1, n_q_heads=2, kv_dtype=kv, hot_window=hot,
                   outlier_frac=0.02 if by >= 2.0**-8 else 0.0)
        ctx.append(0, *(x.to(ctx.kv_dtype) for x in _scaled(torch, 1300, 1, gen, by)))
        q = (torch.randn(1, rows, 2, 128, generator=gen, device="cuda") / by).to(dt)
        for window, sinks in ((None, 0), (700, 20)):
            got = ctx.attend(0, q, window=window, sinks=sinks)
            rel = _relative(torch, ctx, got, q, window, sinks)
            assert rel <= _step(torch, dt), (by, window, rel)
        assert ctx.status() == 0


@pytest.mark.parametrize("kv", ["float32", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, hot", FORMS)
@pytest.mark.parametrize("part", ["keys", "values"])
def test_large_tokens_that_a_window_hides_take_no_digits(torch, kv, dtype, rows, hot, part):
    """Tokens 2^40 times the others stand next to those that are seen, in the uncompressed window or in blocks."""
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(59)
    for n in (500, 1300):
        ctx = _ctx(n_seqs=1, n_kv_heads=2, n_q_heads=4, kv_dtype=kv, hot_window=hot, outlier_frac=0.0)
        k, v = _scaled(torch, n, 2, gen, 1.0)
        first = n - rows - 100  # of the tokens that are seen
        at = slice(first - 7, first)
        if part == "keys":
            # (a block's channels have one scale for all of its tokens: large keys stay in the uncompressed window)
            if at.start < ctx.cold_blocks(n) * ctx.block_tokens:
                continue
            k[0, at, 1] *= 2.0**40
        else:
            v[0, at, 1] *= 2.0**40
        ctx.append(0, k.to(ctx.kv_dtype), v.to(ctx.kv_dtype))
        q = torch.randn(1, rows, 4, 128, generator=gen, device="cuda").to(dt)
        got = ctx.attend(0, q, window=101)
        rel = _relative(torch, ctx, got, q, 101)
        assert rel <= _step(torch, dt), (n, rel)
        assert ctx.status() == 0


def _told(torch, ctx, q, seq_begin, seq_count):
    """What tq_attend_workspace asks for."""
    import ctypes as C

    from turboquant_pro_b200 import _lib

    a = _lib.TqAttendArgs(q=q.data_ptr(), out=q.data_ptr(), q_seq_stride=q.stride(0), q_tok_stride=q.stride(1),
                          q_head_stride=q.stride(2), seq_begin=seq_begin, seq_count=seq_count, n_tokens=q.shape[1],
                          q_dtype={torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[q.dtype])
    size, stream = C.c_size_t(), torch.cuda.current_stream().cuda_stream
    assert ctx._lib.tq_attend_workspace(ctx._h, C.byref(a), stream, C.byref(size)) == 0
    return size.value


@pytest.mark.parametrize("dtype, t, lens, hot", [
    # one sequence takes the form for few rows, all of them that for many, whose share of a sequence is larger
    ("bfloat16", 16, [8192] * 8, 512), ("bfloat16", 16, [8192, 300, 0, 5000, 8000, 1, 700, 8192], 512),
    ("float16", 9, [6000] * 7, 512), ("float16", 5, [4000, 20, 3999] * 3, 200), ("float32", 30, [3000, 2000], 512)])
def test_workspace_of_what_one_sequence_needs_will_do(torch, dtype, t, lens, hot):
    from turboquant_pro_b200._lib import TqError

    gen = torch.Generator(device="cuda").manual_seed(60)
    ctx = _ctx(n_seqs=len(lens), n_kv_heads=8, n_q_heads=32, kv_dtype=dtype, hot_window=hot, max_tokens_per_seq=8192)
    _fill(torch, ctx, lens, gen)
    q = torch.randn(len(lens), t, 32, 128, generator=gen, device="cuda").to(getattr(torch, dtype))
    q_lens = torch.tensor([(5 * i + 3) % (t + 1) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    least = max(_told(torch, ctx, q, s, 1) for s in range(len(lens)))
    for lens_of in (None, q_lens):
        got = ctx.attend(0, q, q_lens=lens_of, max_workspace=least)
        _check(torch, ctx, got, q, q_lens=lens_of)
    out = torch.full_like(q, 3.0)
    with pytest.raises(TqError, match="workspace"):
        ctx.attend(0, q, max_workspace=256, out=out)
    with pytest.raises((TqError, ValueError)):
        ctx.attend(0, q, max_workspace=0, out=out)
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())


def test_a_step_with_arguments_of_another_type_appends_nothing(torch):
    ctx = _ctx(n_seqs=1, n_kv_heads=2, n_q_heads=4, kv_dtype="bfloat16")
    q, k, v = (torch.zeros(1, 3, h, 128, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2))
    f = torch.ones(64, device="cuda")
    for bad in (dict(window=2.5), dict(window="2"), dict(sinks=1.0), dict(sinks=None)):
        with pytest.raises(TypeError):
            ctx.step(0, q, k, v, f, **bad)
    assert ctx.lengths(0, 0)[0] == 0
    ctx.step(0, q, k, v, f, window=torch.tensor(2), sinks=True)
    assert ctx.lengths(0, 0)[0] == 3
