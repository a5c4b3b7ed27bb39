"""The transformers adapter's choices, without a GPU: tiny random models run with a stand-in for the device
context that keeps what is appended as it is, so that prompts, single tokens and chunks, padded batches, sliding
windows, score capping and scales of a layer's own have to give what the model's eager attention gives on the
exact keys and values."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")


class _Context:
    """What the adapter uses of a KVContext, on plain tensors; notes the calls."""

    def __init__(self, n_seqs):
        self.n_seqs, self.kv, self.calls = n_seqs, {}, []

    def append(self, layer, k, v, seq_begin=0):
        old = self.kv.get(layer)
        self.kv[layer] = tuple(x.clone() if old is None else torch.cat((o, x), 1)
                               for x, o in zip((k, v), old or (None, None)))

    def clear(self, layer, seq=-1):
        self.kv.pop(layer, None)

    def dequant(self, layer, seq, start, end):
        return tuple(x[seq, start:end].transpose(0, 1).float() for x in self.kv[layer])

    def attend(self, layer, q, window=None, sinks=0):
        self.calls.append("attend")
        return self._attention(layer, q, window)

    def decode(self, layer, q):
        self.calls.append("decode")
        return self._attention(layer, q[:, None], None)[:, 0].float()

    def _attention(self, layer, q, window):
        k, v = (x.repeat_interleave(q.shape[2] // x.shape[2], 2) for x in self.kv[layer])
        n, t = k.shape[1], q.shape[1]
        p, j = torch.arange(n - t, n)[:, None], torch.arange(n)
        sees = (j <= p) & (j > p - (window or n))
        s = torch.einsum("bthd,bnhd->bhtn", q, k) / math.sqrt(q.shape[3])
        return torch.einsum("bhtn,bnhd->bthd", torch.softmax(s.masked_fill(~sees, -math.inf), -1), v)


COMMON = dict(vocab_size=97, hidden_size=64, intermediate_size=64, num_hidden_layers=3, num_attention_heads=4,
              num_key_value_heads=2, head_dim=32, max_position_embeddings=512)


def _model(kind):
    from transformers import (Gemma2Config, Gemma2ForCausalLM, LlamaConfig, LlamaForCausalLM, MistralConfig,
                              MistralForCausalLM)

    torch.manual_seed(3)
    if kind == "plain":
        model = LlamaForCausalLM(LlamaConfig(**COMMON))
    elif kind == "window":
        model = MistralForCausalLM(MistralConfig(sliding_window=8, **COMMON))
    else:  # windows in every second layer; capped scores, or a scale of its own
        cap, scalar = {"capped": (2.0, 32), "scaled": (None, 9)}[kind]
        model = Gemma2ForCausalLM(Gemma2Config(sliding_window=8, attn_logit_softcapping=cap, query_pre_attn_scalar=scalar,
                                               final_logit_softcapping=None, **COMMON))
    with torch.no_grad():  # (scores large enough that a token more or less, or a cap, shows)
        for name, p in model.named_parameters():
            if "q_proj" in name or "k_proj" in name:
                p.mul_(12.0)
    return model.eval()


PIECES = (20, 1, 1, 3, 1, 9, 1)  # a prompt, single tokens, chunks


def _logits(model, cache, ids, mask):
    out, at = [], 0
    with torch.no_grad():
        for t in PIECES:
            out.append(model(input_ids=ids[:, at:at + t], attention_mask=None if mask is None else mask[:, :at + t],
                             past_key_values=cache, use_cache=True).logits)
            at += t
    return torch.cat(out, 1)


@pytest.mark.parametrize("dense, attend", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("padding", ["none", "no mask", "left"])
@pytest.mark.parametrize("kind", ["plain", "window", "capped", "scaled"])
def test_generates_what_eager_attention_does(monkeypatch, kind, padding, dense, attend):
    from transformers import DynamicCache

    from turboquant_pro_b200 import hf_cache

    model, n = _model(kind), sum(PIECES)
    ids = torch.randint(1, 97, (2, n), generator=torch.Generator().manual_seed(1))
    mask = torch.ones(2, n, dtype=torch.int64)
    if padding == "left":
        mask[0, :6] = 0
    if padding == "no mask":
        mask = None
    model.config._attn_implementation = "eager"
    want = _logits(model, DynamicCache(), ids, mask)  # (a cache that keeps every token, for all layers)
    context = _Context(2)
    monkeypatch.setattr(hf_cache._SharedContext, "get", lambda self, key: context)
    cache = hf_cache.enable_turboquant_cache(model, dense=dense, attend=attend)
    got = _logits(model, cache, ids, mask)
    seen = torch.ones(2, n, dtype=torch.bool) if mask is None else mask.bool()
    assert torch.allclose(got[seen], want[seen], rtol=1e-3, atol=1e-4), (got - want)[seen].abs().max()
    # where nothing is padded the codes are used: by single tokens of layers without a window or anything of their own,
    # and with attend=True by chunks, and by layers with a window
    layers, single, chunks = 3, PIECES.count(1), len(PIECES) - PIECES.count(1) - 1
    decode = {"plain": layers, "window": 0, "capped": 0, "scaled": 0}[kind] * single
    more = {"plain": layers * chunks, "window": layers * (single + chunks), "capped": 0, "scaled": 0}[kind]
    if padding == "left" or dense:
        decode = more = 0
        if kind == "window" and not dense:  # (the window has left the padding behind, and no mask names it)
            more = context.calls.count("attend")
    assert context.calls.count("decode") == decode
    assert context.calls.count("attend") == (more if attend else 0)


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
    masks[1][0, 0, 0, 0] = False  # written again
    assert not hf_cache._remembered(masks[1], (3, 7, None), masks[1].all)
    with torch.inference_mode():
        mask = torch.ones(1, 1, 1, 7, dtype=torch.bool)
        assert hf_cache._mask_is_open(mask) and hf_cache._mask_is_causal(mask, 1, 7, None)


@pytest.mark.parametrize("window", [None, 2])
@pytest.mark.parametrize("softcap", [None, 3.0])
@pytest.mark.parametrize("given", ["none", "padding"])
def test_dense_history_without_a_mask_of_four_dimensions(window, softcap, given):
    """The attention function by itself, on a chunk on history: no mask, or what is padding as [batch, tokens]."""
    from types import SimpleNamespace

    from turboquant_pro_b200 import hf_cache

    gen = torch.Generator().manual_seed(5)
    context = _Context(2)
    cache = hf_cache.TurboQuantCache(n_layers=1, n_q_heads=4)
    cache._shared.ctx = context
    module = SimpleNamespace(layer_idx=0, is_causal=True, sliding_window=window, num_key_value_groups=2, training=False)
    new = lambda h, t: torch.randn(2, h, t, 16, generator=gen)  # noqa: E731
    n, pad = 0, None
    for t in (6, 1, 4):
        q, k, v = new(4, t), new(2, t), new(2, t)
        key, value = cache.layers[0].update(k, v)
        n += t
        if given == "padding":
            pad = torch.ones(2, n, dtype=torch.int64)
            pad[1, :2] = 0
        got, _ = hf_cache.turboquant_attention_forward(module, q, key, value, pad, scaling=0.25, softcap=softcap)
        kk, vv = (x.repeat_interleave(2, 2).transpose(1, 2).double() for x in context.kv[0])
        s = q.double() @ kk.transpose(2, 3) * 0.25
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p, j = torch.arange(n - t, n)[:, None], torch.arange(n)
        sees = ((j <= p) & (j > p - (window or n))).expand(2, 1, t, n)
        if pad is not None:
            sees = sees & (pad != 0)[:, None, None]
        want = (torch.softmax(s.masked_fill(~sees, -1e300), -1) @ vv).transpose(1, 2)
        rows = sees.any(-1)[:, 0]  # (a padding query's row is anything)
        assert torch.allclose(got[rows].double(), want[rows], rtol=1e-5, atol=1e-5)
    assert context.calls == ([] if window or softcap or given == "padding" else ["decode"])


@pytest.mark.parametrize("attend", [False, True])
@pytest.mark.parametrize("kind", ["plain", "window", "capped"])
def test_generate_with_a_padded_batch(monkeypatch, kind, attend):
    from transformers import DynamicCache

    from turboquant_pro_b200 import hf_cache

    model = _model(kind)
    ids = torch.randint(1, 97, (3, 14), generator=torch.Generator().manual_seed(2))
    mask = torch.ones_like(ids)
    mask[0, :5], mask[2, :13] = 0, 0
    args = dict(input_ids=ids, attention_mask=mask, max_new_tokens=8, do_sample=False, pad_token_id=0)
    model.config._attn_implementation = "eager"
    want = model.generate(**args, past_key_values=DynamicCache())
    context = _Context(3)
    monkeypatch.setattr(hf_cache._SharedContext, "get", lambda self, key: context)
    cache = hf_cache.enable_turboquant_cache(model, attend=attend)
    assert torch.equal(model.generate(**args, past_key_values=cache), want)
