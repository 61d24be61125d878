"""Attention over layers that were emptied and filled again, or filled while the attention backend was wired: every token
held is attended to.  Tokens kept dense, on the CPU; packed ones are in test_gpu_layer_history.py."""

import math

import pytest
import torch
from transformers.cache_utils import Cache, DynamicCache

from turboquant.adapters.transformers import disable_turboquant_attention, enable_turboquant_attention
from turboquant.runtime.attention import turboquant_attention_forward, turboquant_prompt_forward
from turboquant.runtime.packed_qmse_cache import PackedMSELayer

from ._tiny_model import tiny_llama

FORWARDS = [turboquant_attention_forward, turboquant_prompt_forward]


@pytest.mark.parametrize("name", ["turboquant", "turboquant_prompt"])
@pytest.mark.parametrize("cropped", [False, True])
@pytest.mark.parametrize("padded", [False, True])
def test_a_model_goes_on_from_an_emptied_cache(name, cropped, padded):
    """A prompt, two single tokens and a chunk of three, with the same results as a dense cache: all fp32, the same sums in
    another order (2^-24 of terms that cancel to a tenth of their size, over 400 of them and four layers' worth)."""
    model = tiny_llama()
    gen = torch.Generator().manual_seed(0)
    old, ids = (torch.randint(0, 94, (2, n), generator=gen) for n in (7, 16))
    mask = torch.ones(2, 16, dtype=torch.long)
    if padded:
        mask[1, :4] = 0
    cache, ref = Cache(layers=[PackedMSELayer(bits=4) for _ in range(2)]), DynamicCache()
    parts = [(0, 11), (11, 12), (12, 13), (13, 16)]
    kw = lambda a, b: dict(input_ids=ids[:, a:b], attention_mask=mask[:, :b] if padded else None)  # noqa: E731
    with torch.no_grad():
        want = [model(**kw(a, b), past_key_values=ref).logits for a, b in parts]
        before = enable_turboquant_attention(model, cache)
        model.config._attn_implementation = name
        if cropped:
            model(old, past_key_values=cache)
            cache.crop(-100)
        assert cache.get_seq_length() == 0
        got = [model(**kw(a, b), past_key_values=cache).logits for a, b in parts]
        disable_turboquant_attention(model, cache, before)
    live = mask.bool()
    for (a, b), x, y in zip(parts, got, want):
        x, y = x[live[:, a:b]], y[live[:, a:b]]
        assert (x - y).abs().max() <= 1e-4 * y.abs().max()


@pytest.mark.parametrize("forward", FORWARDS)
def test_rows_behind_dense_tokens_are_causal(forward):
    """No mask: a row attends to the tokens up to its own, of what the layer holds and not of what the call hands over."""
    class Module(torch.nn.Module):
        is_causal, num_key_value_groups = True, 4

    m, layer = Module(), PackedMSELayer(bits=4)
    m._tq_cache_layer, layer._lazy_update = layer, True
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 2, 9, 128, generator=gen) for _ in range(2))
    q = torch.randn(2, 8, 9, 128, generator=gen)
    x = q.double() @ k.double().repeat_interleave(4, 1).transpose(-1, -2) / math.sqrt(128)
    x = x.masked_fill(torch.ones(9, 9, dtype=torch.bool).triu(1), float("-inf"))
    want = torch.softmax(x, -1) @ v.double().repeat_interleave(4, 1)
    at = 0
    for n in (1, 3, 1, 3, 1):
        new = slice(at, at + n)
        layer.update(k[:, :, new], v[:, :, new])
        got, _ = forward(m, q[:, :, new], k[:, :, new], v[:, :, new], None, scaling=1 / math.sqrt(128))
        # fp32 sums of 128 products and 9 weights of logits below 8: a few 2^-24 of each
        assert (got.transpose(1, 2).double() - want[:, :, new]).abs().max() <= 2e-5
        at += n
