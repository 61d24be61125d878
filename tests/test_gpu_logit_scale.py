"""The attention interfaces' ``scaling``: the steps over packed and shared layers are scaled as the prompt before them is."""

import math

import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import share_prefix
from turboquant.runtime.attention import chunked_turboquant_attention, turboquant_attention_forward, turboquant_prompt_forward
from turboquant.runtime.packed_qmse_cache import PackedMSELayer

from ._packed import D, attend64, check, make_layer, randn, rows64

FORWARDS = [turboquant_attention_forward, turboquant_prompt_forward]


def module(layer):
    m = torch.nn.Module()
    m._tq_cache_layer, m.num_key_value_groups, m.is_causal = layer, 4, True
    return m


def tokens(layer):
    k, v = rows64(layer)
    if layer._dense_len:
        k, v = torch.cat((k, layer._dense_keys.double()), 2), torch.cat((v, layer._dense_values.double()), 2)
    return k, v


@pytest.mark.gpu
@pytest.mark.parametrize("forward", FORWARDS)
@pytest.mark.parametrize("dense", [0, 30])
@pytest.mark.parametrize("split", [0, 4])
def test_steps_over_packed_layers(cuda, forward, dense, split):
    layer = make_layer(2, 2, 300, 4, True, seed=1, dense=dense, num_outlier_channels=split)
    m, q = module(layer), randn((2, 8, 1, D), 3)
    plain, _ = forward(m, q, None, None, None)
    assert torch.equal(forward(m, q, None, None, None, scaling=D ** -0.5)[0], plain)
    got, _ = forward(m, q, None, None, None, scaling=0.031)
    if split:
        assert not torch.equal(got, plain)
        q = (q.float() * (0.031 * math.sqrt(D))).to(q.dtype)
        check(got, forward(m, q, None, None, None)[0].double(), 2e-2)  # the scale rounded into bf16 queries: 2^-9 of logits up to 6
    else:
        check(got[:, 0], attend64(q[:, :, 0], *tokens(layer), scale=0.031)[0])
    layer.attend_blocks(3, recent=1)
    if not split:
        chosen, _ = forward(m, q, None, None, None, scaling=1e-6)  # next to the mean of the values attended to
        assert torch.isfinite(chosen).all() and not torch.equal(chosen, forward(m, q, None, None, None)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("forward", FORWARDS)
@pytest.mark.parametrize("dense", [False, True])
def test_steps_over_shared_layers(cuda, forward, dense):
    prompt, copied = (make_layer(2, 2, 100, 4, True, seed=1) for _ in range(2))
    prompt.quantize_decode = copied.quantize_decode = not dense
    layer = share_prefix(Cache(layers=[prompt]), 3).layers[0]
    copied.batch_repeat_interleave(3)
    layer._lazy_update = True
    k, v = randn((6, 2, 7, D), 5), randn((6, 2, 7, D), 6)
    for x in (layer, copied):
        x.update(k, v)
    m = module(layer)
    k, v = tokens(copied)
    for Sq, tol in ((1, 2e-3), (3, 2e-2)):  # several tokens: bf16 rows and weights
        q = randn((6, 8, Sq, D), 7)
        assert torch.equal(forward(m, q, None, None, None, scaling=D ** -0.5)[0], forward(m, q, None, None, None)[0])
        got, _ = forward(m, q, None, None, None, scaling=0.031)
        for i in range(Sq):
            n = k.shape[2] - Sq + i + 1
            check(got[:, i], attend64(q[:, :, i], k[:, :, :n], v[:, :, :n], scale=0.031)[0], tol)
    hole = torch.ones(6, k.shape[2], dtype=torch.bool, device="cuda")
    hole[1, 40:60] = False
    got, _ = forward(m, q[:, :, :1], None, None, hole, scaling=0.031)
    check(got[:, 0], attend64(q[:, :, 0], k, v, hole[:, None], scale=0.031)[0], 2e-2)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            forward(m, q[:, :, :1], None, None, None, scaling=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 3])
def test_a_mask_with_a_hole(cuda, Sq):
    layer = make_layer(2, 2, 300, 4, True, seed=1)
    m, q = module(layer), randn((2, 8, Sq, D), 3)
    mask = torch.ones(2, 1, Sq, 300, dtype=torch.bool, device="cuda")
    mask[:, :, :, 100:120] = False
    got, _ = turboquant_attention_forward(m, q, None, None, mask, scaling=0.031)
    for i in range(Sq):
        check(got[:, i], attend64(q[:, :, i], *rows64(layer), mask[:, :, i], scale=0.031)[0], 2e-2)  # bf16 rows and weights


def test_rows_decoded_on_the_host():
    q, k, v = (torch.randn(1, h, 9, D, generator=torch.Generator().manual_seed(h)) for h in (4, 2, 2))
    empty = PackedMSELayer(bits=4)
    got = chunked_turboquant_attention(q, empty, k, v, 2, scale=0.3)
    p = torch.softmax(q.double() @ k.double().repeat_interleave(2, 1).transpose(-1, -2) * 0.3, -1)
    want = p @ v.double().repeat_interleave(2, 1)
    assert (got - want).abs().max() <= 1e-5
    again = chunked_turboquant_attention(q, empty, k, v, 2)
    assert torch.equal(again, chunked_turboquant_attention(q, empty, k, v, 2, scale=1 / math.sqrt(D)))
