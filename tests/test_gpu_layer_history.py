"""Layers emptied by crop or keep_tokens and filled again, on the GPU: their attention against a layer that never held
anything else, with generated tokens packed and dense, one channel group and two, wired and not."""

import math

import pytest
import torch

from turboquant.runtime import fused_attention, tree_attention
from turboquant.runtime.attention import turboquant_attention_forward, turboquant_prompt_forward
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16

pytestmark = pytest.mark.gpu

D, B, H, G, S = 128, 2, 2, 4, 37
FORWARDS = [turboquant_attention_forward, turboquant_prompt_forward]


class Module(torch.nn.Module):
    is_causal, num_key_value_groups = True, G


def make(k, v, split, packed, wired=True):
    layer = PackedMSELayer(bits=4, use_qjl_keys=True, num_outlier_channels=4 if split else 0, quantize_decode=packed)
    layer.initialize_from_dense(k, v)
    layer._lazy_update = wired
    return layer


def emptied(layer, how):
    if how == "crop":
        layer.crop(-10 ** 6)
    else:
        for n in (layer._dense_len, layer.packed_seq_length()):  # the dense tokens first, then the packed ones
            layer.keep_tokens(torch.empty(0, dtype=torch.int64), n)
    assert layer.get_seq_length() == 0
    return layer


def attend(q, k, v, mask):
    x = q.double() @ k.double().repeat_interleave(G, 1).transpose(-1, -2) / math.sqrt(D)
    return torch.softmax(x.masked_fill(~mask, float("-inf")), -1) @ v.double().repeat_interleave(G, 1)


def check(got, ref):
    """bf16: half a step of the output and of the weights (2^-8 each), the weights' of the largest value."""
    assert ((got.double() - ref).abs() <= 2 ** -8 * (ref.abs() + ref.abs().max()) + 2e-3 * ref.abs().max()).all()


@pytest.mark.parametrize("forward", FORWARDS)
@pytest.mark.parametrize("how", ["crop", "keep"])
@pytest.mark.parametrize("split", [False, True])
def test_packed_again(cuda, forward, how, split):
    """The refilled prompt is causal over its exact keys; the steps behind it are those of a layer that was built from it."""
    k, v = (kv_bf16((B, H, S + 2, D), seed=i) for i in (0, 1))
    q = torch.randn(B, H * G, S + 2, D, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda).bfloat16()
    m = Module()
    # (a split layer keeps the channels that its first prompt chose: it is emptied of the same prompt)
    layer = m._tq_cache_layer = emptied(make(k[:, :, :S], v[:, :, :S], split, True), how)
    plain = make(k[:, :, :S], v[:, :, :S], split, True)
    layer.update(k[:, :, :S], v[:, :, :S])
    got, _ = forward(m, q[:, :, :S], k[:, :, :S], v[:, :, :S], None, scaling=D ** -0.5)
    check(got.transpose(1, 2), attend(q[:, :, :S], k[:, :, :S], v[:, :, :S], torch.ones(S, S, device=cuda).tril().bool()))
    for t in (S, S + 1):
        one = slice(t, t + 1)
        for x in (layer, plain):
            x.update(k[:, :, one], v[:, :, one])
        got, _ = forward(m, q[:, :, one], k[:, :, one], v[:, :, one], None, scaling=D ** -0.5)
        assert torch.equal(got.transpose(1, 2), fused_attention(q[:, :, one], plain, G))
    assert torch.equal(layer._decode_keys_full(), plain._decode_keys_full())


@pytest.mark.parametrize("forward", FORWARDS)
@pytest.mark.parametrize("how", ["crop", "keep"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense_again(cuda, forward, how, dtype):
    """Tokens kept dense: prompt, steps and a chunk behind it attend to all of them."""
    k, v = (kv_bf16((B, H, S + 5, D), seed=i).to(dtype) for i in (0, 1))
    q = torch.randn(B, H * G, S + 5, D, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda).to(dtype)
    m = Module()
    layer = m._tq_cache_layer = make(k[:, :, :9], v[:, :, :9], False, False)
    layer.update(k[:, :, :3], v[:, :, :3])
    emptied(layer, how)
    for a, b in ((0, S), (S, S + 1), (S + 1, S + 4), (S + 4, S + 5)):
        layer.update(k[:, :, a:b], v[:, :, a:b])
        got, _ = forward(m, q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], None, scaling=D ** -0.5)
        check(got.transpose(1, 2), attend(q[:, :, a:b], k[:, :, :b], v[:, :, :b],
                                          torch.ones(b - a, b, device=cuda).tril(a).bool()))
    got = tree_attention(q[:, :, S + 2:], layer, torch.tensor([-1, 0, 1]), G)
    check(got, attend(q[:, :, S + 2:], k, v, torch.ones(3, S + 5, device=cuda).tril(S + 2).bool()))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("split", [False, True])
def test_without_the_backend(cuda, packed, split):
    """A layer that hands its history over goes on from an empty one."""
    k, v = (kv_bf16((B, H, S + 1, D), seed=i) for i in (0, 1))
    layer = emptied(make(k[:, :, :S], v[:, :, :S], split, packed, wired=False), "crop")
    assert layer._decode_keys_full().shape == (B, H, 0, D)
    got = layer.update(k[:, :, :S], v[:, :, :S])
    assert torch.equal(got[0], k[:, :, :S]) and torch.equal(got[1], v[:, :, :S])
    keys, values = layer.update(k[:, :, S:], v[:, :, S:])
    assert keys.shape == values.shape == (B, H, S + 1, D) and torch.equal(keys[:, :, S:], k[:, :, S:])
    if not packed:
        assert torch.equal(keys, k) and torch.equal(values, v)
