"""The fp16 codebook of a layer's values is there before its first attention, which may be a captured one."""

import dataclasses

import pytest
import torch

from turboquant.runtime import kernels as K
from turboquant.runtime import tree_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.params import layer_codecs
from turboquant.runtime.synthetic import kv_bf16


@pytest.mark.parametrize("bits,qjl", [(1, False), (2, True), (3, False), (4, True)])
def test_it_comes_with_the_codec(bits, qjl):
    value = layer_codecs(128, bits, 77, qjl, "cpu").value
    want = torch.from_numpy(K.value_codebook_f16(value.centers.numpy(), bits))
    assert torch.equal(value.attn_centers, want) and K.attention_value_centers(value) is value.attn_centers
    alone = K.CodecParams(value.bits, value.rotation, value.centers, value.boundaries)
    assert torch.equal(K.attention_value_centers(alone), want)


@pytest.mark.gpu
def test_a_layers_first_attention_captured(cuda):
    layer = PackedMSELayer(bits=3, seed=771, use_qjl_keys=True, quantize_decode=True)  # no other test's codecs
    layer.initialize_from_dense(*(kv_bf16((1, 2, 90, 128), seed=i) for i in (0, 1)))
    q = torch.randn(1, 8, 4, 128, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda).bfloat16()
    parents = torch.tensor([-1, 0, 1, 0], dtype=torch.int32, device=cuda)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tree_attention(q, layer, parents)
    want = tree_attention(q, layer, parents)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("values", [False, True])
@pytest.mark.parametrize("bits", [1, 2, 3, 4])
def test_scaled_codebooks(bits, values):
    """The same products of rotated queries and centroids, from centroids that fp16 holds better."""
    c = layer_codecs(128, bits, 0, False, "cpu").value
    rotation, centers = K.scaled_codec(c, values)
    assert K.scaled_codec(c, values)[0] is rotation and rotation.dtype == centers.dtype == torch.float32
    assert torch.equal(centers, centers.half().float())
    at = torch.argmax(c.rotation.abs())
    s = (c.rotation.flatten()[at].double() / rotation.flatten()[at]).item()
    assert 1.0 <= s < 2.0 + 1e-6 and (rotation * s - c.rotation).abs().max() <= 2.0 ** -23
    x = c.centers.double()
    middle = (x[1:] + x[:-1]) / 2
    n = 1 << 16
    grid = (torch.arange(n).double() + 0.5) / n * 2 - 1
    weight = (1 - grid ** 2) ** 62.5
    share = torch.zeros(1 << bits).double().index_add_(0, torch.bucketize(grid, middle), weight) / weight.sum()
    size = lambda e: (share * e ** 2).sum().sqrt() / (share * x ** 2).sum().sqrt()  # noqa: E731
    err = centers.double() / s - x
    assert size(err) <= 0.8 * size(x.half().double() - x)
    if values:
        assert abs((share * err).sum()) <= 1e-6 * (share * x ** 2).sum().sqrt()


def test_scaled_codebooks_go_with_their_codec():
    """A codec with another codebook does not keep the first one's; codebooks past fp16's range, and of one number, have one."""
    c = layer_codecs(128, 2, 0, False, "cpu").value
    K.scaled_codec(c, True)
    other = dataclasses.replace(c, centers=c.centers * 0.7)
    assert other.attn_values is None and not torch.equal(K.scaled_codec(other, True)[1], K.scaled_codec(c, True)[1])
    exact = dataclasses.replace(c, centers=torch.tensor([-0.5, -0.25, 0.25, 0.5]))
    assert torch.equal(K.scaled_codec(exact, False)[1], exact.centers) and torch.equal(K.scaled_codec(exact, False)[0], c.rotation)
    large = dataclasses.replace(c, centers=torch.tensor([-6e4, -1.0, 1.0, 6e4]))
    assert torch.isfinite(K.scaled_codec(large, True)[1]).all()


def test_codebooks_are_searched_for_once(monkeypatch):
    """Codecs made by hand of the same centroids; each keeps a tensor of its own."""
    c = layer_codecs(128, 4, 0, False, "cpu").value
    K._value_codebook.cache_clear()
    searched, search = [], K.value_codebook_f16
    monkeypatch.setattr(K, "value_codebook_f16", lambda *a: searched.append(a) or search(*a))
    codecs = [K.CodecParams(4, c.rotation, c.centers.clone(), c.boundaries) for _ in range(3)]
    made = [K.attention_value_centers(x) for x in codecs]
    assert len(searched) == 1 and all(torch.equal(m, c.attn_centers) for m in made)
    made[0].zero_()
    assert torch.equal(K.attention_value_centers(K.CodecParams(4, c.rotation, c.centers, c.boundaries)), made[1])
    K.attention_value_centers(dataclasses.replace(codecs[0], centers=c.centers * 0.9, attn_centers=None))
    assert len(searched) == 2
