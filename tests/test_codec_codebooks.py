"""The fp16 codebook of a layer's values is there before its first attention, which may be a captured one."""

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
