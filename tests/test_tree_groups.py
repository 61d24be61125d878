"""How many query heads share a KV head of a tree: from the layer's shapes, on every route."""

import math

import pytest
import torch

from turboquant.runtime import tree_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16


def attend(q, k, v, mask):
    g = q.shape[1] // k.shape[1]
    x = q.double() @ k.double().repeat_interleave(g, 1).transpose(-1, -2) / math.sqrt(128)
    return torch.softmax(x.masked_fill(~mask, -math.inf), -1) @ v.double().repeat_interleave(g, 1)


def test_dense_rows_on_the_cpu():
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 2, 9, 128, generator=gen) for _ in range(2))
    q = torch.randn(2, 8, 3, 128, generator=gen)
    layer = PackedMSELayer(bits=4)
    layer.initialize_from_dense(k, v, force_dense=True)
    parents = torch.tensor([-1, 0, 1])
    want = attend(q, k, v, torch.ones(3, 9).tril(6).bool())
    for groups in ((), (None,), (4,)):
        assert (tree_attention(q, layer, parents, *groups).double() - want).abs().max() <= 1e-5 * want.abs().max()
    for groups in (1, 2, 8):
        with pytest.raises(ValueError, match="2 KV heads"):
            tree_attention(q, layer, parents, groups)
    with pytest.raises(ValueError, match="2 KV heads"):
        tree_attention(q[:, :7], layer, parents)
    with pytest.raises(ValueError, match="2 rows"):
        tree_attention(q[:1], layer, parents)
    assert tree_attention(q[:, :, :0], PackedMSELayer(bits=4), parents[:0]).shape == (2, 8, 0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["packed", "split", "more nodes than the kernel takes", "dense", "fp32 rows"])
def test_every_route_without_the_number(cuda, route):
    T, N = 70 if route.startswith("more") else 5, 100
    k, v = (kv_bf16((2, 2, N + T, 128), seed=i) for i in (0, 1))
    if route == "fp32 rows":
        k, v = k.float(), v.float()
    dense = route in ("dense", "fp32 rows")
    layer = PackedMSELayer(bits=4, use_qjl_keys=True, num_outlier_channels=4 if route == "split" else 0,
                           quantize_decode=not dense)
    layer.initialize_from_dense(k[:, :, :N], v[:, :, :N])
    layer._lazy_update = True
    layer.update(k[:, :, N:], v[:, :, N:])
    q = torch.randn(2, 8, T, 128, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda).bfloat16()
    parents = torch.arange(-1, T - 1)
    assert torch.equal(tree_attention(q, layer, parents), tree_attention(q, layer, parents, 4))
    with pytest.raises(ValueError, match="n_kv_groups 1"):
        tree_attention(q, layer, parents, 1)
