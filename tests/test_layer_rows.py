"""Row numbers that the cache layers of transformers take or refuse: negative ones, ones past the batch, masks of another length."""

import pytest
import torch
from transformers.cache_utils import Cache, DynamicLayer

from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16


def dense_layer(device="cpu", B=3):
    k, v = (torch.randn(B, 2, 5, 128, generator=torch.Generator().manual_seed(i)).bfloat16().to(device) for i in (0, 1))
    layer, plain = PackedMSELayer(bits=4), DynamicLayer()
    layer.initialize_from_dense(k, v, force_dense=True)
    plain.update(k, v)
    return layer, plain


@pytest.mark.parametrize("call,rows", [("reorder_cache", [0, 3]), ("reorder_cache", [-1, 0]), ("batch_select_indices", [3]),
                                       ("batch_select_indices", [0, -4]), ("batch_select_indices", [2 ** 32]),
                                       ("batch_select_indices", [True, False]),
                                       ("batch_select_indices", [True, False, True, True])])
def test_rows_that_there_are_not_are_refused(call, rows):
    """Numbers on the host: transformers refuses the same."""
    for layer in dense_layer():
        with pytest.raises(IndexError):
            getattr(layer, call)(torch.tensor(rows))
        assert layer.get_seq_length() == 5
    layer = PackedMSELayer(bits=4)  # holds nothing
    getattr(layer, call)(torch.tensor(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("rows", [[-1], [0, -2, -3], [2, -1], [True, False, True], [False] * 3])
def test_rows_counted_from_the_last(cuda, where, rows):
    layer, plain = dense_layer(cuda)
    for x in (layer, plain):
        x.batch_select_indices(torch.tensor(rows, device=where))
    assert torch.equal(layer._dense_keys, plain.keys) and torch.equal(layer._dense_values, plain.values)
    packed = PackedMSELayer(bits=4, use_qjl_keys=True)
    k, v = (kv_bf16((3, 2, 40, 128), seed=i) for i in (0, 1))
    packed.initialize_from_dense(k, v)
    before = packed._decode_keys_full()
    Cache(layers=[packed]).batch_select_indices(torch.tensor(rows, device=where))
    assert torch.equal(packed._decode_keys_full(), before[torch.tensor(rows)])


@pytest.mark.gpu
def test_rows_past_the_batch_on_the_device(cuda):
    """They are known on the device only: zeros, as reorder_cache gives."""
    layer, plain = dense_layer(cuda)
    keys = plain.keys.clone()
    layer.batch_select_indices(torch.tensor([3, 1, -4, -1], device=cuda))
    assert (layer._dense_keys[[0, 2]] == 0).all() and torch.equal(layer._dense_keys[[1, 3]], keys[[1, 2]])
