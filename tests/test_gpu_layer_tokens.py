"""Rows and tokens of a cache layer chosen and moved (reorder_cache, batch_select_indices, batch_repeat_interleave, crop,
keep_tokens) against torch indexing of the same layer, byte for byte; prompts, drafts and accepted paths together."""

import copy
import math

import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import fused_attention, prompt_attention, tree_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16

pytestmark = pytest.mark.gpu

D = 128
KINDS = ["flat", "qjl", "split", "qjl and dense", "all dense", "all dense fp32"]


def make(kind, B=3, H=2, N=40, extra=9, seed=0):
    k, v = (kv_bf16((B, H, N + extra, D), seed=seed + i) for i in (0, 1))
    if kind.endswith("fp32"):
        k, v = k.float(), v.float()
    dense = "dense" in kind
    layer = PackedMSELayer(bits=4, use_qjl_keys=kind != "flat", num_outlier_channels=4 if kind == "split" else 0,
                           quantize_decode=not dense, reserve_tokens=20)
    layer.initialize_from_dense(k[:, :, :N], v[:, :, :N], force_dense=kind.startswith("all dense"))
    layer._lazy_update = True
    layer.update(k[:, :, N:], v[:, :, N:])
    return layer


def contents(layer):
    """The layer's tokens as bytes, [B, H, tokens, row] of each buffer: the packed ones, the dense ones."""
    def raw(t):
        t = (t.unsqueeze(-1) if t.dim() == 3 else t).contiguous()
        return t.view(torch.uint8).clone()

    packed = [] if layer._store is None else [raw(b[:, :, :layer._store.length]) for b in layer._store.buffers()]
    dense = [] if layer._dense_buf is None else [raw(b[:, :, :layer._dense_len]) for b in layer._dense_buf]
    return packed, dense


def same(layer, packed, dense):
    got = contents(layer)
    return all(len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b)) for a, b in zip(got, (packed, dense)))


@pytest.mark.parametrize("kind", KINDS)
def test_rows(cuda, kind):
    layer = make(kind)
    cache = Cache(layers=[layer])
    packed, dense = contents(layer)
    total = layer.get_seq_length()
    for call, rows in ((lambda: cache.reorder_cache(torch.tensor([2, 0, 0], device=cuda)), [2, 0, 0]),
                       (lambda: cache.batch_repeat_interleave(2), [2, 2, 0, 0, 0, 0]),
                       (lambda: cache.batch_select_indices(torch.tensor([5, 1])), [0, 2]),
                       (lambda: cache.batch_select_indices(torch.tensor([False, True], device=cuda)), [2])):
        call()
        assert same(layer, [x[rows] for x in packed], [x[rows] for x in dense])
        assert layer.get_seq_length() == total
    # the next token goes behind the others
    k, v = (kv_bf16((1, 2, 1, D), seed=i).to(layer.dtype) for i in (7, 8))
    layer.update(k, v)
    assert layer.get_seq_length() == total + 1
    if dense:
        assert torch.equal(layer._dense_keys[:, :, -1:], k)


@pytest.mark.parametrize("kind", KINDS)
def test_crop(cuda, kind):
    layer = make(kind)
    cache = Cache(layers=[layer])
    packed, dense = contents(layer)
    n_packed, n_dense = (x[0].shape[2] if x else 0 for x in (packed, dense))
    for call, left in ((0, 49), (-4, 45), (45, 45), (60, 45), (42, 42), (-12, 30), (-50, 0)):
        cache.crop(call)
        d = max(left - n_packed, 0)
        assert layer.get_seq_length() == left
        assert same(layer, [x[:, :, :left - d] for x in packed], [x[:, :, :d] for x in dense])


@pytest.mark.parametrize("kind", ["qjl", "split"])
def test_what_crop_leaves_behind_is_not_read(cuda, kind):
    layer, short = make(kind, N=64, extra=70), make(kind, N=64, extra=70)
    for n in layer._store.buffers():
        if n.dim() == 3:
            n[:, :, 70:] = float("nan")
    layer.crop(70)
    short.crop(70)
    for n in short._store.buffers():
        n[:, :, 70:] = 0
    q = torch.randn(3, 8, 5, D, device=cuda).bfloat16()
    assert torch.equal(fused_attention(q[:, :, :1], layer, 4), fused_attention(q[:, :, :1], short, 4))
    parents = torch.arange(-1, 4)
    assert torch.equal(tree_attention(q, layer, parents, 4), tree_attention(q, short, parents, 4))
    assert torch.equal(layer._decode_keys_full(), short._decode_keys_full())


def picked(x, first, index):
    """Tokens [0, first) and first + index of [B, H, tokens, row] bytes."""
    B, H, _, R = x.shape
    while index.dim() < 3:
        index = index[None] if index.dim() == 1 else index[:, None]
    index = index.expand(B, H, -1).to(x.device).long()
    ok = (index >= 0) & (index < x.shape[2] - first)
    rows = x.gather(2, torch.where(ok, first + index, 0)[..., None].expand(-1, -1, -1, R)).masked_fill(~ok[..., None], 0)
    return torch.cat((x[:, :, :first], rows), 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("index", [[0, 3, 5], [], [8, 0, 0, -1, 9], [[0, 1], [2, 3], [4, 8]], list(range(9))])
def test_kept_drafts(cuda, kind, index):
    layer = make(kind)
    packed, dense = contents(layer)
    index = torch.tensor(index, dtype=torch.int64)
    layer.keep_tokens(index, tokens=9)
    if dense:
        dense = [picked(x, x.shape[2] - 9, index) for x in dense]
    else:
        packed = [picked(x, x.shape[2] - 9, index) for x in packed]
    assert same(layer, packed, dense)
    assert layer.get_seq_length() == 40 + index.shape[-1]


@pytest.mark.parametrize("kind", ["qjl", "split", "all dense", "all dense fp32"])
@pytest.mark.parametrize("tokens,n,dims", [(None, 300, 3), (350, 257, 1), (390, 129, 2)])
def test_a_history_thinned_out(cuda, kind, tokens, n, dims):
    """More tokens than are moved in place; -1 names none, also behind tokens that stay."""
    layer = make(kind, B=2, N=380, extra=20)
    packed, dense = contents(layer)
    gen = torch.Generator().manual_seed(n)
    index = torch.randint(-1, tokens or 400, (2, 2)[:dims - 1] + (n,), generator=gen, dtype=torch.int32)
    layer.keep_tokens(index.to(cuda), tokens)
    first = 400 - (tokens or 400)
    assert same(layer, [picked(x, first, index) for x in packed], [picked(x, first, index) for x in dense])
    layer.update(*(kv_bf16((2, 2, 1, D), seed=i).to(layer.dtype) for i in (7, 8)))
    assert layer.get_seq_length() == first + n + 1


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_a_layer_cropped_to_nothing(cuda, kind):
    layer = make(kind)
    layer.crop(-49)
    layer.batch_repeat_interleave(2)
    layer.batch_select_indices(torch.tensor([0, 1]))
    k, v = (kv_bf16((2, 2, 1, D), seed=i).to(layer.dtype) for i in (7, 8))
    layer.update(k, v)
    assert layer.get_seq_length() == 1


def test_numbers_past_32_bits_name_nothing(cuda):
    layer = make("qjl")
    packed, _ = contents(layer)
    layer.reorder_cache(torch.tensor([2 ** 32 + 1, -2 ** 40, 2], device=cuda))
    layer.keep_tokens(torch.tensor([2 ** 32, 3], device=cuda), tokens=9)
    for got, x in zip(contents(layer)[0], packed):
        assert (got[:2] == 0).all() and (got[2, :, 40] == 0).all()
        assert torch.equal(got[2, :, :40], x[2, :, :40]) and torch.equal(got[2, :, 41], x[2, :, 43])


def test_refusals_and_empty_layers(cuda):
    layer = make("qjl and dense")
    with pytest.raises(ValueError, match="keep_tokens: 3 of the last 2"):
        layer.keep_tokens(torch.tensor([0, 1, 2]), tokens=2)
    with pytest.raises(ValueError, match="of 49 tokens"):
        layer.keep_tokens(torch.tensor([0]), tokens=50)
    with pytest.raises(ValueError, match="dense and those before packed"):
        layer.keep_tokens(torch.tensor([0]), tokens=10)
    with pytest.raises(ValueError, match="index must"):
        layer.keep_tokens(torch.tensor([[0], [1]]), tokens=9)
    for bad in (torch.tensor(3), torch.zeros(9, dtype=torch.bool), torch.zeros(3)):
        with pytest.raises(ValueError, match="index must be int"):
            layer.keep_tokens(bad, tokens=9)
    with pytest.raises(ValueError, match="rows must"):
        layer.reorder_cache(torch.tensor([0.0, 1.0, 2.0]))
    assert layer.get_seq_length() == 49
    empty = PackedMSELayer(bits=4)
    empty.reorder_cache(torch.tensor([0]))
    empty.batch_select_indices(torch.tensor([0]))
    empty.batch_repeat_interleave(3)
    empty.crop(-3)
    empty.keep_tokens(torch.empty(0, dtype=torch.int64))
    assert empty.get_seq_length() == 0


def rows64(layer):
    """What the layer's tokens decode to, in 64 bits."""
    from .test_gpu_tree import rows64 as decoded

    return decoded(layer)


def attend(q, k, v, mask):
    g = q.shape[1] // k.shape[1]
    x = q.double() @ k.double().repeat_interleave(g, 1).transpose(-1, -2) / math.sqrt(D)
    return torch.softmax(x.masked_fill(~mask, float("-inf")), -1) @ v.double().repeat_interleave(g, 1)


def test_prompt_drafts_and_accepted_path_together(cuda):
    """A padded batch's prompts, packed; a tree of drafts checked against them; its accepted path kept, twice over;
    and the layer then holds and answers what one that was given the accepted tokens alone does, bit for bit."""
    B, H, g, S = 2, 2, 4, 200
    starts = torch.tensor([0, 37], dtype=torch.int32, device=cuda)
    q, k, v = (torch.randn(B, S, h, D, generator=torch.Generator(device="cuda").manual_seed(i), device=cuda).bfloat16()
               .transpose(1, 2) for i, h in ((1, H * g), (2, H), (3, H)))
    out = prompt_attention(q, k, v, seq_starts=starts)
    pos = torch.arange(S, device=cuda)
    seen = (pos[None, :] <= pos[:, None])[None, None] & (pos[None, None, None, :] >= starts[:, None, None, None])
    ref = attend(q, k, v, seen | torch.eye(S, dtype=torch.bool, device=cuda))
    ref[1, :, :37] = 0.0
    # half a step of the output and of the weights (2^-8 each, of values up to 5), and their product
    assert ((out.double() - ref).abs() <= 2 ** -8 * (ref.abs() + 5)).all()

    layer, plain = (PackedMSELayer(bits=4, use_qjl_keys=True, quantize_decode=True, reserve_tokens=8) for _ in range(2))
    for x in (layer, plain):
        x._lazy_update = True
        x.initialize_from_dense(k, v)
    for turn in range(2):
        T, parents, path = 7, torch.tensor([-1, 0, 0, 1, 2, 4, -1]), [0, 2, 4, 5]
        dk, dv = (kv_bf16((B, H, T, D), seed=50 + 10 * turn + i) for i in (0, 1))
        dq = torch.randn(B, H * g, T, D, generator=torch.Generator(device="cuda").manual_seed(turn), device=cuda).bfloat16()
        layer.update(dk, dv)
        nodes = tree_attention(dq, layer, parents, g, seq_starts=starts)
        layer.keep_tokens(torch.tensor(path, device=cuda), tokens=T)
        for at in path:
            plain.update(dk[:, :, at:at + 1], dv[:, :, at:at + 1])
            kk, vv = rows64(plain)
            n = kk.shape[2]
            mask = torch.arange(n, device=cuda)[None, None, None, :] >= starts[:, None, None, None]
            ref = attend(dq[:, :, at:at + 1], kk, vv, mask)
            got = nodes[:, :, at:at + 1].double()
            assert ((got - ref).abs() <= 2e-3 * ref.abs().max() + 2 ** -8 * ref.abs()).all()
        assert same(layer, *contents(plain))
        one = torch.randn(B, H * g, 1, D, generator=torch.Generator(device="cuda").manual_seed(9), device=cuda).bfloat16()
        assert torch.equal(fused_attention(one, layer, g), fused_attention(one, plain, g))
    # beams forked and one of them dropped
    before = fused_attention(one, layer, g)
    layer.batch_repeat_interleave(2)
    layer.reorder_cache(torch.tensor([3, 0, 1, 2], device=cuda))
    layer.batch_select_indices(torch.tensor([0, 2], device=cuda))
    assert torch.equal(fused_attention(one[[1, 0]], layer, g), before[[1, 0]])


def test_a_copied_layer_stays_as_it_was(cuda):
    """reorder_cache and a thinned history make new buffers: a shallow copy of the layer and its store goes on with the old."""
    layer = make("qjl", N=300)
    other = copy.copy(layer)
    other._store = copy.copy(layer._store)
    packed, dense = contents(layer)
    layer.reorder_cache(torch.tensor([1, 1, 1]))
    layer.keep_tokens(torch.arange(290))
    assert same(other, packed, dense)


def test_beam_search_of_a_model(cuda):
    """HF's beam search reorders the layers; generated tokens are kept dense here, so it ends with the same beams."""
    from ._tiny_model import tiny_llama

    model = tiny_llama(device=cuda, dtype=torch.bfloat16)
    ids = torch.randint(0, 94, (2, 30), generator=torch.Generator().manual_seed(0)).to(cuda)
    ref = model.generate(ids, num_beams=3, num_return_sequences=3, max_new_tokens=8, do_sample=False)
    calls = []

    class Layer(PackedMSELayer):
        def reorder_cache(self, beam_idx):
            calls.append(beam_idx.tolist())
            super().reorder_cache(beam_idx)

    cache = Cache(layers=[Layer(bits=4) for _ in range(2)])
    got = model.generate(ids, num_beams=3, num_return_sequences=3, max_new_tokens=8, do_sample=False, past_key_values=cache)
    assert torch.equal(got, ref)
    assert calls and any(c != list(range(6)) for c in calls)


@pytest.mark.parametrize("kind", ["all dense", "qjl and dense"])
def test_trees_over_layers_without_packed_tokens(cuda, kind):
    layer = make(kind, B=1, extra=12)
    if kind != "all dense":  # every packed token gone, the dense ones left
        layer._store.length = 0
    k, v = layer._dense_keys, layer._dense_values
    n = k.shape[2]
    q = torch.randn(1, 8, 5, D, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda).bfloat16()
    parents = torch.tensor([-1, 0, 0, 2, -1])
    sees = torch.eye(5, dtype=torch.bool)
    for i, p in ((1, 0), (2, 0), (3, 2), (3, 0)):
        sees[i, p] = True
    mask = torch.cat((torch.ones(5, n - 5, dtype=torch.bool), sees), 1).to(cuda)
    ref = attend(q, k, v, mask)
    got = tree_attention(q, layer, parents, 4).double()
    assert ((got - ref).abs() <= 2e-3 * ref.abs().max() + 2 ** -8 * ref.abs()).all()
