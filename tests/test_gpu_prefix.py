"""Attention behind shared prompts (tq_prefix_attention) against the fp64 formula: every bit width, types, tile and block edges,
prompts with different numbers of sequences, padded prompts, rows without tokens, norms at the ends of their range, strides, streams
and captured calls; the shared layer beside a layer that holds the prompt once for each sequence, and a model on both."""

import copy
import math

import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import SharedPrefixLayer, share_prefix, shared_prefix_attention
from turboquant.runtime import kernels as K
from turboquant.runtime.packed_qmse_cache import build_packed_mse_cache
from turboquant.runtime.synthetic import kv_bf16

from ._packed import BITS, D, TOL, arrays, attend64, check, codec, i32, make_layer, randn, rows64
from ._tiny_model import tiny_llama

pytestmark = pytest.mark.gpu


def reference(q, prompts, own, counts, starts=None, lens=None, own_lens=None, scale=None):
    """In 64 bits, sequence by sequence."""
    pk, pv = rows64(prompts)
    ok, ov = rows64(own) if own is not None else (pk[:, :, :0], pv[:, :, :0])
    outs, b = [], 0
    for p, n in enumerate(counts):
        lo, hi = starts[p] if starts else 0, lens[p] if lens else pk.shape[2]
        lo, hi = min(max(lo, 0), pk.shape[2]), min(max(hi, 0), pk.shape[2])
        for _ in range(n):
            m = ok.shape[2] if own_lens is None else min(max(own_lens[b], 0), ok.shape[2])
            k = torch.cat((pk[p:p + 1, :, min(lo, hi):hi], ok[b:b + 1, :, :m] if own is not None else ok[:1]), 2)
            v = torch.cat((pv[p:p + 1, :, min(lo, hi):hi], ov[b:b + 1, :, :m] if own is not None else ov[:1]), 2)
            outs.append(attend64(q[b:b + 1], k, v, scale=scale))
            b += 1
    return torch.cat([o for o, _ in outs]), torch.cat([e for _, e in outs])


def setup(counts, H, g, N, M, bits=4, qjl=True, dtype=torch.bfloat16, seed=0):
    prompts = make_layer(len(counts), H, N, bits, qjl, seed=seed)
    own = make_layer(sum(counts), H, M, bits, qjl, seed=seed + 2) if M else None
    q = randn((sum(counts), H * g, D), seed + 9, dtype)
    kw = dict(n_prefix=N, n_own=M, **codec(prompts))
    if len(set(counts)) > 1:
        kw["cu_rows"] = i32([sum(counts[:i]) for i in range(len(counts) + 1)])
    return prompts, own, q, kw


def call(prompts, own, q, kw):
    return K.prefix_attention(q, arrays(prompts), None if own is None else arrays(own), **kw)


@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("counts,H,g,N,M", [((3, 3), 2, 4, 100, 33), ((20, 1), 1, 7, 517, 5)])
def test_every_bit_width(cuda, bits, qjl, counts, H, g, N, M):
    prompts, own, q, kw = setup(counts, H, g, N, M, bits, qjl)
    got = call(prompts, own, q, kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    check(got, reference(q, prompts, own, counts)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("counts,H,g,N,M", [((1,), 1, 1, 1, 0), ((1,), 2, 4, 1, 1), ((2,), 2, 4, 31, 32), ((8,), 1, 4, 32, 33),
                                            ((9,), 1, 4, 33, 1), ((5, 5, 5), 2, 8, 65, 64), ((64,), 1, 1, 300, 40),
                                            ((70,), 1, 1, 40, 3), ((3,), 1, 64, 129, 31), ((2, 2), 1, 33, 64, 2),
                                            ((1, 7, 0, 2), 2, 5, 700, 100), ((0, 0, 4), 1, 12, 90, 17), ((33,), 2, 2, 2000, 0)])
def test_shapes_and_types(cuda, dtype, counts, H, g, N, M):
    prompts, own, q, kw = setup(counts, H, g, N, M, dtype=dtype, seed=3)
    got, f32, lse = call(prompts, own, q, dict(kw, want_f32=True, want_lse=True))
    ref, ref_lse = reference(q, prompts, own, counts)
    assert got.dtype == dtype
    check(got, ref)
    check(f32, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3


@pytest.mark.parametrize("max_rows", [None, 1, 3, 40])
def test_the_most_rows_are_a_hint(cuda, max_rows):
    counts = (12, 3, 25)
    prompts, own, q, kw = setup(counts, 2, 4, 400, 20, seed=5)
    check(call(prompts, own, q, dict(kw, max_rows=max_rows)), reference(q, prompts, own, counts)[0])


def test_a_long_prompt_and_many_splits(cuda):
    prompts, own, q, kw = setup((6,), 2, 4, 33000, 70, seed=7)
    check(call(prompts, own, q, kw), reference(q, prompts, own, (6,))[0])


@pytest.mark.parametrize("counts", [(4, 4, 4), (2, 9, 1)])
def test_ranges(cuda, counts):
    prompts, own, q, kw = setup(counts, 2, 3, 600, 90, 3, False, seed=9)
    starts, lens = [0, 100, 590], [600, 111, 590]
    mine = [0, 90, 1, 33, 64, 17, 0, 90, 32, 31, 5, 500]
    got, lse = call(prompts, own, q, dict(kw, prefix_starts=i32(starts), prefix_lens=i32(lens), own_lens=i32(mine), want_lse=True))
    ref, ref_lse = reference(q, prompts, own, counts, starts, lens, mine)
    check(got, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3


def test_rows_without_tokens_are_zero(cuda):
    prompts, own, q, kw = setup((2, 2), 2, 4, 64, 8, seed=11)
    got, lse = call(prompts, own, q, dict(kw, prefix_lens=i32([0, 40]), prefix_starts=i32([0, 50]), own_lens=i32([0, 3, -5, 0]),
                                          want_lse=True))
    ref, ref_lse = reference(q, prompts, own, (2, 2), [0, 50], [0, 40], [0, 3, -5, 0])
    assert (got[[0, 2, 3]] == 0).all() and (lse[[0, 2, 3]] == -math.inf).all()
    check(got[1], ref[1])
    got = K.prefix_attention(q, arrays(prompts), n_prefix=0, **codec(prompts))
    assert (got == 0).all()


def test_offsets_that_are_none(cuda):
    """Descending offsets and offsets past the batch are empty prompts and ends of the batch; every sequence has a prompt."""
    prompts, own, q, kw = setup((3, 3, 3), 1, 4, 50, 4, seed=13)
    got = call(prompts, own, q, dict(kw, cu_rows=i32([5, 4, 2, 100])))  # prompts 0: [0, 4), 1: none, 2: [4, 9)
    check(got, reference(q, prompts, own, (4, 0, 5))[0])
    got = call(prompts, own, q, dict(kw, cu_rows=i32([0, -7, 40, 3])))  # prompts 0: none, 1: all
    check(got, reference(q, prompts, own, (0, 9, 0))[0])


def test_many_prompts(cuda):
    """More items than a wave has lanes, and more prompts."""
    counts = tuple((i * 7) % 4 for i in range(90))
    prompts, own, q, kw = setup(counts, 1, 4, 40, 3, seed=15)
    check(call(prompts, own, q, kw), reference(q, prompts, own, counts)[0])
    check(call(prompts, own, q, dict(kw, max_rows=3, own_lens=i32([b % 4 for b in range(sum(counts))]))),
          reference(q, prompts, own, counts, own_lens=[b % 4 for b in range(sum(counts))])[0])


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 3e4])
def test_norms_at_the_ends_of_their_range(cuda, size):
    prompts, own, q, kw = setup((3,), 2, 4, 400, 40, seed=17)
    for layer, n in ((prompts, 400), (own, 40)):
        ramp = torch.linspace(1e-3 if size > 1e-3 else 1.0, 2.0, n, device="cuda")
        layer._store.vn[:, :, :n] = (size * ramp).half()
    got, f32 = call(prompts, own, q, dict(kw, want_f32=True))
    ref = reference(q, prompts, own, (3,))[0]
    check(f32, ref)


def test_what_is_not_attended_to_may_be_anything(cuda):
    prompts, own, q, kw = setup((2, 5), 2, 4, 130, 40, seed=19)
    limits = dict(prefix_starts=i32([7, 0]), prefix_lens=i32([129, 100]), own_lens=i32([0, 3, 40, 1, 33, 31, 32]))
    want = call(prompts, own, q, dict(kw, **limits))
    for layer, lo, hi in ((prompts, [7, 0], [129, 100]), (own, [0] * 7, [0, 3, 40, 1, 33, 31, 32])):
        for b in range(len(lo)):
            for t in (layer._store.kn, layer._store.kr, layer._store.vn):
                t[b, :, :lo[b]] = math.nan
                t[b, :, hi[b]:] = math.inf
    assert torch.equal(call(prompts, own, q, dict(kw, **limits)), want)


def test_queries_in_any_layout(cuda):
    prompts, own, q, kw = setup((3, 4), 2, 4, 70, 9, seed=21)
    want = call(prompts, own, q, kw)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        wide = torch.zeros(8, 7, D + 3, 7, dtype=dtype, device="cuda")
        odd = wide.permute(1, 0, 3, 2)[:, :, 0, 1:D + 1]  # element stride 7: a copy is made
        odd.copy_(q)
        assert torch.equal(call(prompts, own, odd, kw), call(prompts, own, q.to(dtype), kw))
        rows = torch.zeros(7, 3, 8, D + 1, dtype=dtype, device="cuda")[:, 1, :, 1:]  # rows at any element
        rows.copy_(q)
        assert torch.equal(call(prompts, own, rows, kw), call(prompts, own, q.to(dtype), kw))
    assert torch.equal(call(prompts, own, q[:, :, None], kw), want)


def test_a_scale_of_its_own(cuda):
    prompts, own, q, kw = setup((3,), 2, 4, 200, 9, seed=23)
    check(call(prompts, own, q, dict(kw, scale=0.031)), reference(q, prompts, own, (3,), scale=0.031)[0])


def test_streams_and_captured_calls(cuda):
    """Two calls on streams of their own, and a captured call replayed with other queries, offsets and lengths."""
    prompts, own, q, kw = setup((4, 9), 2, 4, 500, 40, seed=25)
    cu, mine = i32([0, 4, 13]), i32([40] * 13)
    kw = dict(kw, cu_rows=cu, own_lens=mine)
    want = call(prompts, own, q, kw)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call(prompts, own, q, kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(prompts, own, q, kw)
    for counts, lens in (((4, 9), [40] * 13), ((0, 13), list(range(13))), ((11, 2), [0, 40] * 6 + [7])):
        cu.copy_(i32([0, counts[0], 13]))
        mine.copy_(i32(lens))
        q.copy_(randn(q.shape, sum(lens)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(prompts, own, q, kw))
        check(out, reference(q, prompts, own, counts, own_lens=lens)[0])


# ---------------------------------------------------------------- the shared layer


def append(layer, B, H, T, seed):
    k, v = kv_bf16((B, H, T, D), seed=seed), kv_bf16((B, H, T, D), seed=seed + 1)
    layer.update(k, v)
    return k, v


def both(counts, H, N, bits=4, qjl=True, quantize=True, seed=0):
    """A shared layer, and one with the prompt copied for every sequence."""
    base = make_layer(len(counts), H, N, bits, qjl, seed=seed)
    base.quantize_decode = quantize
    copied = copy.deepcopy(base)
    copied._take_rows(torch.arange(len(counts)).repeat_interleave(torch.tensor(counts)))
    shared = share_prefix(Cache(layers=[base]), list(counts)).layers[0]
    assert isinstance(shared, SharedPrefixLayer)
    shared._lazy_update = True
    return shared, copied


def fused(q, layer, mask=None):
    from turboquant.runtime import fused_attention

    return fused_attention(q, layer, q.shape[1] // layer._store.H, mask)


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False)])
@pytest.mark.parametrize("quantize", [True, False])
@pytest.mark.parametrize("counts", [(3, 3), (1, 6, 2)])
def test_shared_and_copied_prompts_agree(cuda, bits, qjl, quantize, counts):
    B, H = sum(counts), 2
    shared, copied = both(counts, H, 150, bits, qjl, quantize)
    q = randn((B, 8, 1, D), 5)
    check(shared_prefix_attention(q, shared), fused(q, copied).double(), 2 * TOL)  # no tokens of their own yet
    for i in range(3):
        for layer in (shared, copied):
            append(layer, B, H, 1 + 20 * i, 50 + i)
        assert shared.get_seq_length() == copied.get_seq_length()
        got, want = shared_prefix_attention(q, shared), fused(q, copied)
        assert got.shape == want.shape and got.dtype == want.dtype
        check(got, want.double(), 2 * TOL)
    mask = torch.ones(B, shared.get_seq_length(), dtype=torch.bool, device="cuda")
    mask[:counts[0], :30] = False  # the first prompt is padded on the left
    check(shared_prefix_attention(q, shared, mask), fused(q, copied, mask).double(), 2 * TOL)


def test_masks_that_are_no_shared_range_take_the_decoded_rows(cuda):
    counts, B = (3, 2), 5
    shared, copied = both(counts, 2, 100)
    for layer in (shared, copied):
        append(layer, B, 2, 5, 50)
    q = randn((B, 8, 1, D), 5)
    k, v = rows64(copied)
    hole = torch.ones(B, 105, dtype=torch.bool, device="cuda")
    hole[1, 40:60] = False
    apart = torch.ones(B, 105, dtype=torch.bool, device="cuda")
    apart[1, :30] = False  # one sequence of a prompt alone
    for mask in (hole, apart):
        ref, _ = attend64(q[:, :, 0], k, v, mask[:, None])
        # bf16 rows and weights of torch's attention: 2^-8 of the logits' terms and of the values
        check(shared_prefix_attention(q, shared, mask), ref[:, :, None], 2e-2)
    several = randn((B, 8, 4, D), 6)
    got = shared_prefix_attention(several, shared)
    for i in range(4):
        ref, _ = attend64(several[:, :, i], k[:, :, :102 + i], v[:, :, :102 + i])
        check(got[:, :, i], ref, 2e-2)


def test_rows_and_tokens_move_with_their_prompts(cuda):
    counts = (3, 2)
    shared, copied = both(counts, 2, 100, seed=4)
    for layer in (shared, copied):
        append(layer, 5, 2, 6, 50)

    def agree(B):
        q = randn((B, 8, 1, D), B)
        check(shared_prefix_attention(q, shared), fused(q, copied).double(), 2 * TOL)

    for layer in (shared, copied):
        layer.reorder_cache(torch.tensor([2, 2, 0, 4, 3], device="cuda"))
    agree(5)
    with pytest.raises(ValueError):
        shared.reorder_cache(torch.tensor([3, 1, 2, 0, 4], device="cuda"))
    with pytest.raises(IndexError):
        shared.reorder_cache(torch.tensor([0, 1, 2, 3, 5], device="cuda"))
    for layer in (shared, copied):
        layer.batch_repeat_interleave(2)
    agree(10)
    for layer in (shared, copied):
        layer.batch_select_indices(torch.tensor([0, 1, 5, 7, -1], device="cuda"))
    assert shared.counts == [3, 2]
    agree(5)
    with pytest.raises(ValueError):
        shared.batch_select_indices(torch.tensor([4, 0]))
    for layer in (shared, copied):
        layer.keep_tokens(torch.tensor([1, 3], device="cuda"), tokens=4)
    agree(5)
    for layer in (shared, copied):
        append(layer, 5, 2, 40, 60)
    agree(5)
    for layer in (shared, copied):
        layer.crop(-50)  # into the prompts
    assert shared.get_seq_length() == copied.get_seq_length() == 94
    agree(5)
    for layer in (shared, copied):
        layer.batch_select_indices(torch.tensor([False, False, False, True, True], device="cuda"))
        append(layer, 2, 2, 3, 70)
    assert shared.counts == [0, 2]
    agree(2)


def test_a_model_on_a_shared_prompt(cuda):
    """Samples of one prompt: logits of decode steps on the shared cache beside those on a repeated one, by the backend and without."""
    from turboquant.adapters.transformers import disable_turboquant_attention, enable_turboquant_attention

    model = tiny_llama("cuda", torch.bfloat16, layers=2, heads=8, kv_heads=2)
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 94, (2, 70), generator=gen).cuda()
    mask = torch.ones_like(ids)
    mask[1, :20] = 0
    logits = {}
    for kind in ("shared", "copied", "plain"):
        with torch.no_grad():
            past = model(input_ids=ids, attention_mask=mask, use_cache=True).past_key_values
            cache = build_packed_mse_cache(past, bits=4, use_qjl_keys=True, quantize_decode=True, norm_guard=False)
            if kind == "copied":
                cache.batch_repeat_interleave(3)
            else:
                cache = share_prefix(cache, 3)
            if kind != "plain":
                old = enable_turboquant_attention(model, cache)
            step, out = mask.repeat_interleave(3, 0), []
            for i in range(3):
                token = torch.randint(0, 94, (6, 1), generator=torch.Generator().manual_seed(i)).cuda()
                step = torch.cat((step, step.new_ones(6, 1)), 1)
                out.append(model(input_ids=token, attention_mask=step, past_key_values=cache, use_cache=True).logits.float())
            if kind != "plain":
                disable_turboquant_attention(model, cache, old)
        logits[kind] = torch.cat(out, 1)
    scale = logits["copied"].abs().max()
    # bf16 activations: eight roundings of 2^-9 root mean square a layer
    assert (logits["shared"] - logits["copied"]).abs().max() <= 0.03 * scale
    assert (logits["plain"] - logits["copied"]).abs().max() <= 0.03 * scale


def test_layers_that_cannot_be_shared_are_copied(cuda):
    for layer in (make_layer(2, 2, 40, 4, True, num_outlier_channels=4), make_layer(2, 2, 40, 4, True, dense=3)):
        cache = share_prefix(Cache(layers=[layer]), [1, 3])
        assert cache.layers[0] is layer and layer._batch() == 4
    with pytest.raises(ValueError):
        share_prefix(Cache(layers=[make_layer(2, 2, 40, 4, True)]), [1, 2, 3])
    with pytest.raises(ValueError):
        share_prefix(Cache(layers=[make_layer(2, 2, 40, 4, True)]), 0)


def test_masks_that_leave_a_row_nothing(cuda):
    """A sequence whose row of the mask is empty, beside another of its prompt that is not: zero, and the others as they are."""
    shared, copied = both((3, 2), 2, 100)
    for layer in (shared, copied):
        append(layer, 5, 2, 5, 50)
    k, v = rows64(copied)
    mask = torch.ones(5, 105, dtype=torch.bool, device="cuda")
    mask[1] = False
    added = torch.zeros(5, 1, 1, 105, device="cuda").masked_fill(~mask[:, None, None], -math.inf)
    q = randn((5, 8, 1, D), 5)
    ref, _ = attend64(q[:, :, 0], k, v, mask[:, None])
    for m in (mask, mask.int(), mask[:, None, None], added):
        got = shared_prefix_attention(q, shared, m)
        check(got, ref[:, :, None], 2e-2)  # bf16 rows and weights: 2^-8 of the logits' terms and of the values
        assert (got[1] == 0).all()
    several = randn((5, 8, 3, D), 6)
    for m in (mask, mask[:, None, None] & torch.ones(3, 105, dtype=torch.bool, device="cuda").tril(102)):
        got = shared_prefix_attention(several, shared, m)  # a mask of tokens leaves the order of the new ones to hold
        for i in range(3):
            ref, _ = attend64(several[:, :, i], k[:, :, :103 + i], v[:, :, :103 + i], mask[:, None, :103 + i])
            check(got[:, :, i], ref, 2e-2)


def test_a_mask_known_to_be_ranges_is_not_looked_at(cuda):
    """With the layer told so, a step with a mask can be captured."""
    shared, copied = both((2, 3), 2, 100)
    for layer in (shared, copied):
        append(layer, 5, 2, 5, 50)
    q, mask = randn((5, 8, 1, D), 5), torch.ones(5, 105, dtype=torch.bool, device="cuda")
    mask[:2, :30] = False
    want = shared_prefix_attention(q, shared, mask)
    check(want, fused(q, copied, mask).double(), 2 * TOL)
    shared._tq_mask_contiguous = True
    shared_prefix_attention(q, shared, mask)  # the ranges of this mask are known, and yet looked for at every replay
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = shared_prefix_attention(q, shared, mask)
    # (an eager call before the first replay has ranges of its own)
    check(shared_prefix_attention(q, shared, mask), fused(q, copied, mask).double(), 2 * TOL)
    for i in range(3):
        mask[2:, :10 * i] = False
        graph.replay()
        torch.cuda.synchronize()
        check(out, fused(q, copied, mask).double(), 2 * TOL)
    shared._tq_mask_contiguous = False
    check(shared_prefix_attention(q, shared, mask), fused(q, copied, mask).double(), 2e-2)


def test_a_refused_call_changes_nothing(cuda):
    shared, copied = both((2, 3), 2, 100)
    for layer in (shared, copied):
        append(layer, 5, 2, 5, 50)
    q = randn((5, 8, 1, D), 5)
    want = shared_prefix_attention(q, shared)
    for rows in (torch.zeros(5, dtype=torch.bool), torch.tensor([], dtype=torch.int64), torch.tensor([4, 1])):
        with pytest.raises(ValueError):
            shared.batch_select_indices(rows)
    assert torch.equal(shared_prefix_attention(q, shared), want)
    first, other = make_layer(2, 2, 40, 4, True, dense=3), make_layer(2, 2, 40, 4, True)
    other.attend_blocks(4)
    with pytest.raises(ValueError):
        share_prefix(Cache(layers=[first, other]), 3)
    assert first._batch() == other._batch() == 2
    other.attend_blocks(None)
    assert share_prefix(Cache(layers=[first, other]), 3).layers[1].batch == 6


def test_both_attention_interfaces_take_shared_layers(cuda):
    from turboquant.runtime.attention import turboquant_attention_forward, turboquant_prompt_forward

    shared, copied = both((2, 1), 2, 90)
    for layer in (shared, copied):
        append(layer, 3, 2, 7, 50)
    k, v = rows64(copied)
    module = torch.nn.Module()
    module._tq_cache_layer, module.num_key_value_groups = shared, 4
    for S in (1, 3):
        q = randn((3, 8, S, D), S)
        want = shared_prefix_attention(q, shared).transpose(1, 2)
        for forward in (turboquant_attention_forward, turboquant_prompt_forward):
            got, _ = forward(module, q, None, None, None)
            assert torch.equal(got, want)
    got, _ = turboquant_prompt_forward(module, q, None, None, None, is_causal=False)
    for i in range(3):
        check(got[:, i], attend64(q[:, :, i], k, v)[0], 2e-2)  # bf16 rows and weights, as above
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="packed sequences"):
        turboquant_prompt_forward(module, q, None, None, None, cu_seq_lens_q=cu)


@pytest.mark.parametrize("cap", [0, 40])
def test_caches_without_tokens(cuda, cap):
    """No tokens at all, with room for some or without: zero and -inf."""
    layer = make_layer(2, 2, 40, 4, True)
    empty = {name: t[:, :, :cap].contiguous() for name, t in arrays(layer).items()}
    own = {name: t[:1, :, :cap].expand(4, *t.shape[1:2], *t[:, :, :cap].shape[2:]).contiguous() for name, t in arrays(layer).items()}
    q = randn((4, 8, D), 5)
    for mine in (None, own):
        got, lse = K.prefix_attention(q, empty, mine, n_prefix=0, **codec(layer), want_lse=True)
        assert (got == 0).all() and (lse == -math.inf).all()
    if cap:  # a sequence's own tokens alone
        got = K.prefix_attention(q, empty, own, n_prefix=0, n_own=30, **codec(layer))
        k, v = rows64(layer)
        check(got, attend64(q, *(x[:1, :, :30].expand(4, -1, -1, -1) for x in (k, v)))[0])


def test_as_many_query_heads_as_are_taken(cuda):
    layer = make_layer(2, 1, 70, 4, True)
    k, v = rows64(layer)
    for group in (33, 47, 64):
        q = randn((4, group, D), group)
        got = K.prefix_attention(q, arrays(layer), None, n_prefix=70, **codec(layer))
        check(got, attend64(q, k.repeat_interleave(2, 0), v.repeat_interleave(2, 0))[0])
    with pytest.raises(Exception):
        K.prefix_attention(randn((4, 65, D), 1), arrays(layer), None, n_prefix=70, **codec(layer))


def test_a_prompt_past_32_bits(cuda):
    """Codes of a KV head that begin past 2^32 bytes of their buffer, and a prompt far into its row."""
    layer = make_layer(1, 2, 200, 4, False, seed=11)
    cap, H, first = (1 << 24) - 1, 5, 1 << 23  # 64 bytes a slot: 1 GB a head
    big = {}
    for name, t in arrays(layer).items():
        if t is None:
            big[name] = None
            continue
        big[name] = torch.empty(1, H, cap, *t.shape[3:], dtype=t.dtype, device="cuda")
        big[name][:, :, first:first + 200] = t[:, :1, :200]
    q = randn((3, H * 2, D), 5)
    got = K.prefix_attention(q, big, None, n_prefix=first + 200, prefix_starts=i32([first]), **codec(layer))
    k, v = (x[:, :1].expand(3, H, -1, -1) for x in rows64(layer))
    check(got, attend64(q, k, v)[0])


def test_attention_switched_off_and_on_again(cuda):
    from turboquant.adapters.transformers import disable_turboquant_attention, enable_turboquant_attention

    model = tiny_llama("cuda", torch.bfloat16, layers=2, heads=8, kv_heads=2)
    ids = torch.randint(0, 94, (1, 40), generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        cache = share_prefix(build_packed_mse_cache(model(input_ids=ids, use_cache=True).past_key_values, bits=4, use_qjl_keys=True,
                                                    quantize_decode=True, norm_guard=False), 3)
        mask = torch.ones(3, 40, dtype=torch.int64, device="cuda")
        for i in range(4):
            mask = torch.cat((mask, mask.new_ones(3, 1)), 1)
            old = enable_turboquant_attention(model, cache) if i != 1 else None
            out = model(input_ids=ids[:, i:i + 1].expand(3, 1), attention_mask=mask, past_key_values=cache, use_cache=True).logits
            assert torch.isfinite(out).all() and cache.get_seq_length() == 41 + i
            if i != 1:
                disable_turboquant_attention(model, cache, old)


@pytest.mark.parametrize("large_first", [True, False])
@pytest.mark.parametrize("n_prefix", [0, 40])
@pytest.mark.parametrize("n,H,g,M", [(2, 64, 1, 1024), (9, 130, 4, 128)])
def test_norms_of_neighbours_are_their_own(cuda, n, H, g, M, n_prefix, large_first):
    """Sequences of one prompt whose values' norms are 2^29 apart, whichever come first in the waves' tiles: each as it is alone.  As many KV
    heads as have a wave take tiles of both kinds, in blocks of 32 rows and of 64.  A weight times norm is rounded to fp16 in either call,
    by half a step, 2^-11 of it (those below 2^-25 of the largest by 2^-36 of that): the outputs differ by 2^-10 of the weighted sum of the
    values' sizes, and by the sums' roundings in fp32 and the exponents' (of numbers up to 64), below 2^-17 of it together."""
    prompts, own, q, kw = setup((n,), H, g, 64, M, seed=27)
    kw["n_prefix"] = n_prefix
    large = torch.arange(n, device="cuda") < (n + 3) // 4
    own._store.vn[:, :, :M] = torch.where(large if large_first else ~large, 2.0 ** 15, 2.0 ** -14).half()[:, None, None]
    prompts._store.vn[:, :, :64] = 2.0 ** -14
    _, f32 = call(prompts, own, q, dict(kw, want_f32=True))
    (pk, pv), (ok, ov) = rows64(prompts), rows64(own)
    for b in range(n):
        mine = {name: t[b:b + 1].contiguous() for name, t in arrays(own).items()}
        _, alone = K.prefix_attention(q[b:b + 1], arrays(prompts), mine, **kw, want_f32=True)
        k, v = torch.cat((pk[:, :, :n_prefix], ok[b:b + 1]), 2), torch.cat((pv[:, :, :n_prefix], ov[b:b + 1]), 2)
        sizes, _ = attend64(q[b:b + 1], k, v.abs())
        assert ((f32[b] - alone[0]).double().abs() <= (2.0 ** -10 + 2.0 ** -17) * sizes[0]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("bits", [1, 2, 3, 4])
@pytest.mark.parametrize("each", [2, 12])
def test_rotated_queries_keep_their_bits(cuda, dtype, bits, each):
    """Of one token's logits, where the centroids are fp16 numbers, what is left is the rotation's products (two bf16 terms each: up to 2^-16 of
    one, 2^-16 / sqrt 3 root mean square, is left out) and sums in fp32: of a logit scale |k| <q R^T, C> with |q| = sqrt 128, |k| about 20
    and |C| about 1 1.6e-5 root mean square.  One fp16 term of a rotated query (2^-11 / sqrt 12 and more) leaves 2e-4."""
    layer = make_layer(8, 2, 1, bits, False, seed=29)
    c = layer.codecs.value
    exact = K.CodecParams(c.bits, c.rotation, c.centers.half().float(), c.boundaries)
    layer.codecs = copy.copy(layer.codecs)
    layer.codecs.key = layer.codecs.value = exact
    q = randn((8 * each, 8, D), 5, torch.float32).to(dtype)
    _, lse = K.prefix_attention(q, arrays(layer), None, n_prefix=1, **codec(layer), want_lse=True)
    _, ref = reference(q, layer, None, [each] * 8)
    assert ((lse.double() - ref) ** 2).mean().sqrt() <= 5e-5


@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("size", [1.0, 1e-3])
@pytest.mark.parametrize("each", [2, 12])
def test_fp32_queries_lose_little_to_fp16_codebooks(cuda, bits, qjl, size, each):
    """Of the output's norm: keys' centroids 1.2e-4 of a key, which moves a logit of |q| = sqrt 128 and |k| = 20 by 2.4e-4; values' 1.5e-4;
    weights times norms 1.7e-4; signs' queries 0.8e-4: 3.4e-4 together.  With queries of a thousandth all tokens weigh the same, the values
    nearly cancel, and the errors' mean would be what is left."""
    counts = (each,)
    prompts, own, q, kw = setup(counts, 2, 4, 8192, 64, bits, qjl, torch.float32, seed=31)
    q = q * size
    ref, _ = reference(q, prompts, own, counts)
    assert (call(prompts, own, q, kw).double() - ref).norm() <= 4e-4 * ref.norm()


def test_a_codec_made_by_hand_on_several_streams(cuda):
    """Its codebooks are made at the first call, on that call's stream, and taken by calls on others."""
    prompts, own, q, kw = setup((3, 4), 2, 4, 300, 20, seed=33)
    want = call(prompts, own, q, kw)
    torch.cuda.synchronize()
    kw.update({name: K.CodecParams(c.bits, c.rotation, c.centers, c.boundaries) for name, c in (("key", kw["key"]), ("value", kw["value"]))})
    outs = []
    for held_up in (10_000_000, 0):
        with torch.cuda.stream(torch.cuda.Stream()):
            if held_up:
                torch.cuda._sleep(held_up)
            outs.append(call(prompts, own, q, kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs.append(call(prompts, own, q, kw))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    alone = {name: K.CodecParams(c.bits, c.rotation, c.centers, c.boundaries) for name, c in (("key", kw["key"]), ("value", kw["value"]))}
    K.attention_value_centers(alone["value"])
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):  # a capture that nothing came before
        out = call(prompts, own, q, dict(kw, **alone))
    graph.replay()
    torch.cuda.synchronize()
    check(out, reference(q, prompts, own, (3, 4))[0])
