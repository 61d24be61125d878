"""Causal attention over whole prompts (tq_prompt_attention) against fp64: block and tile edges, grouped heads,
both types, strides, padded batches, packed sequences, values that are not finite, graphs and streams."""

import math

import pytest
import torch

from turboquant.runtime import kernels as K
from turboquant.runtime import prompt_attention

pytestmark = pytest.mark.gpu

D = 128
SCALE = 1.0 / math.sqrt(D)


def randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def oracle(q, k, v, ranges=None, scale=SCALE):
    """fp64 output, log-sum-exp and mean absolute value of the rows; ``ranges`` (batch row, start, end) of each
    sequence, rows outside are 0."""
    B, Hq, S, _ = q.shape
    g = Hq // k.shape[1]
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full((B, Hq, S), float("-inf"), dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    for b, lo, hi in ([(b, 0, S) for b in range(B)] if ranges is None else ranges):
        if hi <= lo:
            continue
        x = q[b, :, lo:hi].double() @ k[b, :, lo:hi].double().repeat_interleave(g, 0).transpose(-1, -2) * scale
        x = x.masked_fill(torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        p = torch.softmax(x, -1)
        vd = v[b, :, lo:hi].double().repeat_interleave(g, 0)
        out[b, :, lo:hi] = (p @ vd).cpu()
        size[b, :, lo:hi] = (p @ vd.abs()).cpu()
        lse[b, :, lo:hi] = torch.logsumexp(x, -1).cpu()
    return out, lse, size


def check(got, ref, size):
    """The output's rounding (half a step of the result), the weights' (half a step of each, so of the mean
    absolute value), and 2e-5 of it for the fp32 logits, weights and sums (logits below 32: their 128
    exact products add up within 128 * 2^-24 * 32 / 16 = 1.6e-5 of what the weights are, the exponentials and
    sums within a few 2^-23)."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    bound = half * ref.abs() + (half + half * half + 2e-5) * size
    if half < 2 ** -9:  # fp16: outputs and weights below 2^-14 lose bits, up to half of 2^-24 each
        bound = bound + 2 ** -24
    assert torch.isfinite(got).all()
    assert ((got - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,g,S", [(1, 1, 1, 1), (2, 1, 3, 2), (1, 2, 4, 31), (1, 8, 4, 64), (2, 2, 7, 65),
                                       (1, 3, 1, 127), (1, 4, 5, 128), (1, 2, 8, 129), (3, 1, 16, 255), (1, 8, 4, 256),
                                       (1, 4, 2, 257), (1, 2, 4, 511), (1, 1, 4, 1025), (2, 8, 4, 700)])
def test_prompts_match_fp64(cuda, dtype, B, Hkv, g, S):
    q = randn((B, S, Hkv * g, D), 1, dtype).transpose(1, 2)
    k, v = randn((B, S, Hkv, D), 2, dtype).transpose(1, 2), randn((B, Hkv, S, D), 3, dtype)
    got, lse = prompt_attention(q, k, v, return_lse=True)
    ref, ref_lse, size = oracle(q, k, v)
    assert got.shape == q.shape and got.dtype == dtype
    check(got, ref, size)
    assert (lse.double().cpu() - ref_lse).abs().max() <= 4e-5


def test_a_long_prompt(cuda):
    q, k, v = (randn((1, h, 5003, D), i, torch.bfloat16) for i, h in ((1, 4), (2, 2), (3, 2)))
    got = prompt_attention(q, k, v)
    ref, _, size = oracle(q, k, v)
    check(got, ref, size)


@pytest.mark.parametrize("S", [70, 300])
def test_large_logits_and_a_scale(cuda, S):
    """Logits up to several hundreds: rows of almost one weight, references that rise often."""
    q, k, v = (randn((1, h, S, D), i, torch.bfloat16) for i, h in ((1, 4), (2, 2), (3, 2)))
    k = k * torch.linspace(0.1, 8, S, device="cuda").to(torch.bfloat16)[None, None, :, None]
    got = prompt_attention(q, k, v, scale=0.5)
    ref, _, size = oracle(q, k, v, scale=0.5)
    # |logits| <= 0.5 * 8 * 128 = 512: products add up within 128 * 2^-24 * 512 = 3.9e-3 at most of every weight
    check_bound = 2 ** -8 * ref.abs() + (2 ** -8 + 4e-3) * size
    assert ((got.double().cpu() - ref).abs() <= check_bound).all()


def test_padded_batches(cuda):
    S = 300
    q, k, v = (randn((5, S, h, D), i, torch.bfloat16).transpose(1, 2) for i, h in ((1, 8), (2, 2), (3, 2)))
    starts = [0, 1, 130, 299, 300]
    ends = [300, 299, 290, 300, 300]
    for b in range(5):  # padding holds anything
        for x in (k, v):
            x[b, :, :starts[b]] = float("nan")
            x[b, :, ends[b]:] = float("inf")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got, lse = prompt_attention(q, k, v, seq_starts=i32(starts), seq_ends=i32(ends), return_lse=True)
    ref, ref_lse, size = oracle(q, k, v, [(b, starts[b], ends[b]) for b in range(5)])
    check(got, ref, size)
    live = torch.isfinite(ref_lse)
    assert (lse.cpu()[~live] == float("-inf")).all()
    assert (lse.double().cpu() - ref_lse)[live].abs().max() <= 4e-5
    only = prompt_attention(q[:2], k[:2], v[:2], seq_starts=i32(starts[:2]).long())
    k[:2, :, 299:] = v[:2, :, 299:] = 1.0
    assert torch.equal(only[0], got[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,tail", [([1], 0), ([300], 0), ([0, 5, 0, 0, 129, 1, 256, 0], 0), ([17] * 150, 3),
                                       ([100, 28], 400), ([0, 0], 5)])
def test_packed_sequences(cuda, dtype, lens, tail):
    total = sum(lens) + tail
    q, k, v = (randn((1, total, h, D), i, dtype).transpose(1, 2) for i, h in ((1, 6), (2, 2), (3, 2)))
    if tail:
        for x in (q, k, v):
            x[:, :, total - tail:] = float("nan")
    at = [sum(lens[:i]) for i in range(len(lens) + 1)]
    cu = torch.tensor(at, dtype=torch.int32, device="cuda")
    got, lse = prompt_attention(q, k, v, cu_seqlens=cu, return_lse=True)
    ref, ref_lse, size = oracle(q, k, v, [(0, a, b) for a, b in zip(at, at[1:])])
    check(got, ref, size)
    live = torch.isfinite(ref_lse)
    assert (lse.cpu()[~live] == float("-inf")).all()
    assert ((lse.double().cpu() - ref_lse)[live].abs() <= 4e-5).all()
    # rows behind the last sequence stay as they were in a given output
    mine = torch.full((1, 6, total, D), 7.0, dtype=dtype, device="cuda")
    assert prompt_attention(q, k, v, cu_seqlens=cu, out=mine) is mine
    assert torch.equal(mine[:, :, :total - tail], got[:, :, :total - tail]) and (mine[:, :, total - tail:] == 7.0).all()


def test_rows_before_the_first_offset_belong_to_no_sequence(cuda):
    q, k, v = (randn((1, h, 200, D), i, torch.bfloat16) for i, h in ((1, 2), (2, 2), (3, 2)))
    cu = torch.tensor([150, 180], dtype=torch.int32, device="cuda")
    ref, _, size = oracle(q, k, v, [(0, 150, 180)])
    check(prompt_attention(q, k, v, cu_seqlens=cu), ref, size)


def test_strided_operands_and_output(cuda):
    buf = randn((2, 90, 20, 3 * D), 1, torch.bfloat16)
    q, k, v = buf[:, :, 2:10, :D].transpose(1, 2), buf[:, 5:, 11:13, D:2 * D].transpose(1, 2), buf[:, 5:, 13:15, 2 * D:].transpose(1, 2)
    q = q[:, :, 5:]
    ref, _, size = oracle(q, k, v)
    into = torch.zeros(2, 8, 85, 2 * D, dtype=torch.bfloat16, device="cuda")
    got = prompt_attention(q, k, v, out=into[..., D:])
    check(got, ref, size)
    assert (into[..., :D] == 0).all()
    # rows that are not 16-byte aligned are copied
    odd = randn((1, 2, 40, D + 1), 4, torch.bfloat16)
    ref, _, size = oracle(odd[..., 1:], odd[..., 1:], odd[..., :-1])
    check(prompt_attention(odd[..., 1:], odd[..., 1:], odd[..., :-1]), ref, size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,at", [(5, 3), (64, 63), (130, 64), (300, 200), (300, 299)])
def test_values_that_are_not_finite_reach_later_rows_only(cuda, dtype, S, at):
    q, k, v = (randn((1, h, S, D), i, dtype) for i, h in ((1, 4), (2, 1), (3, 1)))
    ref, _, size = oracle(q, k, v)
    v[0, 0, at, 3], v[0, 0, at, 7], v[0, 0, at, 100] = float("inf"), float("-inf"), float("nan")
    if at + 1 < S:
        v[0, 0, at + 1, 3] = float("-inf")
    got = prompt_attention(q, k, v)
    check(got[:, :, :at], ref[:, :, :at], size[:, :, :at])
    assert (got[:, :, at, 3] == float("inf")).all() and (got[:, :, at:, 7] == float("-inf")).all()
    assert got[:, :, at:, 100].isnan().all() and got[:, :, at + 1:, 3].isnan().all()
    rest = [d for d in range(D) if d not in (3, 7, 100)]
    check(got[..., rest], ref[..., rest], size[..., rest])


def test_keys_and_queries_that_are_not_finite(cuda):
    q, k, v = (randn((1, 2, 100, D), i, torch.bfloat16) for i in (1, 2, 3))
    ref, _, size = oracle(q, k, v)
    k[0, 0, 50], q[0, 1, 30] = float("nan"), float("nan")
    got = prompt_attention(q, k, v)
    assert got[0, 0, 50:].isnan().all() and got[0, 1, 30].isnan().all()
    check(got[:, 0:1, :50], ref[:, 0:1, :50], size[:, 0:1, :50])
    others = [i for i in range(100) if i != 30]
    check(got[:, 1:, others], ref[:, 1:, others], size[:, 1:, others])


def test_replays_of_a_graph_and_other_streams(cuda):
    q, k, v = (randn((1, h, 333, D), i, torch.bfloat16) for i, h in ((1, 4), (2, 2), (3, 2)))
    cu = torch.tensor([0, 100, 333], dtype=torch.int32, device="cuda")
    eager = prompt_attention(q, k, v, cu_seqlens=cu)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = prompt_attention(q, k, v, cu_seqlens=cu)
    for seed in (1, 11, 21):
        q.copy_(randn(q.shape, seed, torch.bfloat16))
        cu.copy_(torch.tensor([0, 100 + seed, 333 - seed], dtype=torch.int32))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            again = prompt_attention(q, k, v, cu_seqlens=cu)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, again)
    assert not torch.equal(out, eager)


def test_the_same_bits_every_time(cuda):
    q, k, v = (randn((2, h, 900, D), i, torch.bfloat16) for i, h in ((1, 8), (2, 4), (3, 4)))
    first = K.prompt_attention(q, k, v)
    for _ in range(3):
        assert torch.equal(K.prompt_attention(q, k, v), first)


def test_refusals_and_empty_calls(cuda):
    q, k = randn((2, 4, 8, D), 1, torch.bfloat16), randn((2, 2, 8, D), 2, torch.bfloat16)
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="packed"):
        prompt_attention(q, k, k, cu_seqlens=cu)
    with pytest.raises(ValueError, match="backward"):
        prompt_attention(q.float().requires_grad_().bfloat16(), k, k)
    with pytest.raises(RuntimeError, match="tq_prompt_attention"):
        prompt_attention(q, k, k, scale=0.0)
    with pytest.raises(ValueError, match="out must"):
        prompt_attention(q, k, k, out=torch.empty(2, 4, 8, D, device="cuda"))
    assert prompt_attention(q[:, :, :0], k[:, :, :0], k[:, :, :0]).shape == (2, 4, 0, D)
    assert prompt_attention(q[:0], k[:0], k[:0]).shape == (0, 4, 8, D)


# calls of more than 512 blocks of 128 rows take blocks of 256
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hkv,g,S", [(130, 4, 1), (130, 4, 65), (66, 4, 129), (1, 176, 257), (28, 4, 600), (15, 4, 1100)])
def test_many_blocks_match_fp64(cuda, dtype, Hkv, g, S):
    q, k, v = (randn((1, S, h, D), i, dtype).transpose(1, 2) for i, h in ((1, Hkv * g), (2, Hkv), (3, Hkv)))
    got, lse = prompt_attention(q, k, v, return_lse=True)
    ref, ref_lse, size = oracle(q, k, v)
    check(got, ref, size)
    assert (lse.double().cpu() - ref_lse).abs().max() <= 4e-5


def test_many_blocks_of_padded_batches(cuda):
    S = 300
    q, k, v = (randn((5, S, h, D), i, torch.bfloat16).transpose(1, 2) for i, h in ((1, 36), (2, 9), (3, 9)))
    starts, ends = [0, 1, 130, 299, 300], [300, 299, 290, 300, 300]
    for b in range(5):
        for x in (k, v):
            x[b, :, :starts[b]] = float("nan")
            x[b, :, ends[b]:] = float("inf")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = prompt_attention(q, k, v, seq_starts=i32(starts), seq_ends=i32(ends))
    ref, _, size = oracle(q, k, v, [(b, starts[b], ends[b]) for b in range(5)])
    check(got, ref, size)


def test_many_blocks_of_packed_sequences(cuda):
    lens, tail = [300, 0, 5, 129, 1, 256, 0, 513], 40
    total = sum(lens) + tail
    q, k, v = (randn((1, total, h, D), i, torch.float16).transpose(1, 2) for i, h in ((1, 60), (2, 10), (3, 10)))
    for x in (k, v):
        x[:, :, total - tail:] = float("nan")
    at = [sum(lens[:i]) for i in range(len(lens) + 1)]
    cu = torch.tensor(at, dtype=torch.int32, device="cuda")
    mine = torch.full((1, 60, total, D), 7.0, dtype=torch.float16, device="cuda")
    prompt_attention(q, k, v, cu_seqlens=cu, out=mine)
    ref, _, size = oracle(q, k, v, [(0, a, b) for a, b in zip(at, at[1:])])
    check(mine[:, :, :total - tail], ref[:, :, :total - tail], size[:, :, :total - tail])
    assert (mine[:, :, total - tail:] == 7.0).all()


@pytest.mark.parametrize("at", [0, 63, 200, 299])
def test_values_that_are_not_finite_in_many_blocks(cuda, at):
    q, k, v = (randn((1, h, 300, D), i, torch.bfloat16) for i, h in ((1, 176), (2, 2), (3, 2)))
    ref, _, size = oracle(q, k, v)
    v[0, 0, at, 3], v[0, 0, at, 7] = float("-inf"), float("nan")
    got = prompt_attention(q, k, v)
    check(got[:, :88, :at], ref[:, :88, :at], size[:, :88, :at])
    check(got[:, 88:], ref[:, 88:], size[:, 88:])
    assert (got[:, :88, at:, 3] == float("-inf")).all() and got[:, :88, at:, 7].isnan().all()
    rest = [d for d in range(D) if d not in (3, 7)]
    check(got[..., rest], ref[..., rest], size[..., rest])


class Module(torch.nn.Module):
    is_causal, num_key_value_groups = True, 4


def test_attention_interface(cuda):
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    forward, m = ALL_ATTENTION_FUNCTIONS["turboquant_prompt"], Module()
    q, k, v = (randn((1, h, 150, D), i, torch.bfloat16) for i, h in ((1, 8), (2, 2), (3, 2)))
    got, _ = forward(m, q, k, v, None, scaling=0.05)
    assert torch.equal(got, prompt_attention(q, k, v, scale=0.05).transpose(1, 2))
    cu = torch.tensor([0, 60, 150], dtype=torch.int32, device="cuda")
    for other in (cu, cu.clone()):
        got, _ = forward(m, q, k, v, None, scaling=0.05, cu_seq_lens_q=cu, cu_seq_lens_k=other)
        assert torch.equal(got, prompt_attention(q, k, v, scale=0.05, cu_seqlens=cu).transpose(1, 2))
    # what the kernel does not take goes the other way, with the same result as there
    other = ALL_ATTENTION_FUNCTIONS["turboquant"]
    mask = torch.ones(1, 1, 150, 150, dtype=torch.bool, device="cuda").tril()
    mask[..., :9] = False
    mask[..., 0] = True
    for args in ((q, k, v, mask), (q.float(), k.float(), v.float(), None), (q[:, :, -1:], k, v, None),
                 (q[..., :64], k[..., :64], v[..., :64], None)):
        assert torch.equal(forward(m, *args, scaling=0.05)[0], other(m, *args, scaling=0.05)[0])


def test_a_models_prompt_takes_it(cuda, monkeypatch):
    import turboquant
    from turboquant.runtime import attention as A

    from ._tiny_model import CharTokenizer, tiny_llama

    calls = []
    monkeypatch.setattr(A, "prompt_attention", lambda *a, **kw: calls.append(a[0].shape) or prompt_attention(*a, **kw))
    model = tiny_llama(device=cuda, dtype=torch.bfloat16)
    ids = torch.randint(0, 94, (1, 300), generator=torch.Generator().manual_seed(0)).to(cuda)
    with torch.no_grad():
        ref = model(ids).logits.float()
        model.set_attn_implementation("turboquant_prompt")
        got = model(ids).logits.float()
    assert calls == [(1, 8, 300, D)] * 2
    # two layers, each with a few bf16 roundings (2^-8) of activations that both sides round at other places
    assert (got - ref).abs().max() <= 16 * 2 ** -8 * ref.abs().max()
    turboquant.activate(model, CharTokenizer(), bits=4, use_qjl_keys=True, quiet=True)
    assert model.generate(ids, max_new_tokens=5).shape == (1, 305)
    assert len(calls) >= 4


def test_keys_far_apart(cuda):
    """Token strides up to the limit: offsets inside a tile take all of 32 bits."""
    S, st = 130, (1 << 25) - 8
    flat = torch.empty((S - 1) * st + 4 * D, dtype=torch.bfloat16, device="cuda")
    k, v = (flat.as_strided((1, 2, S, D), (0, D, st, 1), at) for at in (0, 2 * D))
    k.copy_(randn(k.shape, 2, torch.bfloat16))
    v.copy_(randn(v.shape, 3, torch.bfloat16))
    q = randn((1, 8, S, D), 1, torch.bfloat16)
    got = prompt_attention(q, k, v)
    ref, _, size = oracle(q, k.contiguous(), v.contiguous())
    check(got, ref, size)
    many = prompt_attention(q.repeat(1, 64, 1, 1), k, v)  # blocks of 256 rows: the first 256 heads share KV head 0
    assert torch.equal(many[:, :256].unflatten(1, (32, 8))[:, :, :4], many[:, :4][:, None].expand(-1, 32, -1, -1, -1))
    ref, _, size = oracle(q.repeat(1, 64, 1, 1)[:, [0, 300]], k.contiguous(), v.contiguous())
    check(many[:, [0, 300]], ref, size)
