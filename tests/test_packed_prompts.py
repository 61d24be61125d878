"""Prompts packed behind one another through the attention interface "turboquant_prompt", where its kernel does not take the
call: each sequence is attended to as when it is run alone.  On the CPU."""

import math

import pytest
import torch

from turboquant.runtime.attention import turboquant_prompt_forward
from turboquant.runtime.packed_qmse_cache import PackedMSELayer

SCALE = 0.07


class Module(torch.nn.Module):
    is_causal, num_key_value_groups = True, 4


def tensors(S, D=128, dtype=torch.float32, keys=None):
    gen = torch.Generator().manual_seed(S)
    return tuple(torch.randn(1, h, n, D, generator=gen).to(dtype) for h, n in ((8, S), (2, keys or S), (2, keys or S)))


def alone(q, k, v, causal=True, window=None):
    """fp64; rows and keys of a sequence end together."""
    n, m = q.shape[2], k.shape[2]
    x = q.double() @ k.double().repeat_interleave(4, 1).transpose(-1, -2) * SCALE
    back = torch.arange(m)[None, :] - torch.arange(n)[:, None] + n - m  # 0: the row's own token
    if causal:
        x = x.masked_fill(back > 0, -math.inf)
    if window:
        x = x.masked_fill(back <= -window, -math.inf)
    return torch.softmax(x, -1) @ v.double().repeat_interleave(4, 1)


def check(got, want, dtype):
    """fp32: sums of 128 products and a few weights.  bf16: torch may round logits (below 8), weights and outputs, half a step each."""
    tol = 1e-5 if dtype == torch.float32 else 2 ** -8 * (8 + 1 + 1)
    assert (got.transpose(1, 2).double() - want).abs().max() <= tol * want.abs().max()


def offsets(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


@pytest.mark.parametrize("dtype,D,grad", [(torch.float32, 128, False), (torch.float32, 64, True), (torch.bfloat16, 128, False),
                                          (torch.bfloat16, 128, True)])
@pytest.mark.parametrize("lens,tail", [([3, 3], 0), ([1, 0, 7, 2], 0), ([5], 0), ([4, 6], 3), ([0, 0], 4)])
def test_each_sequence_as_if_alone(dtype, D, grad, lens, tail):
    total, at = sum(lens) + tail, offsets(lens)
    q, k, v = tensors(total, D, dtype)
    q.requires_grad_(grad)
    got, _ = turboquant_prompt_forward(Module(), q, k, v, None, scaling=SCALE, cu_seq_lens_q=at, cu_seq_lens_k=at.clone())
    for a, b in zip(at.tolist(), at.tolist()[1:]):
        if b > a:
            check(got[:, a:b], alone(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b]), dtype)
    assert (got[:, total - tail:] == 0).all()  # rows of no sequence
    if grad:
        got.sum().backward()
        assert torch.isfinite(q.grad).all()


def test_rows_before_the_first_offset():
    q, k, v = tensors(9)
    got, _ = turboquant_prompt_forward(Module(), q, k, v, None, scaling=SCALE, cu_seq_lens_q=offsets([4, 3], first=2))
    assert (got[:, :2] == 0).all()
    check(got[:, 2:6], alone(q[:, :, 2:6], k[:, :, 2:6], v[:, :, 2:6]), torch.float32)


def test_keys_of_other_lengths_than_the_rows():
    q, k, v = tensors(6, keys=12)
    cq, ck = offsets([2, 4]), offsets([7, 5])
    got, _ = turboquant_prompt_forward(Module(), q, k, v, None, scaling=SCALE, cu_seq_lens_q=cq, cu_seq_lens_k=ck)
    check(got[:, :2], alone(q[:, :, :2], k[:, :, :7], v[:, :, :7]), torch.float32)
    check(got[:, 2:], alone(q[:, :, 2:], k[:, :, 7:], v[:, :, 7:]), torch.float32)


def test_not_causal_and_a_window():
    q, k, v = tensors(11)
    cu = offsets([4, 7])
    both, _ = turboquant_prompt_forward(Module(), q, k, v, None, scaling=SCALE, is_causal=False, cu_seq_lens_q=cu)
    near, _ = turboquant_prompt_forward(Module(), q, k, v, None, scaling=SCALE, sliding_window=3, cu_seq_lens_q=cu)
    for a, b in ((0, 4), (4, 11)):
        x = (q[:, :, a:b], k[:, :, a:b], v[:, :, a:b])
        check(both[:, a:b], alone(*x, causal=False), torch.float32)
        check(near[:, a:b], alone(*x, window=3), torch.float32)


def test_refusals():
    q, k, v = tensors(6)
    m = Module()
    cu = offsets([3, 3])
    with pytest.raises(ValueError, match="batch of 1"):
        turboquant_prompt_forward(m, *(x.repeat(2, 1, 1, 1) for x in (q, k, v)), None, cu_seq_lens_q=cu)
    with pytest.raises(ValueError, match="as many sequences"):
        turboquant_prompt_forward(m, q, k, v, None, cu_seq_lens_q=cu, cu_seq_lens_k=offsets([1, 2, 3]))
    # sequences behind a history that is none of theirs
    m._tq_cache_layer = layer = PackedMSELayer(bits=4)
    layer._lazy_update = True
    layer.update(k, v)
    assert turboquant_prompt_forward(m, q, k, v, None, cu_seq_lens_q=cu)[0].shape == (1, 6, 8, 128)
    layer.update(k, v)
    with pytest.raises(ValueError, match="holds tokens before"):
        turboquant_prompt_forward(m, q, k, v, None, cu_seq_lens_q=cu)


@pytest.mark.parametrize("history", [None, 0, 4])
def test_rows_that_are_not_causal(history):
    """Without packed sequences too: every row attends to all that there is, of the call or of the layer."""
    q, k, v = tensors(6)
    m, keys = Module(), (k, v)
    m.is_causal = False
    if history is not None:
        m._tq_cache_layer = layer = PackedMSELayer(bits=4)
        layer._lazy_update = True
        if history:
            layer.update(k[:, :, :history] * 0.5, v[:, :, :history] * 2)
            keys = torch.cat((k[:, :, :history] * 0.5, k), 2), torch.cat((v[:, :, :history] * 2, v), 2)
        layer.update(k, v)
    got, _ = turboquant_prompt_forward(m, q, k, v, None, scaling=SCALE)
    check(got, alone(q, *keys, causal=False), torch.float32)


def test_a_mask_is_what_counts_and_one_row_is_a_step():
    q, k, v = tensors(6)
    cu, m = offsets([3, 3]), Module()
    mask = torch.ones(1, 1, 6, 6, dtype=torch.bool).tril()
    got, _ = turboquant_prompt_forward(m, q, k, v, mask, scaling=SCALE, cu_seq_lens_q=cu)
    check(got, alone(q, k, v), torch.float32)
    one, _ = turboquant_prompt_forward(m, q[:, :, -1:], k, v, None, scaling=SCALE, cu_seq_lens_q=offsets([1]),
                                       cu_seq_lens_k=offsets([6]))
    check(one, alone(q[:, :, -1:], k, v), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, True)])
def test_the_same_on_the_gpu(cuda, dtype, grad):
    """Where the kernel takes it (no gradient), and where torch does."""
    at = offsets([130, 0, 1, 70])
    q, k, v = (x.to(cuda) for x in tensors(210, dtype=dtype))
    for needs in {False, grad}:
        got, _ = turboquant_prompt_forward(Module(), q.requires_grad_(needs), k, v, None, scaling=SCALE, cu_seq_lens_q=at.to(cuda))
        for a, b in zip(at.tolist(), at.tolist()[1:]):
            if b > a:
                check(got[:, a:b].detach().cpu(), alone(*(x[:, :, a:b].detach().cpu() for x in (q, k, v))), dtype)
        assert (got[:, 201:] == 0).all()
