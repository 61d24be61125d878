"""Weights far below their row's largest, against fp64."""

import math

import pytest
import torch

from turboquant.runtime import prompt_attention

pytestmark = pytest.mark.gpu

D = 128


# one query head takes blocks of 128 rows, 18 of them (576 blocks) blocks of 256
@pytest.mark.parametrize("heads", [1, 18])
@pytest.mark.parametrize("above", [10.0, 12.0])
def test_the_log_sum_exp_of_many_small_weights(cuda, heads, above):
    """4095 weights of e^-above beside one of 1.  fp32 logits below 16 are off by 128 2^-24 16 / 16 = 8e-6 at most, a tile's
    sum of 32 weights a lane by 32 2^-24 of itself, that of 64 tiles by 64 2^-24 = 4e-6, the exponentials and the
    logarithm by a few 2^-23."""
    S = 4096
    q, k = (torch.zeros(1, h, S, D, device="cuda", dtype=torch.bfloat16) for h in (heads, 1))
    q[..., 0], k[:, :, 0, 0] = 8.0, above * math.sqrt(D) / 8
    _, lse = prompt_attention(q, k, k, return_lse=True)
    top = 8.0 * k[0, 0, 0, 0].double() / math.sqrt(D)
    ref = top + torch.log1p(torch.arange(S, device="cuda") * torch.exp(-top))
    assert (lse.double() - ref).abs().max() <= 2e-5
