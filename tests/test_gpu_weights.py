"""Weights far below their row's largest, and values near the ends of their type's range, against fp64."""

import math

import pytest
import torch

from turboquant.runtime import kernels as K
from turboquant.runtime import prompt_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16

from .test_gpu_tree import attend, rows64

pytestmark = pytest.mark.gpu

D = 128


def randn(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def causal(q, k, v, rows):
    """fp64 output and mean absolute value of these rows of one KV head's query heads [Hq, S, D]."""
    x = q[:, rows].double() @ k.double().T / math.sqrt(D)
    x = x.masked_fill(torch.arange(k.shape[0], device=x.device) > rows[:, None], float("-inf"))
    p = torch.softmax(x, -1)
    return p @ v.double(), p @ v.double().abs()


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


@pytest.mark.parametrize("heads", [1, 18])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("above", [10.0, 17.0, 18.4, 20.0])
def test_a_first_token_far_above_the_others_of_a_prompt(cuda, heads, dtype, above):
    """Its value is zero, so the output is what the small weights, all e^-above, give.

    A weight w of a row whose largest is 1 is rounded by half a step, half w, or in fp16 below 2^-25 by half of 2^-35: 4095 of
    them, of values up to 2, by 2^-23 in all.  An fp16 output below 2^-14 is rounded by 2^-25.  fp32 logits of 20 are off by
    128 2^-24 20 / 16 = 1e-5 at most, 2e-5 with the exponentials; the sums of 64 tiles by 64 2^-24 = 4e-6."""
    S = 4096
    q = torch.zeros(1, heads, S, D, device="cuda", dtype=dtype)
    k, v = torch.zeros(1, 1, S, D, device="cuda", dtype=dtype), (1 + randn((1, 1, S, D), 1).sigmoid()).to(dtype)
    q[..., 0], k[:, :, 0, 0], v[:, :, 0] = 8.0, above * math.sqrt(D) / 8, 0.0
    got = prompt_attention(q, k, v)
    rows = torch.tensor([0, 1, 63, 64, 500, 2047, 4000, 4095], device="cuda")
    ref, size = causal(q[0], k[0, 0], v[0, 0], rows)
    half = torch.finfo(dtype).eps / 2
    bound = half * ref.abs() + (half + half * half + 3e-5) * size
    if dtype == torch.float16:
        bound = bound + 2 ** -23 + 2 ** -25
    assert ((got[0][:, rows].double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("heads", [1, 18])
@pytest.mark.parametrize("dtype,most", [(torch.bfloat16, 3.3e38), (torch.float16, 65504.0)])
def test_values_near_the_end_of_their_range(cuda, heads, dtype, most):
    """A weighted mean of finite values is finite, however many they are, also beside an infinity in another dim.  (Weights'
    sums of 64 tiles are off by 64 2^-24, products' of 256 times 16 tokens by 256 2^-24 = 2e-5.)"""
    S = 4096
    q, k = randn((1, heads, S, D), 1).to(dtype), randn((1, 1, S, D), 2).to(dtype)
    v = ((0.5 + randn((1, 1, S, D), 3).sigmoid() / 2) * most).to(dtype)
    v[..., 64:] = -v[..., 64:]
    rows = torch.tensor([0, 1, 2, 63, 64, 500, 2047, 4000, 4095], device="cuda")
    ref, size = causal(q[0], k[0, 0], v[0, 0], rows)
    half = torch.finfo(dtype).eps / 2
    bound = half * ref.abs() + (half + half * half + 5e-5) * size
    for infinite in (False, True):
        if infinite:
            v[:, :, 70, 5] = float("inf")
        got = prompt_attention(q, k, v)[0][:, rows].double()
        if infinite:
            assert (got[:, 5:, 5] == float("inf")).all()
            got[:, 5:, 5] = ref[:, 5:, 5]
        assert torch.isfinite(got).all()
        assert ((got - ref).abs() <= bound).all()


def test_two_tiles_of_one_large_weight_each(cuda):
    """Two values near the end of bf16's range in tiles of 64 tokens that different waves walk: each sum is finite."""
    q, k, v = (torch.zeros(1, 1, 128, D, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    q[..., 0], k[:, :, (5, 70), 0], v[:, :, (5, 70)] = 8.0, 100.0, 3.3e38
    got = prompt_attention(q, k, v)[0].double()
    ref = torch.full((128, 1), float(v[0, 0, 5, 0]), dtype=torch.float64, device="cuda")
    ref[:5] = 0.0
    assert ((got - ref).abs() <= 2 ** -8 * ref + 1e-5 * ref).all()


def test_small_values_beside_nothing_else(cuda):
    """bf16 values down to 2^-100 keep their digits."""
    q, k = randn((1, 2, 300, D), 1).bfloat16(), randn((1, 1, 300, D), 2).bfloat16()
    v = (randn((1, 1, 300, D), 3).bfloat16().float() * 2.0 ** -100).bfloat16()
    got = prompt_attention(q, k, v)
    rows = torch.arange(300, device="cuda")
    ref, size = causal(q[0], k[0, 0], v[0, 0], rows)
    assert ((got[0].double() - ref).abs() <= 2 ** -8 * ref.abs() + (2 ** -8 + 2 ** -16 + 2e-5) * size).all()


@pytest.mark.parametrize("qjl", [False, True])
@pytest.mark.parametrize("nodes", [3, 20])
@pytest.mark.parametrize("above", [10.0, 17.0, 18.4, 19.7])
def test_tokens_far_above_the_others_of_a_tree(cuda, qjl, nodes, above):
    """One token of every 32 far above the others, with a value of next to nothing; the others' keys are zero and their
    values alike, so that the output is what 31 of 32 small weights give.

    Weights times norms are fp16 numbers w in units of 2^-11 of the reference's times a power of two above the largest norm
    (20 of 32 here): below 2^-14 they are off by 2^-25.  The large logits are of the size that the package's tolerance of 2e-3
    is derived for and move all weights alike: the error of 1e-3 root mean square may be four times that."""
    layer = PackedMSELayer(bits=4, use_qjl_keys=qjl, quantize_decode=True)
    N = 4096
    layer.initialize_from_dense(kv_bf16((1, 1, N, D), seed=1), kv_bf16((1, 1, N, D), seed=2))
    st, c, first = layer._store, layer.codecs, slice(7, N - nodes, 32)
    for n in (st.kc, st.ks) if qjl else (st.kc,):
        n[:, :, first] = n[:, :, 7:8].clone()
    st.vc[:, :, :N], st.vn[:, :, :N] = st.vc[:, :, 5:6].clone(), 20.0
    st.vn[:, :, first] = 2.0 ** -24
    for n in (st.kn, st.kr) if qjl else (st.kn,):
        one = n[:, :, 7:8].clone()
        n.zero_()
        n[:, :, first] = one
    k, v = rows64(layer)
    row = k[0, 0, 7]
    q = (row * (above * math.sqrt(D) / (row @ row))).float().expand(1, 4, nodes, D).contiguous()
    _, f32, lse = K.tree_attention(q, torch.full((nodes,), -1, device="cuda"), k_codes=st.kc, k_norms=st.kn, v_codes=st.vc,
                                   v_norms=st.vn, n_tokens=N, key=c.key, value=c.value, k_signs=st.ks, k_rnorms=st.kr,
                                   qjl=c.qjl, want_f32=True, want_lse=True)
    mask = torch.ones(1, nodes, N, dtype=torch.bool, device="cuda")
    mask[:, :, N - nodes:] = torch.eye(nodes, device="cuda").bool()
    ref, ref_lse = attend(q, k, v, mask)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3
    w = 2 ** 11 * math.exp(-above) * 20 / 32
    assert ((f32.double() - ref).abs() <= (6e-3 + 2 ** -25 / w) * ref.abs().max()).all()
