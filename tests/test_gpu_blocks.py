"""Block bounds, block selection and attention over chosen blocks against plain implementations: bounds and selections equal in every
number (infinities, NaN, zeros, subnormal keys, equal scores), attention in 64 bits at block and tile edges, ranges and numbers that name
nothing; the layer's choice kept in step with its tokens, and a run of all three."""

import copy
import math

import numpy as np
import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import block_sparse_attention, fused_attention, share_prefix
from turboquant.runtime import kernels as K
from turboquant.runtime.packed_qmse_cache import BlockChoice
from turboquant.runtime.synthetic import kv_bf16

from ._packed import BITS, D, TOL, arrays, attend64, check, codec, i32, make_layer, randn, rows64

pytestmark = pytest.mark.gpu


def step_of(most):
    """The least 2^e, -100 <= e <= 100, with 127 2^e >= most."""
    e = np.full(most.shape, -100.0)
    for k in range(-99, 101):
        e[127.0 * 2.0 ** (k - 1) < most] = k
    return 2.0 ** e


def bounds_ref(k):
    x = k.double().cpu().numpy()
    x = np.where(np.isnan(x), np.copysign(np.inf, x), x)  # a NaN counts as an infinity of its sign
    cut = np.arange(0, x.shape[2], 64)
    lo, hi = np.minimum.reduceat(x, cut, axis=2), np.maximum.reduceat(x, cut, axis=2)
    step = step_of(np.maximum(-lo, hi).max(-1))
    lohi = np.stack((np.floor(lo / step[..., None]), np.ceil(hi / step[..., None])), -2)
    return np.clip(lohi, -127, 127), step


def bounds(k, cap=None, first=0):
    n = -(-k.shape[2] // 64)
    lohi = torch.full((*k.shape[:2], cap or first + n, 2, D), 77, dtype=torch.int8, device="cuda")
    step = torch.full((*k.shape[:2], cap or first + n), -7.0, device="cuda")
    K.block_bounds(k, lohi, step, first)
    return lohi, step


def same_bounds(k, lohi, step, first=0):
    want, at = bounds_ref(k)
    n = at.shape[-1]
    assert (lohi[:, :, first:first + n].cpu().numpy() == want).all()
    assert (step[:, :, first:first + n].cpu().numpy() == at).all()


@pytest.mark.parametrize("B,H,T,first", [(1, 1, 1, 0), (1, 2, 63, 0), (2, 3, 64, 2), (1, 2, 65, 1), (3, 1, 130, 0), (1, 4, 1000, 5),
                                         (2, 8, 4097, 0)])
def test_bounds(cuda, B, H, T, first):
    k = randn((B, T, H, D), 3).mul(2.0 ** randn((B, T, H, 1), 4).float()).bfloat16().transpose(1, 2)
    n = -(-T // 64)
    lohi, step = bounds(k, first + n + 3, first)
    same_bounds(k, lohi, step, first)
    for t, v in ((lohi, 77), (step, -7.0)):  # the other blocks stay as they were
        assert (t[:, :, :first] == v).all() and (t[:, :, first + n:] == v).all()


def test_bounds_of_special_keys(cuda):
    k = torch.zeros(1, 1, 64 * 12, D, dtype=torch.bfloat16, device="cuda")
    v = k.view(12, 64, D)
    v[1, 5, 3] = math.inf
    v[1, 6, 4] = 2.0
    v[2, 0, 0] = -math.inf
    v[3, 63, 127] = math.nan
    v[3, 1, 2] = -1.0
    v[4, 9, 9] = -torch.tensor(math.nan)  # the sign of a NaN is its bit's
    v[5] = torch.finfo(torch.bfloat16).max
    v[6] = -torch.finfo(torch.bfloat16).max
    v[7, 1, 1] = 2.0 ** -133  # subnormal
    v[8, 2, 2], v[8, 2, 3] = 127.0, -0.5
    v[9, 2, 2], v[9, 2, 3] = 128.0, -128.0  # past 127 steps of 1
    v[10, 2, 2] = 127.0 * 2.0 ** 100 + 0  # the largest there is a step for
    v[11] = -0.0
    lohi, step = bounds(k)
    same_bounds(k, lohi, step)
    assert step[0, 0, 8] == 1.0 and step[0, 0, 9] == 2.0 and step[0, 0, 0] == 2.0 ** -100


def test_bounds_of_numbers_far_below_the_step(cuda):
    """Outward also where a number over the step has no fp32 of its own: behind an infinity, and of finite keys."""
    k = torch.zeros(1, 1, 64 * 5, D, dtype=torch.bfloat16, device="cuda")
    v = k.view(5, 64, D)
    small = 2.0 ** torch.tensor([-40.0, -49, -50, -51, -60, -126, -133], device="cuda")
    for block, largest in enumerate((math.inf, 2.0 ** 31, 2.0 ** 100, 2.0 ** 20, -math.inf)):
        v[block] = 1.0
        v[block, 0, 0] = largest
        v[block, 3, 1:8], v[block, 4, 8:15] = small, -small
        v[block, :, 16:23], v[block, :, 24:31] = small, -small  # nothing else in these channels
        v[block, :, 32], v[block, :, 33] = 0.0, -0.0
    lohi, step = bounds(k)
    same_bounds(k, lohi, step)
    assert (lohi[0, 0, :, 1, 16:23] == 1).all() and (lohi[0, 0, :, 0, 24:31] == -1).all()
    assert (lohi[0, 0, :, :, 32:34] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,T,first", [(1, 1, 1, 0), (1, 2, 63, 0), (2, 3, 64, 2), (1, 2, 65, 1), (2, 4, 1000, 5)])
def test_bounds_of_keys_of_other_types(cuda, dtype, B, H, T, first):
    """Of the keys as given, not of what a rounding to bf16 leaves of them."""
    k = (randn((B, T, H, D), 3, torch.float32) * 2.0 ** randn((B, T, H, 1), 4).float()).to(dtype).transpose(1, 2)
    assert not torch.equal(k, k.bfloat16().to(dtype))
    n = -(-T // 64)
    lohi, step = bounds(k, first + n + 3, first)
    same_bounds(k, lohi, step, first)
    for t, v in ((lohi, 77), (step, -7.0)):  # the other blocks stay as they were
        assert (t[:, :, :first] == v).all() and (t[:, :, first + n:] == v).all()
    wide = torch.zeros(*k.shape[:3], D + 1, dtype=dtype, device="cuda")[..., 1:]  # rows at any element
    wide.copy_(k)
    assert all(torch.equal(a, b) for a, b in zip(bounds(k), bounds(wide)))


def test_bounds_of_special_keys_of_other_types(cuda):
    k = torch.zeros(1, 1, 64 * 10, D, dtype=torch.float16, device="cuda")
    v = k.view(10, 64, D)
    v[0, 3, 5] = 126.0625  # 126 in bf16
    v[1, 5, 3], v[1, 6, 4] = math.inf, 2.0 ** -24
    v[2, 0, 0] = -math.inf
    v[3, 63, 127], v[3, 1, 2] = math.nan, -1.0
    v[4, 9, 9] = -torch.tensor(math.nan)
    v[5], v[6] = 65504.0, -65504.0
    v[7, 1, 1] = -2.0 ** -24  # subnormal
    v[8, 2, 2], v[8, 2, 3] = 127.0, -0.5
    v[9] = -0.0
    for t in (k, k.float()):
        lohi, step = bounds(t)
        same_bounds(t, lohi, step)
        assert lohi[0, 0, 0, 1, 5] == 127 and step[0, 0, 0] == 1.0
    k = torch.zeros(1, 1, 64 * 5, D, device="cuda")
    v = k.view(5, 64, D)
    v[0, 1, 1], v[0, 1, 2] = 2.0 ** -149, -2.0 ** -149
    v[1], v[1, 5] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max
    v[2, 7, 7], v[2, 8, 8], v[2, 9, 9] = 2.0 ** 31, -2.0 ** -126, 2.0 ** -149
    v[3, 7, 7], v[3, 8, 8] = 127.00001, -127.0
    v[4, 0, 0], v[4, 0, 1] = -127.0 * 2.0 ** 100, 1.0 + 2.0 ** -23
    lohi, step = bounds(k)
    same_bounds(k, lohi, step)


def test_bounds_hold_and_arrive_in_any_pieces(cuda):
    k = randn((2, 2, 300, D), 7)
    lohi, step = bounds(k, 5)
    pieces = torch.empty_like(lohi), torch.empty_like(step)
    for first, at, to in ((3, 192, 300), (0, 0, 64), (1, 64, 192)):
        K.block_bounds(k[:, :, at:to], *pieces, first=first)
    assert torch.equal(lohi, pieces[0]) and torch.equal(step, pieces[1])
    low, high = (lohi.float() * step[..., None, None]).unbind(-2)
    at = torch.arange(300, device="cuda") // 64
    assert (k >= low[:, :, at]).all() and (k <= high[:, :, at]).all()


def test_bounds_of_keys_in_any_layout(cuda):
    k = randn((2, 3, 100, D), 9)
    want = bounds(k)
    for other in (k.transpose(1, 2).contiguous().transpose(1, 2), torch.nn.functional.pad(k, (1, 0))[..., 1:], k.float(),
                  k.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)):
        assert all(torch.equal(a, b) for a, b in zip(want, bounds(other)))


# ---------------------------------------------------------------- selection


def select_ref(q, lohi, step, n_tokens, keep, sink, recent, starts=None, lens=None, known=None):
    q, lo, hi = q.double().cpu().numpy(), *(lohi[:, :, :, i].cpu().numpy().astype(np.float64) for i in (0, 1))
    step = step.double().cpu().numpy()
    B, Hq, _ = q.shape
    H, n = step.shape[1:]
    known = n if known is None else known
    out = np.full((B, H, keep), -1)
    for b in range(B):
        end = n_tokens if lens is None else min(max(lens[b], 0), n_tokens)
        start = 0 if starts is None else min(max(starts[b], 0), end)
        first, last = start // 64, -(-end // 64) if end > start else start // 64
        for h in range(H):
            x = np.where(np.isnan(y := q[b, h * Hq // H:(h + 1) * Hq // H]), 0.0, y)
            x = np.clip(np.rint(x / step_of(np.abs(x).max(keepdims=True))), -127, 127)
            score = np.maximum(x[:, None] * lo[b, h], x[:, None] * hi[b, h]).sum(-1).max(0) * step[b, h]
            score[known:] = -np.inf
            fixed = [j for j in range(first, last) if j < first + sink or j >= last - recent]
            rest = sorted(set(range(first, last)) - set(fixed), key=lambda j: (-score[j] if j < n else np.inf, j))
            chosen = sorted((fixed + rest)[:keep])
            out[b, h, :len(chosen)] = chosen
    return torch.from_numpy(out).int()


def index(B, H, N, seed=3):
    k = (randn((B, H, N, D), seed).float() * 2.0 ** randn((B, H, -(-N // 64), 1), seed + 1).float()
         .repeat_interleave(64, 2)[:, :, :N]).bfloat16()
    return bounds(k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,g,N,keep,sink,recent", [(1, 1, 1, 1, 1, 0, 0), (1, 2, 4, 64, 3, 1, 1), (1, 2, 4, 200, 2, 1, 1),
                                                      (2, 2, 7, 1000, 5, 0, 0), (1, 1, 16, 4096, 16, 2, 3),
                                                      (1, 2, 17, 3000, 40, 1, 2), (2, 1, 40, 5000, 1, 0, 1),
                                                      (3, 2, 5, 70000, 128, 1, 2)])
def test_selection(cuda, dtype, B, H, g, N, keep, sink, recent):
    lohi, step = index(B, H, N)
    q = randn((B, H * g, D), 5, dtype)
    got = K.select_blocks(q, lohi, step, n_tokens=N, keep=keep, sink=sink, recent=recent)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), select_ref(q, lohi, step, N, keep, sink, recent))


def test_selection_in_ranges(cuda):
    lohi, step = index(6, 2, 3000)
    q = randn((6, 8, D), 5)
    starts, lens = [0, 100, 2990, 64, -5, 700], [3000, 130, 3000, 1984, 9999, 700]
    got = K.select_blocks(q, lohi, step, n_tokens=3000, keep=6, sink=1, recent=1, seq_starts=i32(starts), seq_lens=i32(lens))
    assert torch.equal(got.cpu(), select_ref(q, lohi, step, 3000, 6, 1, 1, starts, lens))


@pytest.mark.parametrize("keep", [1, 7, 40, 64])
def test_equal_scores_go_by_number(cuda, keep):
    lohi, step = index(1, 2, 64 * 64)
    lohi[:], step[:] = lohi[:, :, :1].clone(), 1.0
    step[:, :, 20::3] = 0.5
    q = randn((1, 8, D), 5)
    got = K.select_blocks(q, lohi, step, n_tokens=64 * 64, keep=keep, sink=0, recent=0)
    assert torch.equal(got.cpu(), select_ref(q, lohi, step, 64 * 64, keep, 0, 0))


def test_queries_at_the_ends_of_their_range(cuda):
    lohi, step = index(5, 1, 64 * 40)
    q = randn((5, 4, D), 5, torch.float32)
    q[0] = 0.0
    q[1, 2, 7] = math.nan
    q[2, 0, 3] = math.inf
    q[3] *= 2.0 ** -120
    q[4] *= 2.0 ** 122
    got = K.select_blocks(q, lohi, step, n_tokens=64 * 40, keep=9, sink=1, recent=1)
    assert torch.equal(got.cpu(), select_ref(q, lohi, step, 64 * 40, 9, 1, 1))


def test_blocks_without_bounds_come_last(cuda):
    lohi, step = index(1, 2, 64 * 20)
    q = randn((1, 8, D), 5)
    for known, keep in ((17, 6), (17, 19), (19, 19)):
        got = K.select_blocks(q, lohi, step, n_tokens=64 * 20, keep=keep, sink=0, recent=3, n_blocks=known)
        assert torch.equal(got.cpu(), select_ref(q, lohi, step, 64 * 20, keep, 0, 3, known=known))


def test_the_most_blocks_chosen_from(cuda):
    n = K.MAX_SCORED
    gen = torch.Generator(device="cuda").manual_seed(3)
    lohi = torch.randint(-127, 128, (1, 1, n, 2, D), generator=gen, device="cuda", dtype=torch.int8).sort(3).values
    step = 2.0 ** torch.randint(-3, 4, (1, 1, n), generator=gen, device="cuda").float()
    q = randn((1, 4, D), 5)
    got = K.select_blocks(q, lohi, step, n_tokens=64 * n, keep=K.MAX_BLOCKS, sink=1, recent=1)
    assert torch.equal(got.cpu(), select_ref(q, lohi, step, 64 * n, K.MAX_BLOCKS, 1, 1))


def test_selection_from_any_layout_of_queries(cuda):
    lohi, step = index(3, 2, 2000)
    q = randn((3, 10, D), 5)
    want = K.select_blocks(q, lohi, step, n_tokens=2000, keep=9)
    assert torch.equal(want, K.select_blocks(q[:, :, None], lohi, step, n_tokens=2000, keep=9))
    rows = torch.zeros(3, 2, 10, D + 1, dtype=torch.bfloat16, device="cuda")[:, 1, :, 1:]
    rows.copy_(q)
    assert torch.equal(want, K.select_blocks(rows, lohi, step, n_tokens=2000, keep=9))
    assert torch.equal(want, K.select_blocks(q.transpose(1, 2).contiguous().transpose(1, 2), lohi, step, n_tokens=2000, keep=9))


# ---------------------------------------------------------------- attention over blocks


def blocks_ref(q, layer, blocks, starts=None, lens=None, scale=None):
    """In 64 bits; a block named twice counts twice."""
    k, v = rows64(layer)
    B, H, n, _ = k.shape
    outs = []
    for b in range(B):
        lo, hi = starts[b] if starts else 0, min(lens[b] if lens else n, n)
        for h in range(H):
            at = [t for j in blocks[b, h].tolist() if j >= 0 for t in range(max(64 * j, lo), min(64 * j + 64, hi))]
            qs = q[b:b + 1, h * q.shape[1] // H:(h + 1) * q.shape[1] // H]
            outs.append(attend64(qs, k[b:b + 1, h:h + 1, at], v[b:b + 1, h:h + 1, at], scale=scale))
    shape = (B, q.shape[1])
    return torch.cat([o for o, _ in outs], 1).view(*shape, D), torch.cat([e for _, e in outs], 1).view(shape)


def some_blocks(B, H, n, keep, seed):
    score = torch.rand(B, H, n, generator=torch.Generator().manual_seed(seed))
    return score.topk(keep, -1).indices.int().cuda()


@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("H,g", [(2, 4), (1, 7)])
def test_every_bit_width(cuda, bits, qjl, H, g):
    layer = make_layer(2, H, 1000, bits, qjl)
    q, blocks = randn((2, H * g, D), 5), some_blocks(2, H, 16, 5, 1)
    got, f32, lse = K.block_attention(q, blocks, **arrays(layer), **codec(layer), n_tokens=1000, want_f32=True, want_lse=True)
    ref, ref_lse = blocks_ref(q, layer, blocks)
    check(got, ref)
    check(f32, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3


@pytest.mark.parametrize("B,H,g,N,keep", [(1, 1, 1, 1, 1), (1, 2, 3, 64, 1), (2, 1, 8, 65, 2), (1, 8, 4, 8195, 129), (3, 2, 5, 700, 4),
                                          (1, 1, 2, 70000, 1000), (40, 8, 1, 300, 3), (1, 1, 6, 2500, 40)])
def test_shapes(cuda, B, H, g, N, keep):
    layer = make_layer(B, H, N, 4, True, seed=3)
    q, blocks = randn((B, H * g, D), 5), some_blocks(B, H, -(-N // 64), keep, 2)
    got = K.block_attention(q, blocks, **arrays(layer), **codec(layer), n_tokens=N)
    check(got, blocks_ref(q, layer, blocks)[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("H,g", [(2, 4), (1, 1), (1, 7), (1, 8)])
def test_queries_of_other_types(cuda, dtype, bits, qjl, H, g):
    """Queries that are no bf16 numbers are not rounded to them, and outputs are in their type."""
    layer = make_layer(2, H, 1000, bits, qjl, seed=25)
    q = randn((2, H * g, D), 5, torch.float32).to(dtype)
    assert not torch.equal(q, q.bfloat16().to(dtype))
    blocks = some_blocks(2, H, 16, 5, 1)
    kw = dict(**arrays(layer), **codec(layer), n_tokens=1000)
    got, f32, lse = K.block_attention(q, blocks, **kw, want_f32=True, want_lse=True)
    assert got.dtype == dtype and f32.dtype == torch.float32
    ref, ref_lse = blocks_ref(q, layer, blocks)
    check(got, ref)
    check(f32, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3
    rows = torch.zeros(2, 3, H * g, D + 1, dtype=dtype, device="cuda")[:, 1, :, 1:]  # rows at any element
    rows.copy_(q)
    assert torch.equal(K.block_attention(rows, blocks, **kw), got)
    assert torch.equal(K.block_attention(q[:, :, None], blocks, **kw), got)
    exact = q.bfloat16()  # numbers that every type has
    want = K.block_attention(exact, blocks, **kw, want_f32=True)[1]
    assert torch.equal(K.block_attention(exact.to(dtype), blocks, **kw, want_f32=True)[1], want)  # the other terms add zeros


@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("size", [1.0, 1e-3])
@pytest.mark.parametrize("g", [4, 7])
def test_fp32_queries_lose_little_to_fp16_values(cuda, bits, qjl, size, g):
    """Of the output's norm: values' centroids up to 1.5e-4, weights times norms up to 2^-11 / sqrt 3 = 2.8e-4: 3.2e-4 together.  With queries of a
    thousandth all tokens weigh the same, the values nearly cancel, and the centroids' mean error would be what is left."""
    layer = make_layer(1, 2, 16384, bits, qjl, seed=27)
    q = randn((1, 2 * g, D), 5, torch.float32) * size
    every = torch.arange(256, dtype=torch.int32, device="cuda").expand(1, 2, 256)
    got = K.block_attention(q, every, **arrays(layer), **codec(layer), n_tokens=16384)
    ref, _ = attend64(q, *rows64(layer))
    assert (got.double() - ref).norm() <= 3.3e-4 * ref.norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("dense", [0, 30])
@pytest.mark.parametrize("g", [4, 7])
def test_layers_take_queries_of_other_types(cuda, dtype, dense, g):
    layer = make_layer(2, 2, 1500, 4, True, seed=15, dense=dense)
    q = randn((2, 2 * g, 1, D), 5, torch.float32).to(dtype)
    got = block_sparse_attention(q, layer, keep=6)
    assert got.shape == q.shape and got.dtype == dtype
    check(got, sparse_ref(q, layer, 6, 1, 2))
    empty = K.block_attention(q, torch.empty(2, 2, 0, dtype=torch.int32, device="cuda"), **arrays(layer), **codec(layer), n_tokens=1500)
    assert empty.dtype == dtype and (empty == 0).all()


def test_the_most_blocks(cuda):
    """As many as are taken, each of them of a short history and many times: like once."""
    layer = make_layer(1, 1, 130, 4, True, seed=5)
    q = randn((1, 8, D), 5)
    every = torch.arange(3, dtype=torch.int32, device="cuda").repeat(1, 1, K.MAX_BLOCKS // 3)
    got = K.block_attention(q, every, **arrays(layer), **codec(layer), n_tokens=130)
    k, v = rows64(layer)
    check(got, attend64(q, k, v)[0])


def test_every_block_is_decode_attention(cuda):
    layer = make_layer(2, 2, 1000, 4, True, seed=7)
    q = randn((2, 8, 1, D), 5)
    every = torch.arange(16, dtype=torch.int32, device="cuda").expand(2, 2, 16)
    kw = dict(**arrays(layer), **codec(layer), n_tokens=1000, seq_starts=i32([0, 70]), seq_lens=i32([1000, 901]))
    check(K.block_attention(q, every, **kw), K.decode_attention(q, **kw).double(), 2 * TOL)


def test_ranges_and_numbers_that_name_nothing(cuda):
    layer = make_layer(4, 2, 500, 3, False, seed=9)
    q = randn((4, 8, D), 5)
    blocks = i32([[[0, 7, -1, 3], [5, 5, 99, 1]], [[2, 1, 0, -1], [1, 1, 1, 1]], [[-1, -1, -1, -1], [1 << 30, -(1 << 31), 7, -7]],
                  [[7, 6, 5, 4], [0, 1, 2, 3]]])
    starts, lens = [0, 70, 0, 0], [500, 131, 500, 200]
    for name in ("kn", "vn"):  # what is not attended to may be anything
        getattr(layer._store, name)[1, :, :70] = math.nan
        getattr(layer._store, name)[1, :, 131:] = math.inf
        getattr(layer._store, name)[3, :, 200:] = math.nan
    got, lse = K.block_attention(q, blocks, **arrays(layer), **codec(layer), n_tokens=500, seq_starts=i32(starts),
                                 seq_lens=i32(lens), want_lse=True)
    k, v = rows64(layer)
    ref, ref_lse = blocks_ref(q, layer, torch.where((blocks >= 0) & (blocks < 8), blocks, -1), starts, lens)
    check(got, ref)
    some = torch.isfinite(ref_lse)
    assert (lse.double() - ref_lse)[some].abs().max() <= 4e-3
    assert (lse[~some] == -math.inf).all() and (got[~some] == 0).all() and not some[2, :4].any() and not some[3, :4].any()
    got, lse = K.block_attention(q, blocks[..., :0], **arrays(layer), **codec(layer), n_tokens=500, want_lse=True)
    assert (got == 0).all() and (lse == -math.inf).all()


def test_a_cache_past_32_bits(cuda):
    """Codes of a KV head that begin past 2^32 bytes of their buffer."""
    layer = make_layer(1, 2, 200, 4, False, seed=11)
    cap = (1 << 24) - 1  # 64 bytes a slot: 1 GB a head
    H = 5
    big = {}
    for name, t in arrays(layer).items():
        if t is None:
            big[name] = None
            continue
        big[name] = torch.empty(1, H, cap, *t.shape[3:], dtype=t.dtype, device="cuda")
        big[name][:, H - 1, 1 << 23:(1 << 23) + 200] = t[:, 0, :200]
    q = randn((1, H * 2, D), 5)
    blocks = i32([[[-1] * 4] * (H - 1) + [[(1 << 17) + j for j in range(4)]]])
    got = K.block_attention(q, blocks, **big, **codec(layer), n_tokens=(1 << 23) + 200)
    k, v = rows64(layer)
    assert (got[:, :-2] == 0).all()
    check(got[:, -2:], attend64(q[:, -2:], k[:, :1], v[:, :1])[0])


def test_streams_and_captured_calls(cuda):
    """A run of the three, captured and replayed with other queries and ranges, beside one on another stream."""
    layer = make_layer(2, 2, 3000, 4, True, seed=13)
    rows = layer._key_rows(0, 3000)
    q, lens = randn((2, 8, D), 5), i32([3000, 3000])
    lohi = torch.empty(2, 2, 47, 2, D, dtype=torch.int8, device="cuda")
    step = torch.empty(2, 2, 47, device="cuda")

    def run():
        K.block_bounds(rows, lohi, step)
        blocks = K.select_blocks(q, lohi, step, n_tokens=3000, keep=8, seq_lens=lens)
        return blocks, K.block_attention(q, blocks, **arrays(layer), **codec(layer), n_tokens=3000, seq_lens=lens)

    run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i, n in enumerate(([3000, 3000], [1700, 64], [0, 2999])):
        lens.copy_(i32(n))
        q.copy_(randn(q.shape, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))
        assert torch.equal(out[0].cpu(), select_ref(q, lohi, step, 3000, 8, 1, 1, lens=n))
        check(out[1], blocks_ref(q, layer, out[0], lens=n)[0])


# ---------------------------------------------------------------- the layer


def sparse_ref(q, layer, keep, sink, recent):
    """A decode step by the formula: bounds of the decoded rows, the choice, attention in 64 bits over it and the dense tokens."""
    n = layer.packed_seq_length()
    rows = layer._key_rows(0, n)
    want, at = bounds_ref(rows)
    lohi, step = torch.from_numpy(want).cuda(), torch.from_numpy(at).cuda()
    q = q[:, :, 0]
    blocks = select_ref(q, lohi, step, n, keep, sink, recent).cuda()
    k, v = rows64(layer)
    slot = torch.arange(n, device="cuda") // 64
    mask = (slot[None, None, :, None] == blocks[:, :, None]).any(-1)
    if layer._dense_len:
        k, v = torch.cat((k, layer._dense_keys.double()), 2), torch.cat((v, layer._dense_values.double()), 2)
        mask = torch.nn.functional.pad(mask, (0, layer._dense_len), value=True)
    return attend64(q, k, v, mask)[0][:, :, None]


@pytest.mark.parametrize("bits,qjl,dense", [(4, True, 0), (3, False, 0), (4, True, 30)])
@pytest.mark.parametrize("g", [4, 7])
def test_block_sparse_attention(cuda, bits, qjl, dense, g):
    layer = make_layer(2, 2, 1500, bits, qjl, seed=15, dense=dense)
    for dtype in (torch.bfloat16, torch.float32):
        q = randn((2, 2 * g, 1, D), 5).to(dtype)
        got = block_sparse_attention(q, layer, keep=6)
        assert got.shape == q.shape and got.dtype == dtype
        check(got, sparse_ref(q, layer, 6, 1, 2))
    few = make_layer(2, 2, 300, bits, qjl, seed=15, dense=dense)
    assert torch.equal(block_sparse_attention(q, few, keep=6), fused_attention(q, few, g))  # no more blocks than that


def test_a_layer_told_to_attend_to_blocks(cuda):
    """The bounds follow the layer's tokens: appended, taken back, chosen and moved between rows."""
    layer = make_layer(2, 2, 700, 4, True, seed=17, reserve_tokens=64)
    layer.attend_blocks(5, sink=1, recent=1)

    def agree(seed):
        q = randn((layer._batch(), 8, 1, D), seed)
        check(fused_attention(q, layer, 4), sparse_ref(q, layer, 5, 1, 1))

    agree(1)
    for i in range(4):
        k, v = kv_bf16((2, 2, 90, D), seed=60 + i), kv_bf16((2, 2, 90, D), seed=70 + i)
        layer.update(k, v)
        agree(2 + i)
    assert layer._bounds.count == 1060 // 64
    layer.reorder_cache(torch.tensor([1, 1], device="cuda"))
    agree(10)
    layer.batch_repeat_interleave(2)
    agree(11)
    layer.crop(-200)
    assert layer._bounds.count == 860 // 64
    k, v = kv_bf16((4, 2, 200, D), seed=80), kv_bf16((4, 2, 200, D), seed=81)
    layer.update(k, v)
    agree(12)
    layer.keep_tokens(torch.tensor([5, 1, 60], device="cuda"), tokens=100)
    agree(13)
    layer.keep_tokens(torch.arange(0, layer.packed_seq_length(), 2, device="cuda"))
    agree(14)
    layer.batch_select_indices(torch.tensor([2, 0], device="cuda"))
    agree(15)
    layer.attend_blocks(None)
    q = randn((2, 8, 1, D), 16)
    k, v = rows64(layer)
    check(fused_attention(q, layer, 4), attend64(q[:, :, 0], k, v)[0][:, :, None])


def test_left_padding(cuda):
    layer = make_layer(2, 2, 900, 4, True, seed=19)
    mask = torch.ones(2, 900, dtype=torch.bool, device="cuda")
    mask[1, :333] = False
    q = randn((2, 8, 1, D), 5)
    got = block_sparse_attention(q, layer, 4, sink=1, recent=1, attention_mask=mask)
    lohi, step, known = layer.block_bounds()
    blocks = select_ref(q[:, :, 0], lohi[:, :, :known], step[:, :, :known], 900, 4, 1, 1, [0, 333], [900, 900])
    check(got, blocks_ref(q[:, :, 0], layer, blocks, [0, 333], [900, 900])[0][:, :, None])
    mask[0, 100:120] = False
    with pytest.raises(ValueError):
        block_sparse_attention(q, layer, 4, attention_mask=mask)


def test_captured_steps_with_a_mask(cuda):
    """Every replay finds the mask's ranges anew, also where an eager step has had them."""
    layer = make_layer(2, 2, 900, 4, True, seed=19)
    layer.attend_blocks(4, sink=1, recent=1)
    layer._tq_mask_contiguous = True
    mask, q = torch.ones(2, 900, dtype=torch.bool, device="cuda"), randn((2, 8, 1, D), 5)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        q.add_(0.0)
        with pytest.raises(ValueError, match="block_bounds"):
            fused_attention(q, layer, 4, mask)
    assert layer._bounds is None
    lohi, step, known = (t[:, :, :900 // 64] if torch.is_tensor(t) else t for t in layer.block_bounds())
    fused_attention(q, layer, 4, mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_attention(q, layer, 4, mask)
    for start in (0, 100, 333):
        mask[1, :start] = False
        graph.replay()
        torch.cuda.synchronize()
        blocks = select_ref(q[:, :, 0], lohi, step, 900, 4, 1, 1, [0, start], [900, 900])
        check(out, blocks_ref(q[:, :, 0], layer, blocks, [0, start], [900, 900])[0][:, :, None])
        check(fused_attention(q, layer, 4, mask), out.double(), 2 * TOL)


def test_a_model_attending_to_blocks(cuda):
    """Every block kept: the logits of full attention; few kept: finite, and other ones."""
    from turboquant.adapters.transformers import disable_turboquant_attention, enable_turboquant_attention
    from turboquant.runtime.packed_qmse_cache import build_packed_mse_cache

    from ._tiny_model import tiny_llama

    model = tiny_llama("cuda", torch.bfloat16, layers=2, heads=8, kv_heads=2)
    ids = torch.randint(0, 94, (1, 500), generator=torch.Generator().manual_seed(3)).cuda()
    logits = {}
    for keep in (None, 8, 3):
        with torch.no_grad():
            cache = build_packed_mse_cache(model(input_ids=ids, use_cache=True).past_key_values, bits=4, use_qjl_keys=True,
                                           quantize_decode=True, norm_guard=False)
            for layer in cache.layers:
                layer.attend_blocks(keep, recent=1)
            old = enable_turboquant_attention(model, cache)
            logits[keep] = torch.cat([model(input_ids=ids[:, i:i + 1], past_key_values=cache, use_cache=True).logits.float()
                                      for i in range(4)], 1)
            disable_turboquant_attention(model, cache, old)
    assert torch.equal(logits[None], logits[8])
    assert torch.isfinite(logits[3]).all() and not torch.equal(logits[3], logits[8])


def test_choices_that_are_none():
    for bad in ((2, 1, 2), (5, -1, 1), (5, 1, 0), (K.MAX_BLOCKS + 1, 1, 1)):
        with pytest.raises(ValueError):
            BlockChoice(*bad)


@pytest.mark.parametrize("cap", [0, 130])
def test_histories_without_tokens(cuda, cap):
    layer = make_layer(2, 2, 130, 4, True)
    cache = {name: t[:, :, :cap].contiguous() for name, t in arrays(layer).items()}
    q, blocks = randn((2, 8, D), 5), torch.arange(3, dtype=torch.int32, device="cuda").expand(2, 2, 3)
    got, lse = K.block_attention(q, blocks, **cache, **codec(layer), n_tokens=0, want_lse=True)
    assert (got == 0).all() and (lse == -math.inf).all()
    bounds = torch.zeros(2, 2, cap // 64, 2, D, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, cap // 64, device="cuda")
    assert (K.select_blocks(q, *bounds, n_tokens=0, keep=4) == -1).all()
    before = [t.clone() for t in bounds]
    K.block_bounds(torch.empty(2, 2, 0, D, dtype=torch.bfloat16, device="cuda"), *bounds)
    assert all(torch.equal(a, b) for a, b in zip(bounds, before))


def test_bounds_past_32_bits(cuda):
    """Bounds of a KV head that begin past 2^32 bytes of their buffer: as of a small one."""
    rows, q = randn((1, 5, 700, D), 3), randn((1, 10, D), 4)
    cap = 1 << 22  # 256 bytes a block: 1 GB a head
    both = [(torch.empty(1, 5, n, 2, D, dtype=torch.int8, device="cuda"), torch.empty(1, 5, n, device="cuda")) for n in (11, cap)]
    for lohi, step in both:
        K.block_bounds(rows, lohi, step)
    assert torch.equal(both[0][0], both[1][0][:, :, :11]) and torch.equal(both[0][1], both[1][1][:, :, :11])
    chosen = [K.select_blocks(q, *b, n_tokens=700, keep=4, n_blocks=11) for b in both]
    assert torch.equal(*chosen) and torch.equal(chosen[0].cpu(), select_ref(q, *both[0], 700, 4, 1, 1))


def test_bounds_that_another_stream_makes(cuda):
    """A step on a stream that waits for the tokens alone attends to the same blocks as the step that makes the bounds, which is
    still held up on its own stream."""
    layer = make_layer(2, 2, 1500, 4, True, seed=21, reserve_tokens=64)
    q, choice = randn((2, 8, 1, D), 5), BlockChoice(5, 1, 1)
    streams = [torch.cuda.Stream() for _ in range(2)]

    def want():
        n = layer.packed_seq_length()
        lohi, step = (torch.from_numpy(t).cuda() for t in bounds_ref(layer._key_rows(0, n)))
        return select_ref(q[:, :, 0], lohi, step, n, 5, 1, 1)

    lohi, step, _ = layer.block_bounds()
    lohi.zero_(), step.zero_()  # bounds by which the first blocks would be chosen
    layer._forget_bounds(0)
    for i in range(3):
        torch.cuda.synchronize()
        got = []
        for s, held_up in ((streams[i % 2], 10_000_000), (streams[1 - i % 2], 0)):
            with torch.cuda.stream(s):
                if held_up:
                    torch.cuda._sleep(held_up)
                got.append(layer.choose_blocks(q, choice))
        got.append(layer.choose_blocks(q, choice))
        torch.cuda.synchronize()
        assert all(torch.equal(g.cpu(), want()) for g in got)
        layer.update(*(kv_bf16((2, 2, 700, D), seed=90 + 2 * i + j) for j in range(2)))  # the buffers grow
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(10_000_000)
        layer.choose_blocks(q, choice)
    with torch.cuda.stream(streams[1]):  # a copy is the stream's that makes it
        other = copy.deepcopy(layer)
        got = other.choose_blocks(q, choice)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), want())


@pytest.mark.parametrize("known", [None, False])
def test_masks_with_a_hole_are_attended_to_in_full(cuda, known):
    """By a model's step; the call for one step over blocks refuses them."""
    from turboquant.runtime.attention import turboquant_attention_forward, turboquant_prompt_forward

    layer = make_layer(2, 2, 900, 4, True, seed=23)
    layer.attend_blocks(4, sink=1, recent=1)
    if known is not None:
        layer._tq_mask_contiguous = known
    module = torch.nn.Module()
    module._tq_cache_layer, module.num_key_value_groups = layer, 4
    mask = torch.ones(2, 900, dtype=torch.bool, device="cuda")
    mask[1, 700:880] = False
    q = randn((2, 8, 1, D), 5)
    want, _ = attend64(q[:, :, 0], *rows64(layer), mask[:, None])
    assert fused_attention(q, layer, 4, mask) is None
    for forward in (turboquant_attention_forward, turboquant_prompt_forward):
        got, _ = forward(module, q, None, None, mask[:, None, None])
        check(got[:, 0], want, 2e-2)  # bf16 rows and weights: 2^-8 of the logits' terms and of the values
    with pytest.raises(ValueError, match="one range"):
        block_sparse_attention(q, layer, 4, attention_mask=mask)


def test_bounds_are_counted_among_a_layers_bytes(cuda):
    from turboquant.runtime.packed_qmse_cache import packed_cache_storage_bytes

    layer = make_layer(2, 3, 1000, 4, True)
    before = layer.storage_bytes()
    layer.block_bounds()
    assert layer.storage_bytes() - before == 2 * 3 * 15 * (2 * D + 4)
    layer.crop(-200)
    one = layer.storage_bytes()
    assert one == before * 800 // 1000 + 2 * 3 * 12 * (2 * D + 4)
    shared = share_prefix(Cache(layers=[layer]), 2)
    assert packed_cache_storage_bytes(shared) == one
