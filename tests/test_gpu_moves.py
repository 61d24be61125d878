"""Tokens of packed buffers moved (tq_gather_tokens, tq_keep_tokens) against torch indexing, byte for byte."""

import pytest
import torch

from turboquant.runtime import kernels as K

pytestmark = pytest.mark.gpu


def buffers(B, H, cap, rows, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = [torch.randint(0, 256, (B, H, cap, r), generator=gen, device="cuda", dtype=torch.uint8) for r in rows]
    return out + [torch.randint(0, 2 ** 15, (B, H, cap), generator=gen, device="cuda", dtype=torch.int16).view(torch.float16)]


def raw(t):
    """Bytes [B, H, cap, row] of a buffer."""
    t = t.unsqueeze(-1) if t.dim() == 3 else t
    return t.view(torch.uint8) if t.dtype != torch.uint8 else t


def taken(buf, index, rows=None):
    """torch's gather over [B, H, cap, ...] bytes; index [n], [B, n] or [B, H, n]."""
    x = raw(buf)
    if rows is not None:
        x = x[rows.long()]
    R, H = x.shape[:2]
    while index.dim() < 3:
        index = index.unsqueeze(index.dim() - 1) if index.dim() == 2 else index.expand(R, -1)
    i = index.expand(R, H, -1).long()
    ok = (i >= 0) & (i < x.shape[2])
    y = x.gather(2, i.clamp(0, x.shape[2] - 1)[..., None].expand(-1, -1, -1, x.shape[3]))
    return y.masked_fill(~ok[..., None], 0)


def same(got, ref):
    return torch.equal(raw(got), ref)


ROWS = [48, 16, 64, 62, 47, 3, 2, 1, 17, 256, 15]


@pytest.mark.parametrize("B,H,cap,tokens,capacity", [(1, 1, 1, 1, None), (2, 3, 70, 61, None), (3, 1, 70, 70, 100),
                                                     (1, 2, 5000, 4999, 5003), (2, 2, 9, 0, 4), (2, 8, 1500, 1037, 1500)])
@pytest.mark.parametrize("rows", [None, [1, 0, 0, 1, 2, -1, 5]])
def test_whole_rows(cuda, B, H, cap, tokens, capacity, rows):
    bufs = buffers(B, H, cap, ROWS)
    r = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
    got = K.gather_tokens(bufs, tokens=tokens, rows=r, capacity=capacity)
    slots = tokens if capacity is None else capacity
    R = B if rows is None else len(rows)
    for g, b in zip(got, bufs):
        assert g.shape == (R, H, slots, *b.shape[3:]) and g.dtype == b.dtype
        for i in range(R):
            src = i if rows is None else rows[i]
            if 0 <= src < B:
                assert torch.equal(raw(g)[i, :, :tokens], raw(b)[src, :, :tokens])
                assert (raw(g)[i, :, tokens:] == 0).all()
            else:
                assert (raw(g)[i] == 0).all()


@pytest.mark.parametrize("dims", [1, 2, 3])
@pytest.mark.parametrize("B,H,cap,tokens,n,capacity", [(1, 1, 1, 1, 1, None), (2, 3, 70, 61, 33, None),
                                                       (2, 2, 3000, 2999, 1777, 1900), (1, 4, 40, 33, 90, None),
                                                       (2, 1, 20, 20, 0, 7)])
def test_chosen_tokens(cuda, dims, B, H, cap, tokens, n, capacity):
    bufs = buffers(B, H, cap, ROWS, seed=1)
    shape = (n,) if dims == 1 else (B, n) if dims == 2 else (B, H, n)
    index = torch.randint(0, tokens, shape, generator=torch.Generator().manual_seed(2)).to("cuda")
    if n > 2:  # outside the valid slots: zeros, whatever stands in the slots behind them
        index[..., 1], index[..., 2] = -1, tokens
    got = K.gather_tokens(bufs, tokens=tokens, index=index, capacity=capacity)
    for g, b in zip(got, bufs):
        assert g.shape[2] == (n if capacity is None else capacity)
        ref = taken(b, torch.where(index >= tokens, -1, index))
        x = raw(g)
        assert torch.equal(x[:, :, :n], ref) and (x[:, :, n:] == 0).all()


def test_rows_and_tokens_at_once(cuda):
    bufs = buffers(3, 2, 50, ROWS, seed=3)
    rows = torch.tensor([2, 2, 0, 1], device="cuda")
    index = torch.randint(0, 50, (4, 2, 21), generator=torch.Generator().manual_seed(4), dtype=torch.int32).to("cuda")
    for g, b in zip(K.gather_tokens(bufs, tokens=50, rows=rows, index=index), bufs):
        assert same(g, taken(b, index, rows))


@pytest.mark.parametrize("B,H,first,tokens,n", [(1, 1, 0, 1, 1), (2, 3, 17, 16, 6), (1, 8, 100, 64, 64), (2, 2, 5, 300, 256),
                                                (3, 1, 9, 40, 0)])
@pytest.mark.parametrize("order", ["ascending", "any"])
def test_kept_tokens(cuda, B, H, first, tokens, n, order):
    bufs = buffers(B, H, first + tokens + 3, ROWS, seed=5)
    before = [b.clone() for b in bufs]
    gen = torch.Generator().manual_seed(6)
    index = (torch.stack([torch.randperm(tokens, generator=gen)[:n].sort().values for _ in range(B)]) if order == "ascending"
             else torch.randint(0, tokens, (B, n), generator=gen)).to("cuda")
    if n > 3 and order == "any":
        index[:, 1], index[:, 3] = -5, tokens
    K.keep_tokens(bufs, index, first=first, tokens=tokens)
    for b, old in zip(bufs, before):
        part = old[:, :, first:first + tokens]
        assert same(b[:, :, first:first + n], taken(part, index))
        assert torch.equal(raw(b)[:, :, :first], raw(old)[:, :, :first])
        assert torch.equal(raw(b)[:, :, first + n:], raw(old)[:, :, first + n:])


def test_a_graph_of_both(cuda):
    bufs = buffers(2, 2, 40, ROWS, seed=7)
    start = [b.clone() for b in bufs]
    index, rows = torch.tensor([0, 3, 9], dtype=torch.int32, device="cuda"), torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.keep_tokens(bufs, index, first=20, tokens=16)
        out = K.gather_tokens(bufs, tokens=23, rows=rows)
    for path in ([0, 3, 9], [2, 1, 15], [15, 15, 0]):
        for b, s in zip(bufs, start):
            b.copy_(s)
        index.copy_(torch.tensor(path, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for o, s in zip(out, start):
            ref = raw(s).clone()
            ref[:, :, 20:23] = raw(s)[:, :, [20 + p for p in path]]
            assert torch.equal(raw(o), ref[[1, 1], :, :23])


def test_more_buffers_than_one_launch_takes(cuda):
    bufs = buffers(1, 2, 30, list(range(1, 20)), seed=8)
    index = torch.tensor([4, 7, 29], device="cuda")
    for g, b in zip(K.gather_tokens(bufs, tokens=30, index=index), bufs):
        assert same(g, taken(b, index))
    before = [b.clone() for b in bufs]
    K.keep_tokens(bufs, index, first=0, tokens=30)
    for b, old in zip(bufs, before):
        assert same(b[:, :, :3], taken(old, index))


def test_offsets_past_32_bits(cuda):
    N = 90_000_000
    bufs = buffers(1, 1, 64, [48, 62, 1])
    big = [torch.zeros((1, 2, N, *b.shape[3:]), dtype=b.dtype, device="cuda") for b in bufs]
    for g, b in zip(big, bufs):
        g[:, 1, N - 64:] = b[:, 0]
    index = torch.tensor([60, 3, 3, 0, 63], device="cuda")
    for got, b in zip(K.gather_tokens(big, tokens=N, index=N - 64 + index), bufs):
        assert torch.equal(raw(got)[:, 1:], taken(b, index)) and (raw(got)[:, 0] == 0).all()
    for got, b in zip(K.gather_tokens(big, tokens=N, rows=torch.tensor([0, 0], device="cuda")), bufs):
        assert torch.equal(raw(got)[1, 1, N - 64:], raw(b)[0, 0]) and not raw(got)[1, 0, -1000:].any()
        del got
    K.keep_tokens(big, index, first=N - 64, tokens=64)
    for g, b in zip(big, bufs):
        assert torch.equal(raw(g)[0, 1, N - 64:N - 59], taken(b, index)[0, 0])
        assert torch.equal(raw(g)[0, 1, N - 59:], raw(b)[0, 0, 5:])
