"""Attention of a tree of drafted tokens over a packed layer (tq_tree_attention) against the fp64 formula: every bit
width, tile and split edges, grouped heads, ragged histories, masks by parents, norms at the ends of their range, and
the layer's route with dense tokens, split layers and wide trees."""

import math

import pytest
import torch

from turboquant.runtime import kernels as K
from turboquant.runtime import tree_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16

pytestmark = pytest.mark.gpu

D = 128


def randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def make_layer(B, Hkv, N, bits, qjl, seed=0, outliers=0, dense=0):
    k, v = kv_bf16((B, Hkv, N + dense, D), seed=seed), kv_bf16((B, Hkv, N + dense, D), seed=seed + 1)
    layer = PackedMSELayer(bits=bits, use_qjl_keys=qjl, num_outlier_channels=outliers, quantize_decode=dense == 0)
    layer.initialize_from_dense(k[:, :, :N], v[:, :, :N])
    layer._lazy_update = True
    if dense:
        layer.update(k[:, :, N:], v[:, :, N:])
    return layer


def unpack(rows, bits, n):
    at = torch.arange(n, device="cuda") * bits
    wide = torch.nn.functional.pad(rows, (0, 1)).int()
    return (((wide[..., at // 8] | (wide[..., at // 8 + 1] << 8)) >> (at % 8)) & ((1 << bits) - 1)).long()


def rows64(layer):
    """Keys and values [B, H, n, D] of a one-group layer in 64 bits."""
    st, c, n = layer._store, layer.codecs, layer.packed_seq_length()
    k = c.key.centers.double()[unpack(st.kc[:, :, :n], c.key_bits, D)] @ c.key.rotation.double()
    k = k * st.kn[:, :, :n].double()[..., None]
    if c.qjl is not None:
        pm = 2.0 * unpack(st.ks[:, :, :n], 1, D).double() - 1.0
        k = k + (pm @ c.qjl.double()) * st.kr[:, :, :n].double()[..., None] * (math.sqrt(math.pi / 2) / D)
    v = c.value.centers.double()[unpack(st.vc[:, :, :n], c.value_bits, D)] @ c.value.rotation.double()
    return k, v * st.vn[:, :, :n].double()[..., None]


def tree_mask(parents, total, starts, ends):
    """[B, T, total]; parents a list per batch row."""
    m = torch.zeros(len(parents), len(parents[0]), total, dtype=torch.bool)
    for b, row in enumerate(parents):
        m[b, :, starts[b]:ends[b]] = True
        for i in range(len(row)):
            j = i
            while True:
                if ends[b] + j < total:
                    m[b, i, ends[b] + j] = True
                if not 0 <= row[j] < j:
                    break
                j = row[j]
    return m.cuda()


def attend(q, k, v, mask, scale=None):
    """fp64 output and log-sum-exp; nodes without tokens are 0."""
    g = q.shape[1] // k.shape[1]
    x = q.double() @ k.repeat_interleave(g, 1).transpose(-1, -2) * (scale or 1.0 / math.sqrt(D))
    if mask is not None:
        x = x.masked_fill(~mask[:, None], float("-inf"))
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
    return p @ v.repeat_interleave(g, 1), lse


def random_tree(T, seed):
    gen = torch.Generator().manual_seed(seed)
    return [-1 if i < 3 else int(torch.randint(-1, i, (1,), generator=gen)) for i in range(T)]


#: Roundings of the kernel, all independent of each other, each to fp16: by at most 2^-11 of the number, 2^-11 / sqrt(3) =
#: 2.8e-4 root mean square.  A logit is a sum of 128 products of a rotated query element and a centroid, both rounded: its error is of the
#: order |q| |k| / sqrt(128) * sqrt(2) * 2.8e-4 / sqrt(128) (|q| 11.3 or less than twice that, |k| about 20 and rarely twice
#: that) = 11.3 * 20 / 128 * 1.4 * 2.8e-4 = 7e-4, with the QJL part as much again; value centroids and weights 2.8e-4 each.
#: Of the output's largest element that is 2e-3 at most, the package's tolerance of its other decode kernels; a bf16
#: output adds half a step, 2^-8 of the element.
TOL = 2e-3


def check(got, ref, tol=TOL):
    assert torch.isfinite(got).all()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    assert ((got.double() - ref).abs() <= tol * ref.abs().max() + 2 * half * ref.abs()).all()


BITS = [(4, True), (3, True), (2, True), (4, False), (3, False), (2, False), (1, False)]


@pytest.mark.parametrize("bits,qjl", BITS)
@pytest.mark.parametrize("B,Hkv,g,N,T", [(1, 2, 4, 100, 8), (2, 1, 7, 517, 20)])
def test_every_bit_width(cuda, bits, qjl, B, Hkv, g, N, T):
    layer = make_layer(B, Hkv, N + T, bits, qjl)
    q = randn((B, T, Hkv * g, D), 5).transpose(1, 2)
    parents = random_tree(T, 1)
    got = tree_attention(q, layer, torch.tensor(parents), g)
    ref, _ = attend(q, *rows64(layer), tree_mask([parents] * B, N + T, [0] * B, [N] * B))
    assert got.shape == q.shape and got.dtype == q.dtype
    check(got, ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hkv,g,N,T", [(1, 1, 1, 0, 1), (1, 2, 3, 1, 1), (2, 2, 4, 55, 8), (1, 2, 5, 63, 1),
                                         (1, 1, 4, 64, 2), (2, 1, 8, 127, 33), (1, 4, 4, 2000, 64), (1, 2, 16, 700, 11),
                                         (1, 1, 12, 4100, 5), (3, 2, 1, 300, 31)])
def test_shapes_and_types(cuda, dtype, B, Hkv, g, N, T):
    layer = make_layer(B, Hkv, N + T, 4, True, seed=3)
    q = randn((B, Hkv * g, T, D), 5, dtype)
    parents = [random_tree(T, b) for b in range(B)]
    st, c = layer._store, layer.codecs
    got, f32, lse = K.tree_attention(q, torch.tensor(parents, device="cuda"), k_codes=st.kc, k_norms=st.kn, v_codes=st.vc,
                                     v_norms=st.vn, n_tokens=N + T, key=c.key, value=c.value, k_signs=st.ks,
                                     k_rnorms=st.kr, qjl=c.qjl, want_f32=True, want_lse=True)
    ref, ref_lse = attend(q, *rows64(layer), tree_mask(parents, N + T, [0] * B, [N] * B))
    assert got.dtype == dtype
    check(got, ref)
    check(f32, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3


def test_a_long_history_and_many_splits(cuda):
    layer = make_layer(1, 2, 33000, 4, True, seed=7)
    q = randn((1, 8, 6, D), 5)
    parents = [-1, 0, 0, 1, -1, 4]
    got = tree_attention(q, layer, torch.tensor(parents), 4)
    ref, _ = attend(q, *rows64(layer), tree_mask([parents], 33000, [0], [32994]))
    check(got, ref)


def test_ragged_histories(cuda):
    B, N, T = 6, 600, 7
    layer = make_layer(B, 2, N, 3, False, seed=9)
    q = randn((B, 6, T, D), 5)
    parents = [random_tree(T, b) for b in range(B)]
    starts, lens = [0, 100, 590, 0, 64, 5], [593, 200, 590, 0, 65, 597]  # the last: some nodes past the stored slots
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = tree_attention(q, layer, torch.tensor(parents), 3, seq_starts=i32(starts), seq_lens=i32(lens))
    ref, _ = attend(q, *rows64(layer), tree_mask(parents, N, starts, lens))
    for b in range(B - 1):
        check(got[b], ref[b])
    seen = [i for i in range(T) if lens[-1] + i < N]
    check(got[-1][:, seen], ref[-1][:, seen])


def test_history_alone_and_nothing_at_all(cuda):
    layer = make_layer(2, 2, 200, 4, True, seed=11)
    q = randn((2, 8, 5, D), 5)
    st, c = layer._store, layer.codecs
    kw = dict(k_codes=st.kc, k_norms=st.kn, v_codes=st.vc, v_norms=st.vn, n_tokens=200, key=c.key, value=c.value,
              k_signs=st.ks, k_rnorms=st.kr, qjl=c.qjl, want_lse=True)
    lens = torch.tensor([200, 150], device="cuda")
    mask = torch.arange(200, device="cuda")[None, None, :] < lens[:, None, None]
    got, lse = K.tree_attention(q, None, seq_lens=lens, **kw)
    ref, ref_lse = attend(q, *rows64(layer), mask.expand(2, 5, 200))
    check(got, ref)
    assert (lse.double() - ref_lse).abs().max() <= 4e-3
    got, lse = K.tree_attention(q, None, seq_lens=torch.tensor([0, 30], device="cuda"),
                                seq_starts=torch.tensor([0, 40], device="cuda"), **kw)
    assert (got == 0).all() and (lse == float("-inf")).all()


def test_parents_that_are_no_earlier_node_are_none(cuda):
    layer = make_layer(1, 1, 80, 4, True, seed=13)
    q = randn((1, 4, 6, D), 5)
    odd, plain = [-7, 1, 5, 2, 1 << 30, 4], [-1, -1, -1, 2, -1, 4]
    a, b = (tree_attention(q, layer, torch.tensor(p), 4) for p in (odd, plain))
    assert torch.equal(a, b)


def test_a_chain_is_causal_and_a_node_alone_is_a_decode_step(cuda):
    layer = make_layer(2, 2, 150, 4, True, seed=15)
    q = randn((2, 8, 4, D), 5)
    chain = tree_attention(q, layer, torch.tensor([-1, 0, 1, 2]), 4)
    st, c = layer._store, layer.codecs
    for i in range(4):
        one = K.decode_attention(q[:, :, i:i + 1].contiguous(), k_codes=st.kc, k_norms=st.kn, v_codes=st.vc, v_norms=st.vn,
                                 n_tokens=147 + i, key=c.key, value=c.value, k_signs=st.ks, k_rnorms=st.kr, qjl=c.qjl)
        check(chain[:, :, i], one.double(), 2 * TOL)


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 3e4])
def test_norms_at_the_ends_of_their_range(cuda, size):
    """Value norms from subnormal to 60000, growing along the history: the output sums' unit rises on the way."""
    layer = make_layer(1, 2, 400, 4, True, seed=17)
    ramp = torch.linspace(1e-3 if size > 1e-3 else 1.0, 2.0, 400, device="cuda")
    layer._store.vn[:, :, :400] = (size * ramp).half()
    q = randn((1, 8, 3, D), 5, torch.float32)
    got = tree_attention(q, layer, torch.tensor([-1, 0, 1]), 4)
    ref, _ = attend(q, *rows64(layer), tree_mask([[-1, 0, 1]], 400, [0], [397]))
    check(got, ref)


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e30])
def test_queries_of_any_size(cuda, size):
    layer = make_layer(1, 2, 200, 4, True, seed=19)
    q = randn((1, 4, 3, D), 5, torch.float32) * size
    scale = 1.0 / math.sqrt(D) / size
    st, c = layer._store, layer.codecs
    got = K.tree_attention(q, torch.tensor([-1, 0, 1], device="cuda"), k_codes=st.kc, k_norms=st.kn, v_codes=st.vc,
                           v_norms=st.vn, n_tokens=200, key=c.key, value=c.value, k_signs=st.ks, k_rnorms=st.kr,
                           qjl=c.qjl, scale=scale)
    ref, _ = attend(q, *rows64(layer), tree_mask([[-1, 0, 1]], 200, [0], [197]), scale)
    check(got, ref)


def test_left_out_tokens_may_hold_anything(cuda):
    layer = make_layer(1, 2, 100, 4, True, seed=21)
    st = layer._store
    q = randn((1, 8, 3, D), 5)
    parents = torch.tensor([-1, 0, -1])
    clean = tree_attention(q, layer, parents, 4)
    for n in (st.kn, st.kr, st.vn):
        n[:, :, 98] = float("nan")  # node 1, seen by itself only
        n[:, :, 100:] = float("nan")
    got = tree_attention(q, layer, parents, 4)
    assert torch.equal(got[:, :, [0, 2]], clean[:, :, [0, 2]]) and got[:, :, 1].isnan().all()
    q[0, 3, 2] = float("nan")
    got = tree_attention(q, layer, parents, 4)
    assert got[0, 3, 2].isnan().all() and torch.equal(got[0, [0, 1, 2, 4, 5, 6, 7]][:, [0, 2]], clean[0, [0, 1, 2, 4, 5, 6, 7]][:, [0, 2]])


@pytest.mark.parametrize("case", ["dense", "dense fp32", "split", "wide", "one node of many"])
def test_the_layers_other_routes(cuda, case):
    """Dense nodes, layers in two channel groups, more nodes than the kernel takes."""
    T = 70 if case == "wide" else 6
    if case.startswith("dense"):
        layer = make_layer(2, 2, 300, 4, True, seed=23, dense=T + 5)
        k, v = rows64(layer)
        k, v = (torch.cat((a, b.double()), 2) for a, b in ((k, layer._dense_keys), (v, layer._dense_values)))
    else:
        layer = make_layer(2, 2, 300, 4, True, seed=23, outliers=4 if case == "split" else 0)
        # the chunked path attends to the decoder's bf16 rows, the packed one to the codes
        k, v = rows64(layer) if case == "one node of many" else (layer._decode_keys_full().double(),
                                                                layer._decode_values_full().double())
    q = randn((2, 8, T, D), 5, torch.float32 if case == "dense fp32" else torch.bfloat16)
    parents = [random_tree(T, b) for b in range(2)]
    starts = [0, 40]
    got = tree_attention(q, layer, torch.tensor(parents), 4, seq_starts=torch.tensor(starts, device="cuda"))
    total = k.shape[2]
    ref, _ = attend(q, k, v, tree_mask(parents, total, starts, [total - T] * 2))
    assert got.dtype == q.dtype
    check(got, ref)


def test_replays_of_a_graph_and_other_streams(cuda):
    layer = make_layer(2, 2, 700, 4, True, seed=25)
    q, parents = randn((2, 8, 9, D), 5), torch.tensor(random_tree(9, 0), dtype=torch.int32, device="cuda")
    tree_attention(q, layer, parents, 4)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tree_attention(q, layer, parents, 4)
    for seed in (31, 32, 33):
        q.copy_(randn(q.shape, seed))
        parents.copy_(torch.tensor(random_tree(9, seed), dtype=torch.int32))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            again = tree_attention(q, layer, parents, 4)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, again)


def test_refusals(cuda):
    layer = make_layer(1, 2, 20, 4, True)
    q = randn((1, 8, 4, D), 5)
    with pytest.raises(ValueError, match="parents"):
        tree_attention(q, layer, torch.tensor([-1, 0]), 4)
    with pytest.raises(ValueError, match="drafted"):
        tree_attention(randn((1, 8, 21, D), 5), layer, torch.full((21,), -1), 4)
    with pytest.raises(ValueError, match="backward"):
        tree_attention(q.requires_grad_(), layer, torch.tensor([-1, 0, 1, 2]), 4)


@pytest.mark.parametrize("B,T,lens", [(3, 2, [4000, 5, 900]), (4, 20, [0, 3000, 0, 64]), (70, 3, [300 - 4 * i for i in range(70)]),
                                      (2, 40, [0, 0]), (5, 1, [33, 0, 5000, 255, 257])])
def test_batches_of_very_different_lengths(cuda, B, T, lens):
    """The splits go to the batch rows by what they have to attend to."""
    layer = make_layer(B, 2, max(lens) + T, 4, True, seed=41)
    q = randn((B, 6, T, D), 5)
    starts = [n // 3 for n in lens]
    parents = [random_tree(T, b) for b in range(B)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for st in (None, starts):
        got = tree_attention(q, layer, torch.tensor(parents), 3, seq_lens=i32(lens), seq_starts=None if st is None else i32(st))
        ref, _ = attend(q, *rows64(layer), tree_mask(parents, max(lens) + T, st or [0] * B, lens))
        check(got, ref)


def test_offsets_past_32_bits(cuda):
    """A cache of 100 million slots: the tokens attended to are its last ones."""
    N, T, H = 100_000_000, 5, 1
    small = make_layer(1, H, 200 + T, 4, True, seed=43)
    st, c = small._store, small.codecs
    big = {n: torch.zeros((1, H, N, *getattr(st, n).shape[3:]), dtype=getattr(st, n).dtype, device="cuda")
           for n in ("kc", "kn", "ks", "kr", "vc", "vn")}
    for n, b in big.items():
        b[:, :, N - 200 - T:] = getattr(st, n)[:, :, :200 + T]
    q = randn((1, 4, T, D), 5)
    parents = random_tree(T, 1)
    got = K.tree_attention(q, torch.tensor(parents), k_codes=big["kc"], k_norms=big["kn"], v_codes=big["vc"], v_norms=big["vn"],
                           n_tokens=N, key=c.key, value=c.value, k_signs=big["ks"], k_rnorms=big["kr"], qjl=c.qjl,
                           seq_starts=torch.tensor([N - 200 - T]))
    ref, _ = attend(q, *rows64(small), tree_mask([parents], 200 + T, [0], [200]))
    check(got, ref)


def test_replays_with_other_lengths(cuda):
    """The sharing out of splits happens on the device: a captured call goes by the lengths of its replay."""
    B, T, N = 3, 4, 3000
    layer = make_layer(B, 2, N + T, 4, True, seed=45)
    q, parents = randn((B, 8, T, D), 5), torch.tensor(random_tree(T, 0), dtype=torch.int32, device="cuda")
    lens = torch.tensor([N, 10, 700], dtype=torch.int32, device="cuda")
    starts = torch.zeros(B, dtype=torch.int32, device="cuda")
    tree_attention(q, layer, parents, 4, seq_starts=starts, seq_lens=lens)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tree_attention(q, layer, parents, 4, seq_starts=starts, seq_lens=lens)
    for st, ln in (([0, 0, 0], [N, 10, 700]), ([5, 100, 0], [5, N, 1]), ([0, 2999, 64], [N, N, N])):
        starts.copy_(torch.tensor(st, dtype=torch.int32))
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        again = tree_attention(q, layer, parents, 4, seq_starts=starts, seq_lens=lens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, again)
        ref, _ = attend(q, *rows64(layer), tree_mask([parents.tolist()] * B, N + T, st, ln))
        check(out, ref)
