"""Refusals of the calls behind shared prompts and over blocks on the host, before any launch: no GPU needed."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from transformers.cache_utils import Cache

from turboquant.runtime import _lib, share_prefix
from turboquant.runtime import kernels as K
from turboquant.runtime.packed_qmse_cache import BlockChoice, PackedMSELayer
from turboquant.runtime.params import layer_codecs

FAKE, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)  # never dereferenced: validation fails first
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
INF, NAN = float("inf"), float("nan")
SIX = (ctypes.c_void_p * 6)(*[1 << 20] * 6)


def six(**odd):
    names = ["kc", "kn", "ks", "kr", "vc", "vn"]
    return (ctypes.c_void_p * 6)(*[odd.get(n, 1 << 20) for n in names])


PREFIX = dict(q=FAKE, q_type=0, batch=4, q_heads=8, kv_heads=2, dim=128, q_sb=1024, q_sh=128, prompts=2, cu=None, most=4, starts=None,
              lens=None, n=100, cap=100, prefix=SIX, own_lens=None, n_own=5, cap_own=8, own=SIX, kb=3, vb=4, qjl=1, rk=FAKE,
              ck=FAKE, s=FAKE, rv=FAKE, cv=FAKE, scale=0.1, of=None, o16=FAKE, lse=None, ws=FAKE, wsb=1 << 40, stream=None)


@pytest.mark.parametrize("status,change", [
    *((INVALID, {name: None}) for name in ("q", "prefix", "own", "rk", "ck", "s", "rv", "cv", "o16")),
    *((INVALID, dict(prefix=six(**{name: None}))) for name in ("kc", "kn", "ks", "kr", "vc", "vn")),
    *((INVALID, dict(own=six(**{name: None}))) for name in ("kc", "kn", "ks", "kr", "vc", "vn")),
    (INVALID, dict(q_type=3)), (INVALID, dict(q_type=-1)), (INVALID, dict(batch=0)), (INVALID, dict(q_heads=9)),
    (INVALID, dict(prompts=0)), (INVALID, dict(prompts=3)), (INVALID, dict(n=-1)), (INVALID, dict(n=101)), (INVALID, dict(n_own=9)),
    (INVALID, dict(n_own=-1)), (INVALID, dict(scale=0.0)), (INVALID, dict(scale=INF)), (INVALID, dict(scale=NAN)),
    (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(q_heads=130)), (UNSUPPORTED, dict(n=1 << 31, cap=1 << 31)),
    (UNSUPPORTED, dict(n=1 << 29, cap=1 << 29)), (UNSUPPORTED, dict(n_own=1 << 23, cap_own=1 << 23)),
    (UNSUPPORTED, dict(n_own=1 << 31, cap_own=1 << 31)), (UNSUPPORTED, dict(batch=1 << 24)),
    (UNSUPPORTED, dict(vb=5, kb=4)), (UNSUPPORTED, dict(vb=4, kb=4)), (UNSUPPORTED, dict(vb=1, kb=0)), (UNSUPPORTED, dict(qjl=0)),
    (UNSUPPORTED, dict(rk=ODD)), (UNSUPPORTED, dict(s=ODD)), (UNSUPPORTED, dict(prefix=six(kc=(1 << 20) + 8))),
    (UNSUPPORTED, dict(prefix=six(ks=(1 << 20) + 4))), (UNSUPPORTED, dict(own=six(vc=(1 << 20) + 8))),
    (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(ws=ODD)), (WORKSPACE, dict(wsb=1000))])
def test_prefix_attention_rejects_on_host(status, change):
    assert _lib.load().tq_prefix_attention(*dict(PREFIX, **change).values()) == status


def test_prefix_workspace_is_host_arithmetic():
    size = _lib.load().tq_prefix_attention_workspace_bytes
    assert 0 < size(2, 8, 2, 128, 1, 0, 2, 0, 0) <= size(64, 32, 8, 128, 1, 0, 64, 32768, 100)
    assert size(64, 32, 8, 128, 3, 1, 64, 32768, 100) > 0
    for bad in ((64, 32, 8, 128, 3, 0, 64, 9, 9), (2, 8, 2, 64, 1, 0, 2, 9, 9), (2, 8, 3, 128, 1, 0, 2, 9, 9), (2, 130, 2, 128, 1, 0, 2, 9, 9),
                (2, 8, 2, 128, 1, 0, 2, -1, 9), (0, 8, 2, 128, 1, 0, 2, 9, 9)):
        assert size(*bad) == 0


BOUNDS = dict(k=FAKE, batch=1, heads=2, tokens=100, dim=128, sb=0, sh=12800, st=128, lohi=FAKE, step=FAKE, cap=4, first=2, stream=None)


@pytest.mark.parametrize("status,change", [
    *((INVALID, {name: None}) for name in ("k", "lohi", "step")), (INVALID, dict(batch=0)), (INVALID, dict(heads=0)),
    (INVALID, dict(tokens=0)), (INVALID, dict(first=-1)), (INVALID, dict(first=3)), (INVALID, dict(cap=1)),
    (INVALID, dict(tokens=129)), (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(st=130)), (UNSUPPORTED, dict(sh=4)),
    (UNSUPPORTED, dict(k=ODD)), (UNSUPPORTED, dict(lohi=ODD)),
    (UNSUPPORTED, dict(tokens=1 << 37, cap=1 << 40)), (UNSUPPORTED, dict(batch=1 << 20, heads=1 << 10, cap=1 << 40))])
def test_block_bounds_rejects_on_host(status, change):
    assert _lib.load().tq_block_bounds(*dict(BOUNDS, **change).values()) == status


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(k_type=3)), (INVALID, dict(k_type=-1)), (INVALID, dict(k=None)), (UNSUPPORTED, dict(st=132)),
    (UNSUPPORTED, dict(k_type=2, st=132)), (UNSUPPORTED, dict(k_type=1, st=130)), (UNSUPPORTED, dict(k_type=1, k=ODD)),
    (UNSUPPORTED, dict(k_type=1, lohi=ODD))])
def test_block_bounds_of_other_types_rejects_on_host(status, change):
    args = {"k": FAKE, "k_type": 0, **BOUNDS}
    assert _lib.load().tq_block_bounds_typed(*dict(args, **change).values()) == status


def test_block_bounds_takes_keys_of_three_types():
    with pytest.raises(ValueError, match="fp16 or fp32"):
        K.block_bounds(torch.zeros(1, 2, 64, 128, dtype=torch.float64), *lohi_step())


SELECT = dict(q=FAKE, q_type=0, batch=1, q_heads=8, kv_heads=2, dim=128, q_sb=1024, q_sh=128, lohi=FAKE, step=FAKE, cap=40, blocks=40,
              n=2500, starts=None, lens=None, keep=8, sink=1, recent=2, out=FAKE, ws=None, wsb=0, stream=None)


@pytest.mark.parametrize("status,change", [
    *((INVALID, {name: None}) for name in ("q", "lohi", "step", "out")), (INVALID, dict(q_type=3)), (INVALID, dict(batch=0)),
    (INVALID, dict(q_heads=9)), (INVALID, dict(blocks=41)), (INVALID, dict(blocks=-1)), (INVALID, dict(n=-1)), (INVALID, dict(keep=0)),
    (INVALID, dict(sink=-1)), (INVALID, dict(recent=-1)), (INVALID, dict(sink=7)), (INVALID, dict(sink=1 << 30, recent=1 << 30)),
    (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(keep=4097)), (UNSUPPORTED, dict(n=32768 * 64 + 1)), (UNSUPPORTED, dict(lohi=ODD)),
    (UNSUPPORTED, dict(batch=1 << 30, kv_heads=8)), (WORKSPACE, dict(n=100000)), (WORKSPACE, dict(n=100000, ws=FAKE, wsb=100)),
    (WORKSPACE, dict(n=100000, ws=ODD, wsb=1 << 30)), (UNSUPPORTED, dict(n=100000, batch=1 << 16, ws=FAKE, wsb=1 << 60))])
def test_select_blocks_rejects_on_host(status, change):
    assert _lib.load().tq_select_blocks(*dict(SELECT, **change).values()) == status


BLOCKS = dict(q=FAKE, batch=1, q_heads=8, kv_heads=2, dim=128, blocks=FAKE, keep=4, starts=None, lens=None, n=100, cap=100, kc=FAKE,
              kn=FAKE, ks=FAKE, kr=FAKE, vc=FAKE, vn=FAKE, kb=3, vb=4, qjl=1, rk=FAKE, ck=FAKE, s=FAKE, rv=FAKE, cv=FAKE, scale=0.1,
              of=None, ob=FAKE, lse=None, ws=FAKE, wsb=1 << 40, stream=None)


@pytest.mark.parametrize("status,change", [
    *((INVALID, {name: None}) for name in ("q", "blocks", "kc", "kn", "ks", "kr", "vc", "vn", "rk", "ck", "s", "rv", "cv", "ob")),
    (INVALID, dict(batch=0)), (INVALID, dict(q_heads=9)), (INVALID, dict(keep=0)), (INVALID, dict(n=-1)), (INVALID, dict(n=101)),
    (INVALID, dict(scale=0.0)), (INVALID, dict(scale=-1.0)), (INVALID, dict(scale=INF)), (INVALID, dict(scale=NAN)),
    (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(q_heads=18)), (UNSUPPORTED, dict(keep=4097)),
    (UNSUPPORTED, dict(n=1 << 24, cap=1 << 24)), (UNSUPPORTED, dict(vb=5, kb=4)), (UNSUPPORTED, dict(vb=4, kb=4)),
    (UNSUPPORTED, dict(qjl=0)), (UNSUPPORTED, dict(batch=32768)), (UNSUPPORTED, dict(q=ODD)), (UNSUPPORTED, dict(kc=ODD)),
    (UNSUPPORTED, dict(ks=ODD)), (UNSUPPORTED, dict(vc=ODD)), (UNSUPPORTED, dict(rk=ODD)), (UNSUPPORTED, dict(rv=ODD)),
    (UNSUPPORTED, dict(s=ODD)), (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(ws=ODD)), (WORKSPACE, dict(wsb=100))])
def test_block_attention_rejects_on_host(status, change):
    assert _lib.load().tq_block_attention(*dict(BLOCKS, **change).values()) == status


@pytest.mark.parametrize("status,change", [(INVALID, dict(q_type=3)), (INVALID, dict(q_type=-1)), (INVALID, dict(q=None)),
                                           (INVALID, dict(q_type=2, ob=None)), (UNSUPPORTED, dict(q_type=1, q=ODD)),
                                           (UNSUPPORTED, dict(q_type=2, q_heads=18)), (WORKSPACE, dict(q_type=1, wsb=100))])
def test_block_attention_of_other_types_rejects_on_host(status, change):
    args = {"q": FAKE, "q_type": 0, **BLOCKS}
    assert _lib.load().tq_block_attention_typed(*dict(args, **change).values()) == status


def test_select_workspace_is_host_arithmetic():
    size = _lib.load().tq_select_blocks_workspace_bytes
    assert size(1, 2, 0) == size(1, 2, 1000) == 0 < size(1, 2, 100000) < size(2, 2, 100000)
    assert size(0, 2, 100000) == size(1, 0, 100000) == size(1, 2, -1) == size(1, 2, 1 << 40) == 0


def test_block_workspace_is_host_arithmetic():
    size = _lib.load().tq_block_attention_workspace_bytes
    assert 0 < size(1, 8, 2, 128, 1) <= size(8, 32, 8, 128, 4096)
    for bad in ((0, 8, 2, 128, 1), (1, 8, 2, 64, 1), (1, 8, 2, 128, 0), (1, 8, 2, 128, 4097)):
        assert size(*bad) == 0


# ---------------------------------------------------------------- the package's functions


def cache(B=1, H=2, cap=100, bits=4):
    u8 = lambda n: torch.zeros(B, H, cap, n, dtype=torch.uint8)  # noqa: E731
    f16 = lambda: torch.ones(B, H, cap, dtype=torch.float16)  # noqa: E731
    return {"k_codes": u8(16 * (bits - 1)), "k_norms": f16(), "k_signs": u8(16), "k_rnorms": f16(), "v_codes": u8(16 * bits),
            "v_norms": f16()}


def lohi_step(B=1, H=2, n=10):
    return torch.zeros(B, H, n, 2, 128, dtype=torch.int8), torch.ones(B, H, n)


def calls(q, k):
    c = layer_codecs(128, 4, 0, True, torch.device("cpu"))
    codec = dict(key=c.key, value=c.value, qjl=c.qjl)
    return [lambda: K.prefix_attention(q, cache(), n_prefix=100, **codec), lambda: K.block_bounds(k, *lohi_step()),
            lambda: K.select_blocks(q, *lohi_step(), n_tokens=600, keep=4),
            lambda: K.block_attention(q, torch.zeros(1, 2, 3, dtype=torch.int32), **cache(), n_tokens=100, **codec)]


def test_there_is_no_cpu_path():
    for f in calls(torch.zeros(1, 8, 128).bfloat16(), torch.zeros(1, 2, 64, 128).bfloat16()):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_gradients_traces_and_transforms_are_refused():
    q, k = torch.zeros(1, 8, 128, requires_grad=True), torch.zeros(1, 2, 64, 128, requires_grad=True)
    for f in calls(q, k):
        with pytest.raises(ValueError, match="backward"):
            f()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
            f()
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t.detach(), torch.ones_like(t)) for t in (q, k)]
        for f in calls(*dual):
            with pytest.raises(ValueError, match="tangent"):
                f()
    q, k = q.detach(), k.detach()
    for i in range(4):
        with pytest.raises(ValueError, match="trace"):
            torch.func.vmap(lambda x: calls(q, k)[i]())(torch.zeros(2))


@pytest.mark.parametrize("shape", [(1, 8, 64), (1, 8, 2, 128), (8, 128), (1, 2, 8, 1, 128)])
def test_queries_of_other_shapes(shape):
    for f in (calls(torch.zeros(shape).bfloat16(), None)[i] for i in (0, 2, 3)):
        with pytest.raises(ValueError):
            f()


def test_queries_of_other_types():
    for f in (calls(torch.zeros(1, 8, 128, dtype=torch.float64), None)[i] for i in (0, 2, 3)):
        with pytest.raises(ValueError, match="bf16"):
            f()


def test_layers_that_hold_nothing_to_share_or_choose_from():
    with pytest.raises(ValueError, match="not in the cache"):
        share_prefix(Cache(layers=[PackedMSELayer(bits=4)]), 2)
    with pytest.raises(ValueError, match="one-group"):
        PackedMSELayer(bits=4).block_bounds()
    layer = PackedMSELayer(bits=4)
    layer.attend_blocks(8)
    assert layer._choice == BlockChoice(8, 1, 2)
    with pytest.raises(ValueError):
        layer.attend_blocks(2)
    layer.attend_blocks(None)
    assert layer._choice is None
