"""Refusals of the prompt, tree and token-moving calls on the host, before any launch: no GPU needed."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from turboquant.runtime import _lib, prompt_attention, tree_attention
from turboquant.runtime import kernels as K
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.params import layer_codecs

FAKE, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)  # never dereferenced: validation fails first
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(q=None)), (INVALID, dict(k=None)), (INVALID, dict(v=None)), (INVALID, dict(out=None)),
    (INVALID, dict(batch=0)), (INVALID, dict(q_heads=0)), (INVALID, dict(kv_heads=0)), (INVALID, dict(q_heads=9)),
    (INVALID, dict(tokens=0)), (INVALID, dict(tokens=-1)), (INVALID, dict(scale=0.0)), (INVALID, dict(scale=-1.0)),
    (INVALID, dict(scale=INF)), (INVALID, dict(scale=NAN)), (INVALID, dict(cu=FAKE, n_seqs=0)),
    (INVALID, dict(cu=FAKE, n_seqs=2, batch=2)), (INVALID, dict(cu=FAKE, n_seqs=2, starts=FAKE)),
    (INVALID, dict(cu=FAKE, n_seqs=2, ends=FAKE)), (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(q_st=130)),
    (UNSUPPORTED, dict(k_sh=4)), (UNSUPPORTED, dict(o_sb=12)), (UNSUPPORTED, dict(k_st=-128)),
    (UNSUPPORTED, dict(v_st=1 << 25)), (UNSUPPORTED, dict(q=ODD)), (UNSUPPORTED, dict(k=ODD)), (UNSUPPORTED, dict(v=ODD)),
    (UNSUPPORTED, dict(out=ODD)), (UNSUPPORTED, dict(tokens=(1 << 30) + 1)), (UNSUPPORTED, dict(tokens=1 << 30, q_heads=32)),
    (UNSUPPORTED, dict(cu=FAKE, n_seqs=(1 << 31) - 1)), (UNSUPPORTED, dict(batch=1 << 22, kv_heads=1, q_heads=4)),
    (UNSUPPORTED, dict(tokens=1, batch=1 << 20, kv_heads=1, q_heads=8))])
def test_prompt_attention_rejects_on_host(status, change):
    args = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=None, f16=0, batch=1, q_heads=8, kv_heads=2, tokens=300, dim=128,
                q_sb=0, q_sh=128, q_st=1024, k_sb=0, k_sh=128, k_st=256, v_sb=0, v_sh=128, v_st=256, o_sb=0, o_sh=128,
                o_st=1024, cu=None, n_seqs=0, starts=None, ends=None, zero=1, scale=0.1, stream=None)
    assert _lib.load().tq_prompt_attention(*dict(args, **change).values()) == status


TREE = dict(q=FAKE, q_type=0, batch=1, q_heads=8, kv_heads=2, nodes=8, dim=128, q_sb=0, q_sh=0, q_st=128, parents=FAKE, psb=0,
            starts=None, lens=None, n=100, cap=100, kc=FAKE, kn=FAKE, ks=FAKE, kr=FAKE, vc=FAKE, vn=FAKE, kb=3, vb=4, qjl=1,
            rk=FAKE, ck=FAKE, s=FAKE, rv=FAKE, cv=FAKE, scale=0.1, of=None, ob=FAKE, lse=None, ws=FAKE, wsb=1 << 40,
            stream=None)


@pytest.mark.parametrize("status,change", [
    *((INVALID, {name: None}) for name in ("q", "kc", "kn", "ks", "kr", "vc", "vn", "rk", "ck", "s", "rv", "cv", "ob")),
    (INVALID, dict(q_type=3)), (INVALID, dict(q_type=-1)), (INVALID, dict(batch=0)), (INVALID, dict(q_heads=9)),
    (INVALID, dict(nodes=0)), (INVALID, dict(n=-1)), (INVALID, dict(n=101)), (INVALID, dict(n=0, cap=0)),
    (INVALID, dict(scale=0.0)), (INVALID, dict(scale=INF)), (INVALID, dict(scale=NAN)),
    (UNSUPPORTED, dict(dim=64)), (UNSUPPORTED, dict(nodes=65)), (UNSUPPORTED, dict(n=1 << 31, cap=1 << 31)),
    (UNSUPPORTED, dict(vb=5, kb=4)), (UNSUPPORTED, dict(vb=4, kb=4)), (UNSUPPORTED, dict(vb=1, kb=0)),
    (UNSUPPORTED, dict(qjl=0)), (UNSUPPORTED, dict(rk=ODD)), (UNSUPPORTED, dict(kc=ODD)), (UNSUPPORTED, dict(vc=ODD)),
    (UNSUPPORTED, dict(ks=ODD)), (UNSUPPORTED, dict(s=ODD)), (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(ws=ODD)),
    (WORKSPACE, dict(wsb=1000))])
def test_tree_attention_rejects_on_host(status, change):
    assert _lib.load().tq_tree_attention(*dict(TREE, **change).values()) == status


def test_tree_workspace_is_host_arithmetic():
    size = _lib.load().tq_tree_attention_workspace_bytes
    assert 0 < size(1, 8, 2, 1, 128, 0) <= size(8, 32, 8, 64, 128, 32768)
    assert size(1, 8, 2, 0, 128, 9) == size(1, 8, 2, 65, 128, 9) == size(1, 9, 2, 4, 128, 9) == size(1, 8, 2, 4, 64, 9) == 0


def moves(n):
    return (ctypes.c_void_p * max(n, 1))(*[1 << 20] * n), (ctypes.c_int * max(n, 1))(*[48] * n)


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(n_buffers=0)), (INVALID, dict(n_buffers=17)), (INVALID, dict(src=None)), (INVALID, dict(dst=None)),
    (INVALID, dict(row=None)), (INVALID, dict(row=[0])), (INVALID, dict(row=[1025])), (INVALID, dict(src_batch=0)),
    (INVALID, dict(heads=0)), (INVALID, dict(tokens=-1)), (INVALID, dict(tokens=101)), (INVALID, dict(dst_batch=0)),
    (INVALID, dict(dst_cap=0)), (INVALID, dict(dst_cap=79)), (INVALID, dict(dst_batch=3)),
    (INVALID, dict(index=FAKE, n_index=-1)), (INVALID, dict(index=FAKE, n_index=101)),
    (UNSUPPORTED, dict(src_batch=1 << 20, dst_batch=1 << 20, heads=64, dst_cap=1 << 20))])
def test_gather_tokens_rejects_on_host(status, change):
    ptrs, rows = moves(17)
    args = dict(n_buffers=2, src=ptrs, dst=ptrs, row=rows, src_batch=2, heads=4, src_cap=100, tokens=80, dst_batch=2,
                dst_cap=100, rows=None, index=None, sb=0, sh=0, n_index=0, stream=None)
    if isinstance(change.get("row"), list):
        change = dict(change, row=(ctypes.c_int * 2)(48, *change["row"]))
    assert _lib.load().tq_gather_tokens(*dict(args, **change).values()) == status


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(n_buffers=0)), (INVALID, dict(n_buffers=17)), (INVALID, dict(buffers=None)), (INVALID, dict(row=None)),
    (INVALID, dict(index=None)), (INVALID, dict(batch=0)), (INVALID, dict(heads=0)), (INVALID, dict(first=-1)),
    (INVALID, dict(tokens=-1)), (INVALID, dict(first=41)), (INVALID, dict(n_index=-1)), (INVALID, dict(n_index=61)),
    (UNSUPPORTED, dict(cap=1000, tokens=900, n_index=257)), (UNSUPPORTED, dict(batch=1 << 20, heads=16)),
    (UNSUPPORTED, dict(cap=1000, tokens=900, n_index=65, row=[1024]))])
def test_keep_tokens_rejects_on_host(status, change):
    ptrs, rows = moves(17)
    args = dict(n_buffers=2, buffers=ptrs, row=rows, batch=2, heads=4, cap=100, first=40, tokens=60, index=FAKE, sb=0, sh=0,
                n_index=8, stream=None)
    if isinstance(change.get("row"), list):
        change = dict(change, row=(ctypes.c_int * 2)(48, *change["row"]))
    assert _lib.load().tq_keep_tokens(*dict(args, **change).values()) == status


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_wrappers_refuse_shapes_types_and_cpu_tensors():
    q, k = bf16(1, 8, 4, 128), bf16(1, 2, 4, 128)
    for bad, text in (((q[0], k, k), "expected q"), ((q, k, k[:, :, :3]), "expected q"), ((bf16(1, 8, 4, 64),) * 3, "head_dim"),
                      ((q, k[:, :, :3], k[:, :, :3]), "do not match"), ((q[:, :7], k, k), "do not match"),
                      ((q, k.half(), k), "bf16"), ((q.float(), k.float(), k.float()), "bf16")):
        with pytest.raises(ValueError, match=text):
            prompt_attention(*bad)
    with pytest.raises(ValueError, match="backward"):
        prompt_attention(q.requires_grad_(), k, k)
    q = q.detach()
    with pytest.raises(RuntimeError, match="GPU"):
        prompt_attention(q, k, k)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        prompt_attention(q.requires_grad_(), k, k)
    q = q.detach()
    with pytest.raises(ValueError, match="backward"):
        prompt_attention(q, k, k, out=torch.zeros_like(q).requires_grad_())
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        prompt_attention(q, forward_ad.make_dual(k, k), k)

    q = q.detach()
    lc = layer_codecs(128, 4, 0, False, "cpu")
    codes, norms = torch.zeros(1, 2, 9, 64, dtype=torch.uint8), torch.zeros(1, 2, 9, dtype=torch.float16)
    kw = dict(k_codes=codes, k_norms=norms, v_codes=codes, v_norms=norms, n_tokens=9, key=lc.value, value=lc.value)
    parents = torch.tensor([-1, 0, 1, 2])
    for query, change, text in ((q[0], {}, "expected q"), (q.double(), {}, "bf16, fp16"), (bf16(1, 8, 65, 128), {}, "1 to 64"),
                                (q[:, :, :0], {}, "1 to 64"), (q[:, :7], {}, "do not match"),
                                (q, dict(k_signs=codes), "Q_prod")):
        with pytest.raises(ValueError, match=text):
            K.tree_attention(query, parents, **dict(kw, **change))
    with pytest.raises(RuntimeError, match="GPU"):
        K.tree_attention(q, parents, **kw)

    for call in (lambda b: K.gather_tokens(b, tokens=9), lambda b: K.keep_tokens(b, torch.tensor([0]), first=0, tokens=9)):
        with pytest.raises(RuntimeError, match="GPU"):
            call([codes, norms])
        with pytest.raises(ValueError, match="no buffers"):
            call([])
        with pytest.raises(ValueError, match="one shape"):
            call([codes, norms[:, :, :8]])
        with pytest.raises(ValueError, match="contiguous"):
            call([codes.transpose(1, 2)])
        with pytest.raises(ValueError, match="1025 bytes"):
            call([torch.zeros(1, 2, 9, 1025, dtype=torch.uint8)])


def test_layer_calls_refuse_before_they_launch():
    layer = PackedMSELayer(bits=4)
    layer.initialize_from_dense(bf16(1, 2, 9, 128), bf16(1, 2, 9, 128), force_dense=True)
    q = bf16(1, 8, 3, 128)
    with pytest.raises(ValueError, match="parents must"):
        tree_attention(q, layer, torch.tensor([-1, 0]), 4)
    with pytest.raises(ValueError, match="10 drafted tokens"):
        tree_attention(bf16(1, 8, 10, 128), layer, torch.full((10,), -1), 4)
    with pytest.raises(ValueError, match="seq_lens needs"):
        tree_attention(q, layer, torch.tensor([-1, 0, 1]), 4, seq_lens=torch.tensor([3]))
    with pytest.raises(ValueError, match="of the last 10 of 9 tokens"):
        layer.keep_tokens(torch.tensor([0]), tokens=10)
    with pytest.raises(RuntimeError, match="GPU"):
        layer.keep_tokens(torch.tensor([0]), tokens=3)
    with pytest.raises(RuntimeError, match="GPU"):
        layer.reorder_cache(torch.tensor([0]))
    layer.crop(-2)
    assert layer.get_seq_length() == 7
