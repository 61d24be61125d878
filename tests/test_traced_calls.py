"""Prompt attention, tree attention and the token moves under a trace or a transform: refused before they launch, since torch
would not see what they write.  No GPU needed."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from turboquant.runtime import kernels as K
from turboquant.runtime import prompt_attention, tree_attention
from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.params import layer_codecs

PARENTS = torch.tensor([-1, 0, 1, 2])


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def prompt(q):
    return prompt_attention(q, bf16(1, 2, 4, 128), bf16(1, 2, 4, 128))


def tree(q):
    c = layer_codecs(128, 4, 0, False, "cpu").value
    codes, norms = torch.zeros(1, 2, 9, 64, dtype=torch.uint8), torch.zeros(1, 2, 9, dtype=torch.float16)
    return K.tree_attention(q, PARENTS, k_codes=codes, k_norms=norms, v_codes=codes, v_norms=norms, n_tokens=9, key=c, value=c)


def gather(q):
    return K.gather_tokens([q], tokens=4)[0]


def keep(q):
    K.keep_tokens([q], torch.tensor([1]), first=0, tokens=4)
    return q


def vmapped(f, q):
    return torch.vmap(f)(q[None])


def faked(f, q):
    with FakeTensorMode(allow_non_fake_inputs=True):
        return f(q)


CALLS = [prompt, tree, gather, keep]


@pytest.mark.parametrize("call", CALLS, ids=lambda f: f.__name__)
@pytest.mark.parametrize("watch", [lambda f, q: torch.jit.trace(f, (q,)), lambda f, q: make_fx(f)(q), faked, vmapped],
                         ids=["trace", "make_fx", "fake tensors", "vmap"])
@pytest.mark.filterwarnings("ignore")
def test_refused(call, watch):
    with torch.no_grad(), pytest.raises(ValueError, match="cannot be traced or transformed"):
        watch(call, bf16(1, 8, 4, 128))


@pytest.mark.parametrize("call", CALLS, ids=lambda f: f.__name__)
def test_modes_that_look_on_are_none_of_it(call):
    with FlopCounterMode(display=False), pytest.raises(RuntimeError, match="GPU only"):
        call(bf16(1, 8, 4, 128))


def test_a_tree_of_torch_operations_can_be_traced():
    layer = PackedMSELayer(bits=4)
    layer.initialize_from_dense(bf16(1, 2, 9, 128), bf16(1, 2, 9, 128), force_dense=True)
    q = bf16(1, 8, 4, 128)
    assert make_fx(lambda x: tree_attention(x, layer, PARENTS))(q)(q).shape == q.shape
