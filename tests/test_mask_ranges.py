"""The ranges of a mask's rows, kept from layer to layer of a step."""

import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import attention as A
from turboquant.runtime import share_prefix

from ._packed import D, make_layer, randn

def ranges(mask, **kw):
    B, total = mask.shape
    return [t.tolist() for t in A._valid_range(mask, B, total, mask.device, **kw)]


@pytest.fixture
def computed(monkeypatch):
    calls, compute = [], A._compute_range
    monkeypatch.setattr(A, "_compute_range", lambda *a: calls.append(a[0]) or compute(*a))
    A._tls.last_range = None
    return calls


def test_a_mask_is_looked_at_once_until_it_changes(computed):
    mask = torch.ones(2, 9, dtype=torch.bool)
    for _ in range(3):
        assert ranges(mask) == [[0, 0], [9, 9]]
    assert len(computed) == 1
    mask[1, :4] = False
    assert ranges(mask) == [[0, 4], [9, 9]] and len(computed) == 2
    mask[0, 3] = False
    for _ in range(2):
        with pytest.raises(A._HoleyMask):
            ranges(mask)
    assert len(computed) == 3
    assert ranges(mask, check_contiguous=False) == [[0, 4], [9, 9]]


def test_masks_made_in_inference_mode(computed):
    """They have no version counter: each look is a new one."""
    with torch.inference_mode():
        mask = torch.ones(2, 9, dtype=torch.bool)
        assert ranges(mask) == [[0, 0], [9, 9]]
        mask[1, :4] = False
        assert ranges(mask) == [[0, 4], [9, 9]]
        mask[1, 6] = False
        with pytest.raises(A._HoleyMask):
            ranges(mask)
        mask[1, 6] = True
        assert ranges(mask) == [[0, 4], [9, 9]]
    assert len(computed) == 4


@pytest.mark.gpu
def test_a_step_on_another_stream_finds_its_own_ranges(cuda, computed):
    mask = torch.ones(2, 9, dtype=torch.bool, device="cuda")
    mask[1, :4] = False
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        first = A._valid_range(mask, 2, 9, mask.device, check_contiguous=False)
    second = A._valid_range(mask, 2, 9, mask.device, check_contiguous=False)
    assert len(computed) == 2 and second is not first
    assert [t.tolist() for t in second] == [[0, 4], [9, 9]]
    assert A._valid_range(mask, 2, 9, mask.device, check_contiguous=False) is second
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def shared(counts, seed=0):
    base = make_layer(len(counts), 2, 100, 4, True, seed=seed)
    layer = share_prefix(Cache(layers=[base]), list(counts)).layers[0]
    layer._lazy_update = True
    layer.update(*(randn((sum(counts), 2, 5, D), i) for i in (1, 2)))
    return layer


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["packed", "blocks", "shared"])
def test_captured_steps_with_masks(cuda, kind):
    """The step before the capture has looked at the mask; every replay finds its ranges anew.  Without such a step, and after a
    change of the mask, a refusal that says what to do, and the program goes on."""
    layer = shared((2, 3)) if kind == "shared" else make_layer(5, 2, 1005, 4, True)
    if kind == "blocks":
        layer.attend_blocks(4, sink=1, recent=1)
        layer.block_bounds()
    n = layer.get_seq_length()
    q, mask = randn((5, 8, 1, D), 5), torch.ones(5, n, dtype=torch.bool, device="cuda")
    mask[:2, :30] = False

    def step():
        return A.shared_prefix_attention(q, layer, mask) if kind == "shared" else A.fused_attention(q, layer, 4, mask)

    def refused():
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            q.add_(0.0)
            with pytest.raises(ValueError, match="_tq_mask_contiguous"):
                step()

    A._tls.last_range = A._tls.last_shared = None
    refused()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        mask[2:, :10 * i] = False
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())
    mask[4, 0] = False
    refused()


@pytest.mark.gpu
@pytest.mark.parametrize("hole", [True, False])
def test_captured_steps_of_shared_layers_over_decoded_rows(cuda, hole):
    """Masks that the step before found no shared ranges in: the captured step takes the decoded rows as well."""
    layer = shared((2, 3))
    q, mask = randn((5, 8, 1, D), 5), torch.ones(5, 105, dtype=torch.bool, device="cuda")
    mask[1, slice(40, 60) if hole else slice(0, 30)] = False
    want = A.shared_prefix_attention(q, layer, mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.shared_prefix_attention(q, layer, mask)
    for i in range(3):
        mask[3, 70 + i] = False
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, A.shared_prefix_attention(q, layer, mask)) and not torch.equal(out, want)
