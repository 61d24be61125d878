"""The ranges of a mask's rows, kept from layer to layer of a step."""

import pytest
import torch
from transformers.cache_utils import Cache

from turboquant.runtime import _lib
from turboquant.runtime import attention as A
from turboquant.runtime import kernels as K
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


@pytest.mark.gpu
def test_a_capture_finds_the_ranges_once_for_its_layers(cuda, computed):
    """And anew in another capture, for another mask and behind a change of the mask within the capture."""
    layers = [make_layer(2, 2, 300, 4, True, seed=i) for i in range(3)]
    masks = [torch.ones(2, 300, dtype=torch.bool, device="cuda") for _ in range(2)]
    masks[1][1, :7] = False
    q = randn((2, 8, 1, D), 5)
    for layer in layers:
        layer._tq_mask_contiguous = True

    def steps():
        first = [A.fused_attention(q, layer, 4, masks[0]) for layer in layers]
        other = [A.fused_attention(q, layer, 4, masks[1]) for layer in layers]
        masks[1][0, :100] = False
        changed = [A.fused_attention(q, layer, 4, masks[1]) for layer in layers]
        masks[1][0, :100] = True
        return first + other + changed

    want = [t.clone() for t in steps()]
    assert len(computed) == 3
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = steps()
        graphs.append((graph, out))
        assert len(computed) == 6 + 3 * i
    for _ in range(2):
        for graph, out in reversed(graphs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    masks[0][1, :60] = False
    want = [t.clone() for t in steps()]
    for graph, out in graphs:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_captures_have_ids_of_their_own(cuda):
    ids, x = [], torch.zeros(3, device="cuda")
    assert K.capture_id(x.device) == 0
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ids.append(K.capture_id(x.device))
            x.add_(1.0)
            assert K.capture_id(x.device) == ids[-1]
    assert 0 not in ids and ids[0] != ids[1] and K.capture_id(x.device) == 0


def test_a_capture_id_needs_a_place_to_go():
    assert _lib.load().tq_capture_id(None, None) == 1  # TQ_ERR_INVALID_ARGUMENT
