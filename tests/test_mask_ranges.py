"""The ranges of a mask's rows, kept from layer to layer of a step."""

import pytest
import torch

from turboquant.runtime import attention as A

CPU = torch.device("cpu")


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
