"""CPU checks of where results may go: tensors whose elements lie on each other."""
import itertools

import pytest
import torch

from streamvoxel_amd import _lib


def places(t):
    return [t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))]


def test_elements_on_each_other():
    """Never missed, and what a program lays out (contiguous, permuted, sliced, interleaved) is never taken for it."""
    flat = torch.zeros(5000)
    g = torch.Generator().manual_seed(1)
    draw = lambda low, high: int(torch.randint(low, high, (1,), generator=g))
    found = 0
    for _ in range(4000):
        shape = [draw(1, 4) for _ in range(4)]
        t = flat.as_strided(shape, [draw(0, 40) for _ in shape])
        at = places(t)
        if len(set(at)) < len(at):
            found += 1
            assert _lib.stacked(t), (t.shape, t.stride())
    assert found > 1000
    for _ in range(500):
        t = torch.zeros([draw(1, 6) for _ in range(4)]).permute(torch.randperm(4, generator=g).tolist())
        t = t[tuple(slice(draw(0, 2), None, draw(1, 3)) for _ in range(4))]
        assert not _lib.stacked(t), (t.shape, t.stride())
        assert not _lib.stacked(t.unsqueeze(2).expand(-1, -1, 1, -1, -1))
    rows = torch.zeros(2, 7, 3, 8)
    for t in (rows[:, :, 1], rows[:, :, :2].transpose(1, 2), rows.unfold(1, 2, 2), rows.unfold(1, 3, 4), rows[:0].expand(0, 7, 3, 8)):
        assert not _lib.stacked(t)
    for t in (rows[:, :1].expand(2, 7, 3, 8), torch.zeros(40).unfold(0, 8, 4), torch.zeros(40).unfold(0, 8, 7),
              rows.as_strided((2, 2, 2, 8), (4, 48, 16, 1))):
        assert _lib.stacked(t)


def test_spans_and_what_meets_them():
    g = torch.Generator().manual_seed(2)
    draw = lambda low, high: int(torch.randint(low, high, (1,), generator=g))
    flat = torch.zeros(400)
    met = 0
    for _ in range(2000):
        a, b, c = [flat.as_strided([draw(0 if i else 1, 4) for _ in range(3)], [draw(0, 12) for _ in range(3)], draw(0, 300))
                   for i in range(3)]
        for t in (a, b, c):
            at = places(t)
            first, last = _lib.byte_span(t)
            assert (last - first == 0) if not at else (first, last) == (flat.data_ptr() + 4 * min(at), flat.data_ptr() + 4 * max(at) + 4)
        share = lambda t: _lib.byte_span(a)[0] < _lib.byte_span(t)[1] and _lib.byte_span(t)[0] < _lib.byte_span(a)[1]
        assert _lib.overlaps(a, b) == share(b)
        assert _lib.overlaps_any(a, b, None, c) == (share(b) or share(c))
        if set(places(a)) & set(places(b)):
            met += 1
            assert _lib.overlaps_any(a, b)
    assert met > 20 and not _lib.overlaps_any(a, None)
