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
