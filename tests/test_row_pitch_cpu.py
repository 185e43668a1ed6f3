"""Row pitches of pitched views: what rmsnorm() tells the kernel has to be where the rows really are, and every view whose
rows follow one another at one pitch has to be taken, dimensions of length one among them."""
from __future__ import annotations

import itertools
import random

import pytest
import torch

from onnxsharp_b200.ops import _row_pitch


def _rows(t):
    """Offset of every row of t, in order."""
    return [sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape[:-1]))]


def _check(t):
    rows, cols = _rows(t), t.shape[-1]
    steps = {b - a for a, b in zip(rows, rows[1:])}
    fits = len(steps) <= 1 and (cols == 1 or t.stride(-1) == 1) and all(s >= cols for s in steps)
    if fits:
        pitch = _row_pitch("t", t, cols)
        assert [i * pitch for i in range(len(rows))] == rows, (t.shape, t.stride(), pitch)
    else:
        with pytest.raises(ValueError, match="pitch"):
            _row_pitch("t", t, cols)
    return fits


def test_slices():
    x = torch.zeros(2, 10, 96)
    assert not _check(x[:, None, :3])  # rows 0, 1, 2, 10, 11, 12: was taken as rows 0 to 5
    assert not _check(x[:, :3])
    assert _check(x[:, -1:])  # the last token of every sequence: was refused
    assert _check(x[:, -1:, :32])
    assert _check(x[:, :, :32])
    assert _check(x[:, None, :, :32])
    assert _check(x[:1, 2:5, 1:33])
    assert _check(x[1, 3])
    assert not _check(x.transpose(0, 1))
    assert not _check(x.transpose(1, 2))
    assert not _check(x[:1, :1].expand(2, 1, 96))
    assert _check(torch.zeros(4, 5)[:, :1])


def test_random_views():
    rng, taken = random.Random(7), 0
    for _ in range(4000):
        dims = [rng.choice([1, 1, 2, 3]) for _ in range(rng.randint(1, 4))]
        t = torch.zeros([n + rng.choice([0, 0, 1]) for n in dims] + [rng.choice([1, 4, 7])])
        view = t[tuple(slice(0, n) for n in dims)]
        if rng.random() < 0.3:
            view = view[..., : rng.randint(1, view.shape[-1])]
        if rng.random() < 0.3 and view.dim() > 2:
            view = view.transpose(rng.randrange(view.dim() - 1), rng.randrange(view.dim() - 1))
        if rng.random() < 0.3:
            view = view.unsqueeze(rng.randrange(view.dim()))
        taken += _check(view)
    assert 1000 < taken < 3900
