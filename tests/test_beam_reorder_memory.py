"""Which states a reordering takes for apart from each other, on the CPU."""

import random

import pytest
import torch

from kempnerforge_b200.ops import beam


def test_slices_of_one_tensor_that_are_not_dense():
    """Keys and values beside each other at every position."""
    both = torch.arange(2 * 3 * 5 * 2 * 4.0).view(2, 3, 5, 2, 4).clone()
    parents = torch.tensor([[1, 0, 0], [2, 2, 1]])
    want = both.clone()
    want[:, :, :3] = torch.stack([both[i, parents[i]] for i in range(2)])[:, :, :3]
    beam.reorder([both[:, :, :, 0], both[:, :, :, 1]], parents, 3)
    assert torch.equal(both, want)
    # every second value and the others
    want = torch.stack([both[i, parents[i]] for i in range(2)])
    beam.reorder([both[..., ::2], both[..., 1::2]], parents)
    assert torch.equal(both, want)


def test_slices_that_meet():
    parents = torch.tensor([[1, 0], [1, 1]])
    flat = torch.zeros(200)
    wide = torch.zeros(2, 2, 5, 4)
    for a, b in (
        # beams of one value in steps of 10 and 11: the second of the one is the third of the other
        (flat.as_strided((2, 2, 1), (10, 11, 1), 0), flat.as_strided((2, 2, 1), (10, 11, 1), 1)),
        (wide[..., :3], wide[..., 1:]), (wide[:, :, :4], wide[:, :, 1:]), (wide[..., ::2], wide[..., ::2]), (wide[:, :, :, 0], wide[:, :, :, 0]),
        # the first beam of the one is the second of the other
        (flat.as_strided((2, 2, 3), (40, 8, 1), 0), flat.as_strided((2, 2, 3), (40, 8, 1), 8)),
        # of other types, whose values lie across each other's
        (flat.as_strided((2, 2, 3), (40, 8, 1), 0), flat.view(torch.int16).as_strided((2, 2, 3), (80, 16, 2), 3)),
    ):
        with pytest.raises(ValueError):
            beam.reorder([a, b], parents)


def test_against_every_address():
    """Steps of any order and with gaps: apart is what has no byte in common."""
    rng = random.Random(0)
    flat, index = torch.zeros(4000, dtype=torch.int16), torch.arange(4000)
    count = 0
    for _ in range(500):
        shape = [rng.randint(1, 4) for _ in range(rng.randint(2, 4))]
        steps, step = [], rng.randint(1, 3)
        for n in reversed(shape):
            steps.append(step)
            step = step * n + rng.choice([0, 0, 1, 2, 5])
        order = rng.sample(range(len(shape)), len(shape))
        shape, steps = [shape[i] for i in order], [steps[::-1][i] for i in order]
        at = rng.randint(0, min(60, step + 2))
        a, b = flat.as_strided(shape, steps, 0), flat.as_strided(shape, steps, at)
        met = set(index.as_strided(shape, steps, 0).flatten().tolist()) & set(index.as_strided(shape, steps, at).flatten().tolist())
        count += bool(met)
        parents = torch.arange(shape[1]).expand(shape[0], shape[1]).contiguous()
        if met:
            with pytest.raises(ValueError):
                beam.reorder([a, b], parents)
        else:
            beam.reorder([a, b], parents)
    assert 100 < count < 400
