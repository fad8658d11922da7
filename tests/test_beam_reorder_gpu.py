"""Reordering on a GPU as a search uses it: in place, by the native call."""

import pytest
import torch

from kempnerforge_b200.models import SharedPrefixCache
from kempnerforge_b200.ops import beam

pytestmark = pytest.mark.gpu

PARENTS = [[2, 0, 0, 3], [1, 0, 3, 2]]


def test_in_place_by_the_native_call(native_lib):
    """What a search moves at every step: histories and the table of rows, whose beams have room behind them."""
    parents = torch.tensor(PARENTS, device="cuda")
    tokens = torch.randint(0, 99, (2, 4, 20), device="cuda")
    rows = SharedPrefixCache.new_rows(2, 4, 20, "cuda")
    rows.copy_(torch.randint(0, 4, rows.shape, device="cuda", dtype=torch.uint8))
    at, length = torch.arange(2, device="cuda")[:, None], 13
    want = [t.clone() for t in (tokens, rows)]
    for t in want:
        t[:, :, :length] = t[at, parents][:, :, :length]
    versions = [t._version for t in (tokens, rows)]
    launches = native_lib.LAUNCH_COUNT
    assert native_lib.beam_reorder_call([tokens, rows], parents, length, None) is True
    assert native_lib.LAUNCH_COUNT == launches + 1
    assert all(torch.equal(x, y) for x, y in zip((tokens, rows), want))
    assert all(t._version > v for t, v in zip((tokens, rows), versions))
    assert native_lib.beam_reorder_call([tokens, rows], parents, None, None) is True
    assert all(torch.equal(x, y[at, parents]) for x, y in zip((tokens, rows), want))


def test_shared_memory_is_left_to_the_rules(native_lib):
    parents = torch.tensor(PARENTS, device="cuda")
    x, wide = torch.randn(2, 4, 8, device="cuda"), torch.randn(2, 4, 16, device="cuda")
    for states, out in (([x, x], None), ([wide[:, :, :9], wide[:, :, 8:]], None), ([x], [x]), ([wide[:, :, :8]], [wide[:, :, 4:12]]), ([parents], None)):
        assert native_lib.beam_reorder_call(states, parents, None, out) is False
        with pytest.raises(ValueError):
            beam.reorder(states, parents, out=out)
