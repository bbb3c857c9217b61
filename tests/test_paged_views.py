"""One sequence's view of a paged cache: what may move the pages of the others is refused."""
import types

import pytest
import torch

from frink_b200 import _lib, device


def test_compacting_a_view_is_refused():
    with pytest.raises(_lib.Invalid, match="view"):
        device.pages_compact(types.SimpleNamespace(_whole=False))


@pytest.mark.gpu
def test_a_view_is_not_compacted_and_the_whole_cache_is():
    pg = device.Pages.alloc(1, 8, 16, 1, 64, 3, 2, device="cuda")
    for s in range(3):
        device.pages_grow(pg.seq(s), 20)
        device.pages_advance(pg.seq(s), 20)
    device.pages_free(pg, [0])
    was = pg.table.clone(), pg.refs.clone(), pg.lens.clone()
    with pytest.raises(_lib.Invalid, match="view"):
        device.pages_compact(pg.seq(1))
    assert all(torch.equal(a, b) for a, b in zip(was, (pg.table, pg.refs, pg.lens)))
    assert device.pages_compact(pg).item() == 4
    assert pg.refs.tolist() == [1] * 4 + [0] * 4 and sorted(pg.table[1:].flatten().tolist()) == [0, 1, 2, 3] and device.device_error() == 0
