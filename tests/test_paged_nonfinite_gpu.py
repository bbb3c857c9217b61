"""Paged attention of a few rows: keys and values that are infinite or NaN spoil the rows that see them and no other, wherever the
rows lie in a block of columns."""
import pytest
import torch

from tests import paged_plain as plain
from tests.helpers import rel_l2
from tests.test_paged_gpu import TOL, TYPES, attend_fast, cache, queries

pytestmark = pytest.mark.gpu
SHAPES = [(24, 8, 128), (2, 2, 64), (10, 5, 96), (3, 3, 8), (16, 2, 64), (32, 2, 128)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("x", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,n_kv,hd", SHAPES)
def test_a_whole_token(dtype, x, heads, n_kv, hd):
    for rows, lens, window, first, bad in ((2, [0], 0, 0, [(0, 1, x)]), (5, [33, 0], 0, 0, [(0, 36, x), (1, 2, x), (1, 4, x)]), (7, [60], 5, 2, [(0, 57, x), (0, 63, x), (0, 66, x)]),
                                           (16, [100, 3], 20, 0, [(0, 85, x), (0, 90, x), (1, 9, x)])):
        attend_fast(lens, [rows] * len(lens), rows, heads, n_kv, hd, 16, TYPES[dtype], window=window, first=first, seed=rows, bad=bad)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("x", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,n_kv,hd", SHAPES)
@pytest.mark.parametrize("rows,n,window,first,at", [(3, 0, 0, 0, 1), (4, 29, 0, 0, 31), (6, 500, 8, 3, 496), (12, 40, 30, 0, 45), (40, 2000, 0, 0, 2039)])
def test_one_value(dtype, x, heads, n_kv, hd, rows, n, window, first, at):
    """One value of one head: the other dims and heads of the rows that see it keep their precision, too."""
    from frink_b200 import device
    pg, data = cache([n], [rows], n_kv, hd, 16, TYPES[dtype], seed=rows)
    q = queries(rows, heads * hd, rows)
    kvh, d = n_kv - 1, hd // 2 + 1
    page = pg.table[0, at // 16].item()
    pg.data[0, page, 1, kvh, at % 16, d] = x
    data[0, page, 1, kvh, at % 16, d] = 0
    got = device.attention_paged(q.cuda(), pg, 0, heads, window=window, first=first).cpu().view(rows, heads, hd)
    assert device.device_error() == 0
    want = plain.attention(q, data[0], pg.table.cpu().tolist(), [n], heads, [rows], window=window, first=first)[0].view(rows, heads, hd)
    p = n + torch.arange(rows)
    sees = (at <= p) & ((at > p - window) | (at < first) if window else True)
    assert 0 < int(sees.sum()) < rows
    hit = torch.zeros(rows, heads, hd, dtype=torch.bool)
    hit[sees, kvh * (heads // n_kv):, d] = True
    assert not torch.isfinite(got[hit]).any() and torch.isfinite(got[~hit]).all()
    assert rel_l2(got[~hit].numpy(), want[~hit].numpy()) <= TOL
