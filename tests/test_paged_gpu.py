"""The paged KV cache's operators against plain restatements in 64 bits (tests/paged_plain.py).

Attention's tolerance, relative L2 3e-6.  A weight is 2^(s - m): the exponential's error is 2^-22 = 2.4e-7; s is a sum of at
most 128 products, exact to 24 bits each and added in f32, cut off inside the tensor cores over 6 steps (6 * 2^-24) and rounded
at 4 joins, so within 10 * 2^-24 = 6e-7 of its size, and |s| is below 8 in units of log2 here where the weights count: at most
5e-6 for a single weight, on average (random signs, typical |s| of 1) 6e-7.  The sum over the keys averages those errors; the
sums of weights and values are rounded at every tile of 16 keys, a random walk of 2^-24 * sqrt(n / 64) <= 3e-6 at the longest
case's 131072 keys.  bf16 and f32 parts hold q and weights to 2^-24, f16 parts to 2^-23."""
import numpy as np
import pytest
import torch

from tests import paged_plain as plain
from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = 3e-6


def cache(lens, counts, n_kv, hd, page, dtype, seed=0, stale=float("nan"), n_layers=1, scale=1.0):
    """Pages scattered over a pool whose unused pages and unused slots hold `stale`; -> (Pages, data on the CPU)."""
    from frink_b200 import device
    g = torch.Generator().manual_seed(seed)
    held = [max(1, -(-(a + b) // page)) for a, b in zip(lens, counts)]
    n_pages = sum(held) + 2
    order = torch.randperm(n_pages, generator=g)
    table = torch.full((len(lens), max(held)), -1, dtype=torch.int32)
    data = torch.full((n_layers, n_pages, 2, n_kv, page, hd), stale, dtype=torch.float32)
    refs, at = torch.zeros(n_pages, dtype=torch.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h].int()
        refs[table[s, :h].long()] = 1
        at += h
        n = lens[s] + counts[s]
        x = torch.randn((n_layers, 2, n_kv, n, hd), generator=g) * scale
        for j in range(h):
            m = min(page, n - j * page)
            if m > 0:
                data[:, table[s, j], :, :, :m] = x[:, :, :, j * page:j * page + m]
    data = data.to(dtype)
    return device.Pages(data.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), refs.cuda()), data


def queries(n, width, seed):
    return torch.randn((n, width), generator=torch.Generator().manual_seed(1000 + seed)) * 1.5


def attend(lens, counts, rows, heads, n_kv, hd, page, dtype, window=0, first=0, sinks=False, seed=0, ragged=False, tol=TOL, **kw):
    from frink_b200 import device
    pg, data = cache(lens, counts, n_kv, hd, page, dtype, seed, **kw)
    q = queries(len(lens) * rows, heads * hd, seed)
    sk = torch.randn(heads, generator=torch.Generator().manual_seed(seed)) if sinks else None
    out = torch.full((q.shape[0], heads * hd), 7.0, device="cuda")
    n_new = torch.tensor(counts, dtype=torch.int32).cuda() if ragged else None
    got = device.attention_paged(q.cuda(), pg, data.shape[0] - 1, heads, n_new=n_new, window=window, first=first, sinks=None if sk is None else sk.cuda(), out=out).cpu()
    assert device.device_error() == 0
    want, real = plain.attention(q, data[-1], pg.table.cpu().tolist(), lens, heads, counts, window=window, first=first, sinks=sk)
    assert (got[~real] == 7.0).all()                       # rows that do not exist are left as they were
    assert torch.isfinite(got[real]).all()
    if real.any():
        assert rel_l2(got[real].numpy(), want[real].numpy()) <= tol
    return got, pg


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,n_kv,hd", [(24, 8, 128), (64, 8, 64), (32, 4, 128), (6, 2, 80), (16, 1, 128), (5, 5, 8), (3, 1, 96), (40, 2, 64)])
@pytest.mark.parametrize("lens", [[0], [16, 0, 1, 15, 33], [700, 64]])
def test_decode(dtype, heads, n_kv, hd, lens):
    attend(lens, [1] * len(lens), 1, heads, n_kv, hd, 16, TYPES[dtype], seed=hd)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window,first,sinks", [(0, 0, True), (1, 0, False), (50, 0, True), (50, 4, False), (64, 16, True), (100, 40, False), (40, 1000, False), (1000, 3, False),
                                                 (1, 1, True)])
def test_windows_first_tokens_and_sinks(dtype, page, window, first, sinks):
    attend([0, 3, 130, 257, 400], [1] * 5, 1, 16, 2, 64, page, TYPES[dtype], window=window, first=first, sinks=sinks, seed=window)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,lens,counts", [(2, [40, 0], [2, 2]), (5, [33, 0, 64], [5, 0, 3]), (16, [0], [16]), (40, [100, 0, 7], [40, 31, 0]), (131, [0, 50], [131, 1])])
@pytest.mark.parametrize("heads,n_kv,hd,window,first", [(24, 8, 128, 0, 0), (16, 2, 64, 24, 3), (6, 2, 80, 17, 0), (16, 1, 128, 0, 0)])
def test_several_rows(dtype, rows, lens, counts, heads, n_kv, hd, window, first):
    attend(lens, counts, rows, heads, n_kv, hd, 32, TYPES[dtype], window=window, first=first, sinks=True, seed=rows, ragged=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_long_cache_is_split_and_joined(dtype):
    """131071 tokens: the pages' offsets pass 2^31 bytes only in larger pools, the split runs over every CTA."""
    from frink_b200 import device
    n, heads, n_kv, hd, page = 131071, 8, 1, 64, 64
    held = -(-(n + 1) // page)
    g = torch.Generator(device="cuda").manual_seed(3)
    data = torch.randn((1, held, 2, n_kv, page, hd), generator=g, device="cuda").to(TYPES[dtype])
    table = torch.randperm(held, generator=g, device="cuda").int()[None].contiguous()
    pg = device.Pages(data, table, torch.tensor([n], dtype=torch.int32, device="cuda"), torch.ones(held, dtype=torch.int32, device="cuda"))
    q = queries(1, heads * hd, 5).cuda()
    k, v = (data[0, table[0].long(), i, 0].reshape(-1, hd)[:n + 1].double() for i in (0, 1))
    w = (q.view(heads, hd).double() @ k.T * hd ** -0.5).softmax(1)
    for _ in range(2):
        assert rel_l2(device.attention_paged(q, pg, 0, heads).view(heads, hd).cpu().numpy(), (w @ v).cpu().numpy()) <= TOL
    a, b = (device.attention_paged(q, pg, 0, heads) for _ in range(2))
    assert torch.equal(a, b)                               # the join's order does not depend on which CTA comes last
    assert device.device_error() == 0


def test_offsets_pass_32_bits():
    """A pool of more than 2^32 values: the sequence's pages are the last ones."""
    from frink_b200 import device
    n_kv, hd, page, heads = 8, 128, 128, 8
    per = 2 * n_kv * page * hd
    n_pages = 2 ** 32 // per + 5
    data = torch.zeros((1, n_pages, 2, n_kv, page, hd), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    tail = torch.randn((3, 2, n_kv, page, hd), generator=g, device="cuda").bfloat16()
    data[0, -3:] = tail
    table = torch.tensor([[n_pages - 1, n_pages - 3, n_pages - 2]], dtype=torch.int32, device="cuda")
    pg = device.Pages(data, table, torch.tensor([300], dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda"))
    q, k, v = (queries(1, h * hd, 6 + h).cuda() for h in (heads, n_kv, n_kv))
    rot = device.rope_kv_paged(q, k, v, pg, 0, heads, 1e4)
    tail[1, 1, :, 300 % page] = v.view(n_kv, hd).bfloat16()          # token 300 is in the table's third page, the pool's last but one
    assert torch.equal(data[0, n_pages - 2, 1], tail[1, 1])
    got = device.attention_paged(rot, pg, 0, heads).cpu()
    want, _ = plain.attention(rot, data[0, -3:], [[2, 0, 1]], [300], heads, [1])
    assert rel_l2(got.numpy(), want.numpy()) <= TOL


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_behind_a_mask_do_not_matter(dtype, bad):
    """NaN and infinity in keys and values outside the window, and in a later row's own key and value."""
    from frink_b200 import device
    heads, n_kv, hd, page, n = 16, 2, 64, 16, 90
    for rows, window, first in ((1, 20, 2), (3, 20, 2), (3, 0, 0), (9, 30, 0)):
        pg, data = cache([n], [rows], n_kv, hd, page, TYPES[dtype], seed=8)
        q = queries(rows, heads * hd, 9)
        want, _ = plain.attention(q, data[0], pg.table.cpu().tolist(), [n], heads, [rows], window=window, first=first)
        if window:
            for j in (first, n - window):                  # invisible to every row
                pg.data[0, pg.table[0, j // page].long(), :, :, j % page] = bad
        rows_ok = rows
        if rows > 1:                                        # the last row's own token: only that row sees it
            j = n + rows - 1
            pg.data[0, pg.table[0, j // page].long(), :, :, j % page] = bad
            rows_ok = rows - 1
        got = device.attention_paged(q.cuda(), pg, 0, heads, window=window, first=first).cpu()
        assert rel_l2(got[:rows_ok].numpy(), want[:rows_ok].numpy()) <= TOL
        if rows > 1:
            assert not torch.isfinite(got[-1]).any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_scores_and_far_apart_values(dtype):
    """Scores up to about 60 in units of log2 (one key takes most): 10 * 2^-24 of that is 3.6e-5, times ln 2 = 2.5e-5.  Then
    queries outside f16's range on keys and values next to its smallest ones."""
    attend([200], [1], 1, 8, 1, 128, 16, TYPES[dtype], seed=11, scale=8.0, tol=2.5e-5)
    from frink_b200 import device
    pg, data = cache([100], [1], 1, 64, 16, TYPES[dtype], seed=12, scale=2.0 ** -17)
    q = queries(1, 8 * 64, 12) * 2.0 ** 20
    got = device.attention_paged(q.cuda(), pg, 0, 8).cpu()
    want, _ = plain.attention(q, data[0], pg.table.cpu().tolist(), [100], 8, [1])
    assert rel_l2(got.numpy(), want.numpy()) <= 2.5e-5


def test_wrong_pages_and_lengths_are_raised():
    from frink_b200 import device
    pg, _ = cache([40, 40], [1, 1], 2, 64, 16, torch.bfloat16, seed=13, stale=0.0)
    q, out = queries(2, 8 * 64, 1).cuda(), torch.full((2, 8 * 64), 7.0, device="cuda")
    pg.table[0, 1] = pg.n_pages
    device.attention_paged(q, pg, 0, 8, out=out)
    assert device.device_error() == 97 and torch.isfinite(out).all()
    out.fill_(7.0)
    pg.table[0, 1] = -1
    device.attention_paged(q, pg, 0, 8, out=out)
    assert device.device_error() == 97
    pg.lens[0] = 48
    out.fill_(7.0)
    device.attention_paged(q, pg, 0, 8, out=out)
    assert device.device_error() == 95 and (out[0] == 7.0).all() and (out[1] != 7.0).any()
    k = queries(2, 128, 2).cuda()
    rot = torch.full_like(q, 7.0)
    device.rope_kv_paged(q, k, k, pg, 0, 8, 1e4, out=rot)
    assert device.device_error() == 95 and (rot[0] == 7.0).all() and (rot[1] != 7.0).any()
    pg.lens[0], pg.table[0, 2] = 40, 99999
    before = pg.data.clone()
    device.rope_kv_paged(q[:1].contiguous(), k[:1].contiguous(), k[:1].contiguous(), pg.seq(0), 0, 8, 1e4)
    assert device.device_error() == 97 and torch.equal(before, pg.data)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("neox,norm", [(False, False), (True, True), (False, True)])
@pytest.mark.parametrize("heads,n_kv,hd", [(24, 8, 128), (6, 2, 80), (5, 5, 8), (64, 8, 64)])
def test_append(dtype, neox, norm, heads, n_kv, hd):
    """q f32: the factors are rounded once (2^-24), two products and a sum (3 * 2^-24), the norm 4 more: 8 * 2^-24 = 5e-7.
    Pages: that, and one rounding to the type (half a step)."""
    from frink_b200 import device
    lens, rows, counts = [0, 131, 100000], 3, [3, 2, 3]
    page, T = 16, TYPES[dtype]
    pg = device.Pages.alloc(2, 9, page, n_kv, hd, 3, 6300, dtype=T)
    pg.lens.copy_(torch.tensor(lens))
    for s, c, p in ((0, 0, 3), (1, 8, 5), (2, 6250, 7)):    # only the pages that the rows go to
        pg.table[s, c] = p
    W = (heads + 2 * n_kv) * hd
    qkv = queries(9, W, hd).cuda()                          # column slices of one buffer
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + n_kv) * hd], qkv[:, (heads + n_kv) * hd:]
    g = torch.Generator().manual_seed(2)
    qw, kw = (1 + 0.1 * torch.randn(hd, generator=g) for _ in range(2))
    out = torch.full((9, heads * hd), 7.0, device="cuda")
    kept = qkv.clone()
    device.rope_kv_paged(q, k, v, pg, 1, heads, 1e6, neox=neox, n_new=torch.tensor(counts, dtype=torch.int32).cuda(), q_norm=qw.cuda() if norm else None,
                         k_norm=kw.cuda() if norm else None, eps=1e-5, out=out)
    assert device.device_error() == 0 and torch.equal(kept, qkv)
    at = [lens[r // rows] + r % rows for r in range(9)]
    real = torch.tensor([r % rows < counts[r // rows] for r in range(9)])
    rq = plain.rotate(q, heads, at, 1e6, neox, qw if norm else None, 1e-5)
    rk = plain.rotate(k, n_kv, at, 1e6, neox, kw if norm else None, 1e-5)
    assert (out.cpu()[~real] == 7.0).all()
    assert rel_l2(out.cpu()[real].numpy(), rq[real].numpy()) <= 5e-7
    half = torch.finfo(T).eps / 2
    table, data = pg.table.cpu(), pg.data.cpu()
    assert not data[0].any()                                # the other layer
    seen = set()
    for r in range(9):
        if not real[r]:
            continue
        p, sl = int(table[r // rows, at[r] // page]), at[r] % page
        seen.add((p, sl))
        assert rel_l2(data[1, p, 0, :, sl].double().numpy(), rk[r].view(n_kv, hd).numpy()) <= half + 5e-7
        assert torch.equal(data[1, p, 1, :, sl], v[r].cpu().view(n_kv, hd).to(T))
    written = {tuple(x) for x in data[1].float().abs().sum((1, 2, 4)).nonzero().tolist()}
    assert written <= seen                                   # and nothing else was written


def test_in_place_rotation_and_one_row():
    from frink_b200 import device
    pg = device.Pages.alloc(1, 8, 16, 2, 64, 1, 4)
    device.pages_grow(pg, 1)
    q, k, v = (queries(1, h * 64, h).cuda() for h in (8, 2, 3))
    want = plain.rotate(q, 8, [0], 1e4, False)
    r = device.rope_kv_paged(q, k, v[:, :128], pg, 0, 8, 1e4, out=q)
    assert r.data_ptr() == q.data_ptr() and rel_l2(q.cpu().numpy(), want.numpy()) <= 5e-7


# ---- the pool's bookkeeping
def same(pg, ref):
    assert torch.equal(pg.table.cpu(), ref.table())
    assert pg.lens.cpu().tolist() == ref.lens and pg.refs.cpu().tolist() == ref.refs
    assert torch.equal(pg.data.cpu(), ref.data)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("page,n_kv,hd,n_layers,n_pages", [(16, 2, 64, 3, 40), (32, 1, 8, 1, 5000), (128, 3, 80, 2, 17)])
def test_pool_against_lists(dtype, page, n_kv, hd, n_layers, n_pages):
    """Random grows, forks, frees and compactions, every step compared whole."""
    from frink_b200 import device
    n_seqs, max_pages = 6, n_pages
    pg = device.Pages.alloc(n_layers, n_pages, page, n_kv, hd, n_seqs, max_pages, dtype=TYPES[dtype])
    pg.data.copy_(torch.randn(pg.data.shape, generator=torch.Generator().manual_seed(1)))
    ref = plain.Pool(pg.data.cpu().clone(), n_seqs, max_pages)
    rng = np.random.default_rng(n_pages)
    big = max(2, n_pages * page // 20)
    for step in range(40):
        op = rng.integers(0, 5)
        if op <= 1:
            n = rng.integers(0, big, n_seqs) * (rng.random(n_seqs) < 0.5)
            need = sum(max(0, -(-(l + int(a)) // page) - len(r)) for l, a, r in zip(ref.lens, n, ref.rows))
            if need > ref.refs.count(0):
                continue
            nd = torch.tensor(n, dtype=torch.int32).cuda()
            device.pages_grow(pg, nd)
            device.pages_advance(pg, nd)
            ref.grow(n.tolist())
            ref.advance(n.tolist())
        elif op == 2:
            empty = [s for s in range(n_seqs) if not ref.rows[s]]
            full = [s for s in range(n_seqs) if ref.rows[s]]
            if not empty or not full:
                continue
            src = rng.choice(full, len(empty)).tolist()
            cut = None if rng.random() < 0.5 else [int(rng.integers(-1, ref.lens[s] + 1)) for s in src]
            if ref.refs.count(0) < len(src):
                continue
            device.pages_fork(pg, src, empty, cut)
            ref.fork(src, empty, cut)
        elif op == 3:
            seqs = rng.choice(n_seqs, rng.integers(1, 3), replace=False).tolist()
            device.pages_free(pg, seqs)
            ref.free(seqs)
        else:
            assert device.pages_compact(pg).item() == ref.compact()
        same(pg, ref)
    assert device.device_error() == 0


def test_pool_refusals_change_nothing():
    from frink_b200 import device
    pg = device.Pages.alloc(1, 4, 16, 1, 8, 4, 3)
    device.pages_grow(pg, torch.tensor([20, 0, 0, 0], dtype=torch.int32).cuda())
    device.pages_advance(pg, torch.tensor([20, 0, 0, 0], dtype=torch.int32).cuda())
    ref = plain.Pool(pg.data.cpu().clone(), 4, 3)
    ref.grow([20, 0, 0, 0])
    ref.advance([20, 0, 0, 0])
    same(pg, ref)

    def raises(code, fn, *a):
        fn(*a)
        assert device.device_error() == code
        same(pg, ref)

    raises(96, device.pages_grow, pg, 16)                   # three more sequences and one more page than there is
    raises(95, device.pages_grow, pg, torch.tensor([29, 0, 0, 0], dtype=torch.int32).cuda())
    raises(98, device.pages_fork, pg, [0], [1], [21])
    raises(96, device.pages_fork, pg, [0, 0, 0], [1, 2, 3])
    device.pages_fork(pg, [0], [1], [16])
    ref.fork([0], [1], [16])
    raises(98, device.pages_fork, pg, [0], [1])             # it holds something
    raises(98, device.pages_fork, pg, [2], [1], [0])
    device.pages_fork(pg, [2], [3])                         # nothing of nothing
    ref.fork([2], [3])
    same(pg, ref)
    device.pages_free(pg, [0, 1, 2, 3])
    ref.free([0, 1, 2, 3])
    same(pg, ref)
    assert device.pages_compact(pg).item() == 0 and device.device_error() == 0


def test_many_sequences_grow_at_once():
    from frink_b200 import device
    n = 4096
    pg = device.Pages.alloc(1, 9000, 16, 1, 8, n, 5)
    add = torch.tensor(np.random.default_rng(5).integers(0, 50, n), dtype=torch.int32)
    device.pages_grow(pg, add.cuda())
    ref = plain.Pool(pg.data.cpu(), n, 5)
    at, rows = 0, []
    for a in add.tolist():
        k = -(-a // 16)
        rows.append(list(range(at, at + k)))
        at += k
    ref.rows = rows
    assert torch.equal(pg.table.cpu(), ref.table()) and pg.refs.sum().item() == at and device.device_error() == 0


def test_a_captured_step_grows_by_itself():
    """Grow, append, attend and advance in one graph, replayed over page edges, against the same steps one by one."""
    from frink_b200 import device
    heads, n_kv, hd = 8, 2, 64

    def fresh():
        pg = device.Pages.alloc(1, 40, 16, n_kv, hd, 3, 12, dtype=torch.float16)
        device.pages_grow(pg, torch.tensor([14, 0, 31], dtype=torch.int32).cuda())
        device.pages_advance(pg, torch.tensor([14, 0, 31], dtype=torch.int32).cuda())
        return pg

    q, k, v = (queries(3, h * hd, h).cuda() for h in (heads, n_kv, 3))
    v = v[:, :n_kv * hd]

    def step(pg):
        device.pages_grow(pg, 1)
        r = device.rope_kv_paged(q, k, v, pg, 0, heads, 1e4)
        o = device.attention_paged(r, pg, 0, heads)
        device.pages_advance(pg, 1)
        return o

    one, two = fresh(), fresh()
    warm = fresh()
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(two)
    for i in range(40):
        q.copy_(queries(3, heads * hd, 100 + i))
        graph.replay()
        assert torch.equal(step(one), out)
    assert torch.equal(one.table, two.table) and torch.equal(one.refs, two.refs) and torch.equal(one.data, two.data) and one.lens.tolist() == [54, 40, 71]
    assert device.device_error() == 0


def test_two_caches_on_two_streams():
    """Caches with workspaces of their own may be read at the same time."""
    from frink_b200 import device
    made = [cache([900 + 7 * i], [1], 2, 64, 16, torch.bfloat16, seed=20 + i) for i in range(2)]
    qs = [queries(1, 16 * 64, 30 + i) for i in range(2)]
    want = [plain.attention(q, d[0], pg.table.cpu().tolist(), pg.lens.tolist(), 16, [1])[0].numpy() for (pg, d), q in zip(made, qs)]
    qd = [q.cuda() for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(device.attention_paged(qd[i], made[i][0], 0, 16))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert rel_l2(o.cpu().numpy(), want[i]) <= TOL


def test_a_server_round():
    """Prompts, decode steps, a fork, a free and a compaction, as a serving loop has them: after each, attention over the
    pages is attention over the sequence's own tokens."""
    from frink_b200 import device
    heads, n_kv, hd, page = 12, 4, 64, 16
    pg = device.Pages.alloc(2, 30, page, n_kv, hd, 4, 8, dtype=torch.bfloat16)
    hist = [[] for _ in range(4)]                            # (k, v) per token, as stored
    rng = [0]

    def feed(view, s, n):
        rng[0] += 1
        q, k, v = (queries(n, h * hd, 50 * rng[0] + j).cuda() for j, h in enumerate((heads, n_kv, n_kv)))
        device.pages_grow(view, n)
        for layer in (0, 1):
            r = device.rope_kv_paged(q, k, v, view, layer, heads, 1e4)
            o = device.attention_paged(r, view, layer, heads, window=40, first=2)
        base = len(hist[s])
        rk = plain.rotate(k, n_kv, list(range(base, base + n)), 1e4, False).float().bfloat16()
        hist[s] += [(rk[i], v[i].cpu().bfloat16()) for i in range(n)]
        device.pages_advance(view, n)
        kc = torch.stack([a for a, _ in hist[s]]).view(-1, n_kv, hd).permute(1, 0, 2)
        vc = torch.stack([b for _, b in hist[s]]).view(-1, n_kv, hd).permute(1, 0, 2)
        one = torch.stack([kc, vc])[None]                   # one page that holds everything
        want, _ = plain.attention(r, one, [[0]], [base], heads, [n], window=40, first=2)
        # a rotated key may be rounded to the other neighbour than the plain one: one in some hundred, each by 2^-8
        assert rel_l2(o.cpu().numpy(), want.numpy()) <= 1e-3

    for s, n in ((0, 50), (2, 16), (1, 7)):
        feed(pg.seq(s), s, n)
    for _ in range(3):
        for s in (0, 1, 2):
            feed(pg.seq(s), s, 1)
    device.pages_fork(pg, [0], [3], [37])
    hist[3] = list(hist[0][:37])
    feed(pg.seq(3), 3, 5)
    feed(pg.seq(0), 0, 2)
    device.pages_free(pg, [2])
    hist[2] = []
    used = device.pages_compact(pg)
    assert used.item() == int((pg.refs > 0).sum()) == int((pg.refs[:used.item()] > 0).sum())
    for s in (0, 1, 3):
        feed(pg.seq(s), s, 9)
    feed(pg.seq(2), 2, 20)
    assert device.device_error() == 0


# ---- prompts: 128 (row, head) pairs and more of a KV head go to the tensor cores' tcgen05 kernel
def attend_fast(lens, counts, rows, heads, n_kv, hd, page, dtype, window=0, first=0, sinks=False, seed=0, bad=()):
    """`attend` with the 64-bit restatement as matrix products on the GPU (long prompts); bad: (sequence, key, value) to plant."""
    from frink_b200 import device
    pg, data = cache(lens, counts, n_kv, hd, page, dtype, seed)
    S, grp = len(lens), heads // n_kv
    for s, j, x in bad:
        pg.data[0, pg.table[s, j // page].long(), :, :, j % page] = x
    q = queries(S * rows, heads * hd, seed).cuda()
    sk = torch.randn(heads, generator=torch.Generator().manual_seed(seed)).cuda() if sinks else None
    out = torch.full((S * rows, heads * hd), 7.0, device="cuda")
    device.attention_paged(q, pg, 0, heads, n_new=torch.tensor(counts, dtype=torch.int32).cuda(), window=window, first=first, sinks=sk, out=out)
    assert device.device_error() == 0
    worst = 0.0
    for s in range(S):
        n, T = counts[s], lens[s] + counts[s]
        got = out[s * rows:(s + 1) * rows].view(rows, heads, hd)
        assert (got[n:] == 7.0).all()
        if n == 0:
            continue
        kv = pg.data[0, pg.table[s, :-(-T // page)].long()].permute(1, 2, 0, 3, 4).reshape(2, n_kv, -1, hd)[:, :, :T].double()
        p, j = torch.arange(lens[s], T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
        hide = (j > p) | ((j <= p - window) & (j >= first) if window else torch.zeros_like(j > p))
        clean = torch.ones(n, dtype=torch.bool, device="cuda")
        for ss, jj, _ in bad:
            if ss == s and jj < T:
                clean &= hide[:, jj]
                kv[:, :, jj] = 0
        for h in range(heads):
            x = q[s * rows:s * rows + n, h * hd:(h + 1) * hd].double() @ kv[0, h // grp].T * hd ** -0.5
            x = x.masked_fill(hide, float("-inf"))
            m = x.amax(1, keepdim=True)
            if sinks:
                m = m.clamp(min=float(sk[h]))
            w = (x - m).exp()
            want = w @ kv[1, h // grp] / (w.sum(1, keepdim=True) + ((float(sk[h]) - m).exp() if sinks else 0.0))
            worst = max(worst, rel_l2(got[:n, h][clean].cpu().numpy(), want[clean].cpu().numpy()))
            assert not torch.isfinite(got[:n, h][~clean]).any()
    assert worst <= TOL
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd", [(24, 8, 128), (64, 8, 64), (8, 8, 128), (16, 1, 64), (130, 1, 64), (128, 1, 128), (6, 2, 80), (10, 5, 96), (12, 2, 8), (4, 1, 120)])
@pytest.mark.parametrize("page,rows,lens,counts", [(16, 300, [0], [300]), (64, 257, [700, 3], [257, 100]), (32, 129, [0, 1000, 64], [0, 129, 128]), (128, 200, [129], [200])])
def test_prompt(dtype, heads, n_kv, hd, page, rows, lens, counts):
    attend_fast(lens, counts, rows, heads, n_kv, hd, page, TYPES[dtype], seed=rows)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window,first,sinks", [(1, 0, True), (100, 4, False), (64, 64, True), (300, 70, False), (128, 1000, True), (5000, 3, False)])
def test_prompt_windows(dtype, window, first, sinks):
    attend_fast([900, 0], [400, 333], 400, 16, 2, 64, 32, TYPES[dtype], window=window, first=first, sinks=sinks, seed=window)
    attend_fast([900, 0], [150, 133], 150, 6, 2, 128, 16, TYPES[dtype], window=window, first=first, sinks=sinks, seed=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("x", [float("nan"), float("inf")])
def test_prompt_values_behind_a_mask_do_not_matter(dtype, x):
    """A bad token poisons the rows that see it and no other: in the middle of a causal tile, where a window leaves it behind,
    several at once."""
    attend_fast([100], [300], 300, 16, 2, 64, 16, TYPES[dtype], seed=3, bad=[(0, 390, x)])
    attend_fast([100], [300], 300, 24, 8, 128, 16, TYPES[dtype], seed=4, bad=[(0, 150, x), (0, 152, x), (0, 399, x)])
    attend_fast([100], [300], 300, 6, 2, 80, 16, TYPES[dtype], seed=4, bad=[(0, 150, x), (0, 399, x)])
    attend_fast([500], [300], 300, 16, 2, 64, 64, TYPES[dtype], window=70, first=3, seed=5, bad=[(0, 3, x), (0, 440, x), (0, 600, x), (0, 799, x)])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,window", [(16, 8, 64, 300), (16, 8, 128, 0), (30, 10, 96, 64), (24, 24, 40, 1000)])
def test_prompt_of_several_items_a_cta(dtype, heads, n_kv, hd, window):
    """Hundreds of (row block, KV head) items, some of rows that do not exist, bad tokens in several of them."""
    nan, inf = float("nan"), float("inf")
    attend_fast([0, 90, 200, 31], [1500, 0, 700, 1], 1500, heads, n_kv, hd, 16, TYPES[dtype], window=window, first=5 if window else 0, sinks=True, seed=hd,
                bad=[(0, 700, nan), (0, 702, inf), (0, 1400, inf), (2, 300, nan), (2, 850, inf), (2, 899, nan), (3, 31, inf)])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_long_prompt_keeps_its_precision_and_repeats(dtype):
    a = attend_fast([20000], [256], 256, 4, 1, 128, 128, TYPES[dtype], seed=6)
    assert torch.equal(a, attend_fast([20000], [256], 256, 4, 1, 128, 128, TYPES[dtype], seed=6))


def test_rows_in_any_stride_and_a_wrong_page_of_a_prompt():
    from frink_b200 import device
    pg, data = cache([0], [200], 2, 64, 16, torch.bfloat16, seed=9, stale=0.0)
    wide = torch.randn((200, 16 * 64 + 32), generator=torch.Generator().manual_seed(1)).cuda()
    q = wide[:, 16:16 + 16 * 64]
    assert torch.equal(device.attention_paged(q, pg, 0, 16), device.attention_paged(q.contiguous(), pg, 0, 16))
    pg.table[0, 5] = 1 << 20
    out = device.attention_paged(q, pg, 0, 16)
    assert device.device_error() == 97 and torch.isfinite(out).all()
    pg.table[0, 5], pg.lens[0] = 0, 100
    out.fill_(7.0)
    device.attention_paged(q, pg, 0, 16, out=out)
    assert device.device_error() == 95 and (out == 7.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n_seqs,rows,heads,n_kv,hd", [(33, 1, 4, 1, 64), (40, 1, 6, 2, 128), (300, 1, 3, 1, 8), (170, 3, 6, 1, 64), (512, 1, 8, 1, 64), (513, 1, 8, 1, 64), (200, 3, 16, 2, 64),
                                                       (1000, 1, 2, 2, 128)])
def test_many_sequences(dtype, n_seqs, rows, heads, n_kv, hd):
    """More sequences than a warp's lanes, and around the number from which each item has a CTA of its own."""
    rng = np.random.default_rng(n_seqs)
    lens = rng.integers(0, 200, n_seqs)
    lens[::7] = 0
    counts = rng.integers(0, rows + 1, n_seqs)
    attend(lens.tolist(), counts.tolist(), rows, heads, n_kv, hd, 32, TYPES[dtype], window=100, first=3, sinks=True, seed=n_seqs, ragged=True)


@pytest.mark.parametrize("rows,lens", [(1, [3000, 5]), (300, [0, 77])])
def test_attention_in_place(rows, lens):
    from frink_b200 import device
    pg, _ = cache(lens, [rows] * 2, 2, 128, 16, torch.bfloat16)
    q = queries(2 * rows, 8 * 128, 3).cuda()
    want = device.attention_paged(q, pg, 0, 8)
    assert device.attention_paged(q, pg, 0, 8, out=q) is q and torch.equal(q, want)


def test_a_row_for_all_is_refused():
    from frink_b200 import _lib, device
    pg, _ = cache([5, 9], [1, 1], 1, 64, 16, torch.bfloat16)
    q = queries(1, 64, 3).cuda().expand(2, 64)
    with pytest.raises(_lib.Invalid, match="over one another"):
        device.attention_paged(q, pg, 0, 1)
    with pytest.raises(_lib.Invalid, match="over one another"):
        device.rope_kv_paged(q, q, q, pg, 0, 1, 1e4)


def test_more_missing_pages_than_32_bits_count():
    """4096 sequences that ask for 2^20 pages each: 2^32 in all."""
    from frink_b200 import device
    pg = device.Pages.alloc(1, 50, 16, 1, 8, 4096, 1 << 20)
    device.pages_grow(pg, 1 << 24)
    assert device.device_error() == 96
    assert pg.table[:, :40].max().item() == -1 and pg.refs.sum().item() == 0
    device.pages_grow(pg, torch.zeros(4096, dtype=torch.int32, device="cuda"))
    assert device.device_error() == 0


def test_more_columns_than_the_deal_holds():
    """Tens of thousands of (sequence, block of columns) pairs of 32-bit pages."""
    attend([10, 0], [2050, 7], 2050, 130, 1, 8, 64, torch.float32, window=60, first=2, sinks=True, seed=9, ragged=True)


def test_table_rows_of_two_million_pages():
    """Rows so long that the work of full ones would not be counted in 32 bits."""
    from frink_b200 import device
    n, lens = 512, torch.arange(512, dtype=torch.int32, device="cuda") % 127
    data = torch.randn((1, n, 2, 1, 128, 8), generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    table = torch.full((n, (1 << 21) + 1), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(n, device="cuda").flip(0)
    refs = torch.ones(n, dtype=torch.int32, device="cuda")
    q = queries(n, 16, 5).cuda()
    short = device.attention_paged(q, device.Pages(data, table[:, :1].contiguous(), lens, refs), 0, 2)
    full = device.attention_paged(q, device.Pages(data, table, lens, refs), 0, 2)
    assert device.device_error() == 0 and rel_l2(full.cpu().numpy(), short.cpu().numpy()) <= 2 * TOL
