"""`tests.cpu_ops` with a paged cache and logit rules: a CPU stand-in for `frink_b200.device`, for the tests of
`frink_b200.decoder` over pages.  TEST ONLY."""
import torch

from tests import paged_plain as plain
from tests.cpu_ops import *  # noqa: F401,F403


class Pages:
    def __init__(self, data, table, lens, refs):
        self.data, self.table, self.lens, self.refs = data, table, lens, refs
        self.n_pages, self.page, self.n_kv, self.head_dim = data.shape[1], data.shape[4], data.shape[3], data.shape[5]
        self.n_seqs, self.max_pages = table.shape

    @classmethod
    def alloc(cls, n_layers, n_pages, page, n_kv, head_dim, n_seqs, max_pages, dtype=torch.bfloat16, device="cpu"):
        i32 = dict(dtype=torch.int32)
        return cls(torch.zeros((n_layers, n_pages, 2, n_kv, page, head_dim), dtype=dtype), torch.full((n_seqs, max_pages), -1, **i32), torch.zeros(n_seqs, **i32),
                   torch.zeros(n_pages, **i32))

    def seq(self, s):
        return Pages(self.data, self.table[s:s + 1], self.lens[s:s + 1], self.refs)


def _counts(pg, n_new):
    return n_new.tolist() if isinstance(n_new, torch.Tensor) else [n_new] * pg.n_seqs


def pages_grow(pg, n_new):
    for s, a in enumerate(_counts(pg, n_new)):
        have, want = -(-int(pg.lens[s]) // pg.page), -(-(int(pg.lens[s]) + a) // pg.page)
        for j in range(have, want):
            if pg.table[s, j] < 0:
                p = int((pg.refs == 0).nonzero()[0])
                pg.table[s, j], pg.refs[p] = p, 1


def pages_advance(pg, n_new):
    pg.lens += torch.tensor(_counts(pg, n_new), dtype=torch.int32)


def pages_free(pg, seqs):
    for s in seqs:
        for p in pg.table[s][pg.table[s] >= 0].tolist():
            pg.refs[p] -= 1
        pg.table[s], pg.lens[s] = -1, 0


def pages_fork(pg, src, dst, n=None):
    for i, (a, b) in enumerate(zip(src, dst)):
        k = int(pg.lens[a]) if n is None or n[i] < 0 else n[i]
        full = k // pg.page
        pg.table[b, :full] = pg.table[a, :full]
        for p in pg.table[a, :full].tolist():
            pg.refs[p] += 1
        if k % pg.page:
            p = int((pg.refs == 0).nonzero()[0])
            pg.refs[p], pg.table[b, full] = 1, p
            pg.data[:, p, :, :, :k % pg.page] = pg.data[:, pg.table[a, full], :, :, :k % pg.page]
        pg.lens[b] = k


def rope_kv_paged(q, k, v, pg, layer, n_heads, theta, neox=False, n_new=None, q_norm=None, k_norm=None, eps=0.0, out=None):
    rows = q.shape[0] // pg.n_seqs
    counts = [rows] * pg.n_seqs if n_new is None else n_new.tolist()
    at = [int(pg.lens[r // rows]) + r % rows for r in range(q.shape[0])]
    rk = plain.rotate(k, pg.n_kv, at, theta, neox, k_norm, eps).float()
    for r, p in enumerate(at):
        if r % rows < counts[r // rows]:
            pg.data[layer, pg.table[r // rows, p // pg.page], 0, :, p % pg.page] = rk[r].view(pg.n_kv, -1).to(pg.data.dtype)
            pg.data[layer, pg.table[r // rows, p // pg.page], 1, :, p % pg.page] = v[r].view(pg.n_kv, -1).to(pg.data.dtype)
    return plain.rotate(q, n_heads, at, theta, neox, q_norm, eps).float()


def attention_paged(q, pg, layer, n_heads, n_new=None, scale=None, window=0, first=0, sinks=None, out=None):
    rows = q.shape[0] // pg.n_seqs
    counts = [rows] * pg.n_seqs if n_new is None else n_new.tolist()
    o, real = plain.attention(q, pg.data[layer], pg.table.tolist(), pg.lens.tolist(), n_heads, counts, scale, window, first, sinks)
    r = torch.zeros_like(q) if out is None else out
    r[real] = o[real].float()
    return r


def logit_rules(logits, history=None, penalties=None, bias=None, mask=None, out=None, tokens=None):
    x, t = plain.rules(logits, history, penalties, bias, mask)
    return torch.from_numpy(x).float(), torch.tensor(t, dtype=torch.int32)
