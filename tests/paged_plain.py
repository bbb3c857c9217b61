"""Plain restatements of the paged cache's operators for the tests: numpy / torch in 64 bits, one sequence, row and head at a
time, and the pool's bookkeeping page by page.  TEST ONLY."""
import numpy as np
import torch


def attention(q, data, table, lens, n_heads, counts, scale=None, window=0, first=0, sinks=None):
    """q [n_seqs * rows, n_heads * hd], data one layer [n_pages, 2, n_kv, page, hd] -> (out f64, which rows are real)."""
    n_pages, _, n_kv, page, hd = data.shape
    S, grp = len(lens), n_heads // n_kv
    R = q.shape[0] // S
    q = q.double().cpu().view(S, R, n_heads, hd)
    kv = data.double().cpu()
    scale = hd ** -0.5 if scale is None else scale
    out, real = torch.zeros(S, R, n_heads, hd, dtype=torch.float64), torch.zeros(S, R, dtype=torch.bool)
    for s in range(S):
        for i in range(counts[s]):
            p = lens[s] + i
            js = [j for j in range(p + 1) if not window or j > p - window or j < first]
            pages, slots = torch.tensor([int(table[s][j // page]) for j in js]), torch.tensor([j % page for j in js])
            real[s, i] = True
            for g in range(n_kv):
                k, v = kv[pages, 0, g, slots], kv[pages, 1, g, slots]
                x = q[s, i, g * grp:(g + 1) * grp] @ k.T * scale
                m = x.amax(1, keepdim=True)
                if sinks is not None:
                    z = sinks.double().cpu()[g * grp:(g + 1) * grp, None]
                    m = torch.maximum(m, z)
                w = (x - m).exp()
                den = w.sum(1, keepdim=True) + ((z - m).exp() if sinks is not None else 0.0)
                out[s, i, g * grp:(g + 1) * grp] = w @ v / den
    return out.view(S * R, -1), real.view(-1)


def rotate(x, heads, at, theta, neox, w=None, eps=0.0):
    """x [n, heads * hd] at positions `at`, f64."""
    n = x.shape[0]
    x = x.double().cpu().view(n, heads, -1)
    hd = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()
    ang = torch.tensor(at, dtype=torch.float64)[:, None, None] * float(np.float32(theta)) ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    i = torch.arange(hd // 2)
    ia, ib = (i, i + hd // 2) if neox else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    y = torch.empty_like(x)
    y[..., ia], y[..., ib] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    return y.reshape(n, -1)


class Pool:
    """The bookkeeping, page by page, on lists; `data` [n_layers, n_pages, 2, n_kv, page, hd] is a CPU tensor."""

    def __init__(self, data, n_seqs, max_pages):
        self.data, self.page, self.max_pages = data, data.shape[4], max_pages
        self.rows, self.lens, self.refs = [[] for _ in range(n_seqs)], [0] * n_seqs, [0] * data.shape[1]

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def grow(self, n):
        want = [-(-(l + a) // self.page) if a else len(r) for l, a, r in zip(self.lens, n, self.rows)]
        assert max(want) <= self.max_pages
        for r, w in zip(self.rows, want):
            while len(r) < w:
                r.append(self._take())

    def advance(self, n):
        self.lens = [a + b for a, b in zip(self.lens, n)]

    def free(self, seqs):
        for s in seqs:
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = [], 0

    def fork(self, src, dst, n=None):
        n = [self.lens[a] if n is None or n[i] < 0 else n[i] for i, a in enumerate(src)]
        # pages are taken for the last parts first, in the order of the list; the shared ones are in use anyway
        tails = [self._take() if k % self.page else None for k in n]
        for a, b, k, t in zip(src, dst, n, tails):
            full = k // self.page
            self.rows[b] = self.rows[a][:full]
            for p in self.rows[b]:
                self.refs[p] += 1
            if t is not None:
                self.data[:, t, :, :, :k % self.page] = self.data[:, self.rows[a][full], :, :, :k % self.page]
                self.rows[b] = self.rows[b] + [t]
            self.lens[b] = k

    def compact(self):
        U = sum(r > 0 for r in self.refs)
        holes = [p for p in range(U) if not self.refs[p]]
        movers = [p for p in range(U, len(self.refs)) if self.refs[p]]
        new = dict(zip(movers, holes))
        for a, b in new.items():
            self.data[:, b] = self.data[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[new.get(p, p) for p in r] for r in self.rows]
        return U

    def table(self):
        return torch.tensor([r + [-1] * (self.max_pages - len(r)) for r in self.rows], dtype=torch.int32)


def rules(logits, history, penalties, bias, mask):
    """(f64 logits, tokens); history / bias / mask: lists, arrays or None."""
    x = logits.double().cpu().numpy().copy()
    n, V = x.shape
    tok = []
    for r in range(n):
        if history is not None:
            rep, freq, pres = (float(v) for v in penalties[r])
            ids, cnt = np.unique([t for t in history[r].tolist() if 0 <= t < V], return_counts=True)
            for t, c in zip(ids.astype(int), cnt):
                y = x[r, t]
                x[r, t] = (y / rep if y > 0 else y * rep) - c * freq - pres
        if bias is not None:
            x[r] += (bias if bias.dim() == 1 else bias[r]).double().cpu().numpy()
        if mask is not None:
            w = (mask if mask.dim() == 1 else mask[r]).cpu().numpy().astype(np.uint32)
            v = np.arange(V)
            x[r, ((w[v // 32] >> (v % 32).astype(np.uint32)) & 1) == 0] = -np.inf
        y = np.where(np.isnan(x[r]), -np.inf, x[r])
        tok.append(int(y.argmax()) if y.max() > -np.inf else -1)
    return x, tok
