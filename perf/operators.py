"""The serving operators over a paged key-value cache: what they are measured on.

  attend   attention of each sequence's newest rows over the pages that hold its keys and values: one row a sequence
           (a decode step) or the rows of a prompt, causal, with an optional window, first tokens that stay visible and
           a sink logit per head (`device.attention_paged`)
  append   rotation of q and k and the append of k and v into the pages (`device.rope_kv_paged`)
  fork     a round of a beam search: losing sequences freed, winners forked, room for the next tokens
           (`device.pages_free`, `pages_fork`, `pages_grow`)
  compact  the pages in use moved to the front of the pool (`device.pages_compact`)
  rules    penalties for repeated tokens, biases and a grammar's mask on logits, and the greedy token (`device.logit_rules`)

The cache of all layers is data [layers, pages, 2 (K, V), kv heads, page, head_dim]; table [sequences, pages a sequence may
hold] names a sequence's pages in order (-1: none), lens [sequences] counts the tokens it holds and refs [pages] the
sequences that hold a page.  Head counts and vocabularies are those of the benchmark's three models and their
neighbourhood."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ----------------------------------------------------------------
def listed():
    return [
        # the first step after a one-line prompt: latency is all there is
        _attend("decode 1x17 f32", seqs=1, len=17, rows=1, heads=24, kv=8, head_dim=128, page=16, type="f32"),
        # a decode batch in mid-conversation
        _attend("decode 8x4000 bf16", seqs=8, len=4000, rows=1, heads=24, kv=8, head_dim=128, page=16, type="bf16"),
        # one user with a very long document: the split over the length is everything
        _attend("decode 1x131071 f16 sinks", seqs=1, len=131071, rows=1, heads=64, kv=8, head_dim=64, page=64, type="f16", sinks=True),
        # a full server: ragged lengths, windowed layers whose first tokens stay visible
        _attend("decode 64x16000 window bf16", seqs=64, len=16000, rows=1, heads=32, kv=4, head_dim=128, page=32, type="bf16", ragged=True,
                window=4096, first=4),
        # a prompt of ordinary length into an empty cache
        _attend("prompt 512 bf16", seqs=1, len=0, rows=512, heads=24, kv=8, head_dim=128, page=16, type="bf16"),
        # chunks of several long prompts, windowed, ragged
        _attend("prompt 4x1001 window f16", seqs=4, len=8000, rows=1001, heads=64, kv=8, head_dim=64, page=64, type="f16", ragged=True,
                window=2048, first=4, sinks=True),
        # the append of a decode step
        dict(name="append 8 rows bf16", op="append", seqs=8, len=5000, rows=1, heads=24, kv=8, head_dim=128, page=16, type="bf16", neox=False, norm=False,
             theta=500000.0),
        # the append of a prompt's last chunk, far into the context, with the per-head norms
        dict(name="append 4096 rows f16 far", op="append", seqs=1, len=125001, rows=4096, heads=32, kv=4, head_dim=128, page=32, type="f16", neox=True,
             norm=True, theta=1000000.0),
        # four beams replaced in a cache of every layer
        dict(name="fork 4 of 1000 bf16", op="fork", forks=4, len=1000, layers=28, kv=8, head_dim=128, page=16, type="bf16"),
        # a pool after hours of arrivals and departures, pushed together
        dict(name="compact 2048 pages bf16", op="compact", pages=2048, used=1200, moves=500, layers=28, kv=8, head_dim=128, page=16, type="bf16"),
        # one sequence's rules, no grammar
        dict(name="rules 1x128256", op="rules", rows=1, vocab=128256, history=64, mask=False, bias=False),
        # a batch under a grammar, long histories, the largest vocabulary
        dict(name="rules 64x201088 grammar", op="rules", rows=64, vocab=201088, history=1000, mask=True, bias=True),
    ]


def _attend(name, **kw):
    return dict(dict(name=name, op="attend", ragged=False, window=0, first=0, sinks=False), **kw)


def _lg(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv, head_dim = rng.choice([(24, 8, 128), (32, 4, 128), (64, 8, 64), (32, 8, 128), (8, 8, 64), (6, 2, 80), (16, 1, 128), (5, 5, 96)])
    page, typ = rng.choice([16, 32, 64, 128]), rng.choice(["f32", "f16", "bf16", "bf16"])
    op = rng.choice(["decode", "decode", "prompt", "append", "fork", "compact", "rules"])
    if op in ("decode", "prompt"):
        if op == "decode":
            seqs = _lg(rng, 1, 64)
            length, rows = _lg(rng, 1, min(131072, 200000 // seqs)), rng.choice([1, 1, 1, 2, 5])
        else:
            seqs, rows = rng.randint(1, 4), _lg(rng, 9, 900)
            length = rng.choice([0, _lg(rng, 1, 8000)])
        return dict(op="attend", seqs=seqs, len=length, rows=rows, heads=heads, kv=kv, head_dim=head_dim, page=page, type=typ, ragged=rng.random() < 0.5,
                    window=rng.choice([0, 0, 128, _lg(rng, 1, 8000)]), first=rng.choice([0, 0, 1, 4, 70]), sinks=rng.random() < 0.3)
    if op == "append":
        seqs = _lg(rng, 1, 64)
        return dict(op="append", seqs=seqs, len=_lg(rng, 1, 131072 // seqs), rows=1 if rng.random() < 0.5 else _lg(rng, 2, max(2, 4000 // seqs)), heads=heads, kv=kv,
                    head_dim=head_dim, page=page, type=typ, neox=rng.random() < 0.5, norm=rng.random() < 0.5, theta=rng.choice([10000.0, 150000.0, 1000000.0]))
    if op == "fork":
        return dict(op="fork", forks=rng.randint(1, 16), len=_lg(rng, 3, 4000), layers=rng.randint(1, 32), kv=kv, head_dim=head_dim, page=page, type=typ)
    if op == "compact":
        pages = _lg(rng, 16, 1024 * 16 // page)
        used = rng.randint(pages // 4, pages * 3 // 4)
        return dict(op="compact", pages=pages, used=used, moves=rng.randint(0, min(used, pages - used)), layers=rng.randint(1, 16), kv=kv, head_dim=head_dim,
                    page=page, type=typ)
    return dict(op="rules", rows=_lg(rng, 1, 64), vocab=_lg(rng, 2000, 201088), history=rng.choice([0, _lg(rng, 1, 4000)]), mask=rng.random() < 0.5,
                bias=rng.random() < 0.5)


# ---- sizes that follow from a case -----------------------------------------------
def _lengths(c):
    """Tokens every sequence holds before the rows of the call."""
    n = c["seqs"]
    return [c["len"] * (i + 1) // n if c.get("ragged") else c["len"] for i in range(n)]


def _counts(c):
    """Rows every sequence really has (a prompt's last chunk is shorter than the batch is wide)."""
    return [max(0, c["rows"] - (i % 4) * (c["rows"] // 5)) if c.get("ragged") and c["rows"] > 1 else c["rows"] for i in range(c["seqs"])]


def _cdiv(a, b):
    return -(-a // b)


# ---- inputs -----------------------------------------------------------------------
def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g).mul_(scale)


def _scattered(g, c, held):
    """A table of pages in random order and the pool's reference counts; held: pages of every sequence."""
    n_pages = sum(held) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(held), max(held)), -1, dtype=torch.int32, device="cuda")
    refs, at = torch.zeros(n_pages, dtype=torch.int32, device="cuda"), 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    refs[order[:at].long()] = 1
    return table, refs, n_pages


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, op = dict(case), case["op"]
    st = {"case": c}
    if op in ("attend", "append"):
        lens, counts = _lengths(c), _counts(c)
        held = [max(1, _cdiv(a + b, c["page"])) for a, b in zip(lens, counts)]
        st["table"], st["refs"], n_pages = _scattered(g, c, held)
        st["data"] = _normal(g, (1, n_pages, 2, c["kv"], c["page"], c["head_dim"]), TYPES[c["type"]])
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["n_new"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if c.get("ragged") and c["rows"] > 1 else None
        n, hd = c["seqs"] * c["rows"], c["head_dim"]
        st["q"] = _normal(g, (n, c["heads"] * hd), scale=1.5)
        if op == "attend":
            st["sinks"] = _normal(g, (c["heads"],)) if c["sinks"] else None
            st["out"] = torch.zeros((n, c["heads"] * hd), dtype=torch.float32, device="cuda")
        else:
            st["k"], st["v"] = _normal(g, (n, c["kv"] * hd)), _normal(g, (n, c["kv"] * hd))
            st["q_norm"] = 1 + _normal(g, (hd,), scale=0.1) if c["norm"] else None
            st["k_norm"] = 1 + _normal(g, (hd,), scale=0.1) if c["norm"] else None
    elif op == "fork":
        # sequence 0 .. forks - 1 are alive, forks .. 2 forks - 1 are the losing beams that are replaced
        m, P = c["forks"], c["page"]
        lens = [max(1, c["len"] - 2 * i) for i in range(m)]
        held = [_cdiv(n, P) for n in lens] + [_cdiv(max(1, n // 2), P) for n in lens]
        table, refs, n_pages = _scattered(g, c, held)
        n_pages += 2 * m + sum(held)
        st["table"] = torch.full((2 * m, max(held) + 2), -1, dtype=torch.int32, device="cuda")
        st["table"][:, :table.shape[1]] = table
        st["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st["refs"][:refs.numel()] = refs
        st["lens"] = torch.tensor(lens + [max(1, n // 2) for n in lens], dtype=torch.int32, device="cuda")
        st["data"] = _normal(g, (c["layers"], n_pages, 2, c["kv"], P, c["head_dim"]), TYPES[c["type"]])
        st["src"], st["dst"] = list(range(m)), list(range(m, 2 * m))
        st["src_dev"], st["dst_dev"] = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in (st["src"], st["dst"]))
    elif op == "compact":
        U, N, M = c["used"], c["pages"], min(c["moves"], c["used"], c["pages"] - c["used"])
        low = torch.randperm(U, generator=g, device="cuda")[:U - M]
        high = U + torch.randperm(N - U, generator=g, device="cuda")[:M]
        pages = torch.cat([low, high])[torch.randperm(U, generator=g, device="cuda")].to(torch.int32)
        cols = _cdiv(U, 8)
        st["table0"] = torch.full((8, cols), -1, dtype=torch.int32, device="cuda")
        st["table0"].view(-1)[:U] = pages
        st["refs0"] = torch.zeros(N, dtype=torch.int32, device="cuda")
        st["refs0"][pages.long()] = 1
        st["table"], st["refs"] = st["table0"].clone(), st["refs0"].clone()
        st["lens"] = (st["table0"] >= 0).sum(1).to(torch.int32) * c["page"]
        st["data"] = _normal(g, (c["layers"], N, 2, c["kv"], c["page"], c["head_dim"]), TYPES[c["type"]])
    else:
        n, V = c["rows"], c["vocab"]
        st["logits"] = _normal(g, (n, V), scale=3.0)
        # the tokens that came before: a few of them again and again, some places of the list empty
        h = torch.randint(0, V, (n, c["history"]), generator=g, device="cuda")
        h = torch.where(torch.rand((n, c["history"]), generator=g, device="cuda") < 0.3, h % 50, h)
        st["history"] = torch.where(torch.rand((n, c["history"]), generator=g, device="cuda") < 0.1, torch.full_like(h, -1), h).to(torch.int32)
        pen = torch.empty((n, 3), device="cuda")
        pen[:, 0].uniform_(1.0, 1.3, generator=g)
        pen[:, 1].uniform_(0.0, 0.5, generator=g)
        pen[:, 2].uniform_(0.0, 0.5, generator=g)
        st["penalties"] = pen
        st["bias"] = torch.where(torch.rand((V,), generator=g, device="cuda") < 0.01, 2.0, 0.0) if c["bias"] else None
        # a grammar: each row may go on with a thirtieth of the vocabulary
        if c["mask"]:
            words = _cdiv(V, 32)
            bits = (torch.rand((n, words * 32), generator=g, device="cuda") < 0.03).view(n, words, 32)
            weights = (torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")).view(1, 1, 32)
            w = (bits.to(torch.int64) * weights).sum(-1)
            st["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
        else:
            st["mask"] = None
    return st


# ---- one pass -----------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from frink_b200 import device
    c, op = st["case"], st["case"]["op"]
    if op == "rules":
        out, tokens = device.logit_rules(st["logits"], history=st["history"], penalties=st["penalties"], bias=st["bias"], mask=st["mask"])
        return {"logits": out, "tokens": tokens}
    pg = st.get("pages")
    if pg is None:
        pg = st["pages"] = device.Pages(st["data"], st["table"], st["lens"], st["refs"])
    if op == "attend":
        return device.attention_paged(st["q"], pg, 0, c["heads"], n_new=st["n_new"], window=c["window"], first=c["first"], sinks=st["sinks"], out=st["out"])
    if op == "append":
        q = device.rope_kv_paged(st["q"], st["k"], st["v"], pg, 0, c["heads"], c["theta"], neox=c["neox"], n_new=st["n_new"], q_norm=st["q_norm"],
                                 k_norm=st["k_norm"], eps=1e-6)
        return {"q": q, "data": st["data"]}
    if op == "fork":
        device.pages_free(pg, st["dst"])
        device.pages_fork(pg, st["src"], st["dst"])
        device.pages_grow(pg, c["page"])
        return _state(st)
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])
    used = device.pages_compact(pg)
    return dict(_state(st), used=used)


def _state(st):
    """The pool as whole numbers: its bits, tables and counts."""
    return {"data": st["data"].view(torch.int32 if st["data"].dtype == torch.float32 else torch.int16), "table": st["table"], "refs": st["refs"],
            "lens": st["lens"]}


def _run_plain(st):
    return {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact, "rules": _plain_rules}[st["case"]["op"]](st)


def _plain_attend(st):
    c = st["case"]
    S, R, H, KV, hd, P = c["seqs"], c["rows"], c["heads"], c["kv"], c["head_dim"], c["page"]
    T, dev = st["table"].shape[1] * P, st["q"].device
    kv = st["data"][0][st["table"].clamp(min=0).long()].float()                    # [S, pages, 2, KV, P, hd]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, S, KV, T, hd)
    n_new = st["n_new"] if st["n_new"] is not None else torch.full((S,), R, dtype=torch.int32, device=dev)
    at = st["lens"][:, None] + torch.arange(R, device=dev)                          # [S, R]: every row's position
    j = torch.arange(T, device=dev)
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (j > at[..., None] - c["window"]) | (j < c["first"])
    real = torch.arange(R, device=dev) < n_new[:, None]
    held = (j < (st["lens"] + n_new)[:, None])[:, None, :, None]
    k, v = (torch.where(held, x, torch.zeros((), device=dev)) for x in (kv[0], kv[1]))
    q = st["q"].view(S, R, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(S, KV, -1, hd)
    s = (q @ k.transpose(2, 3)).view(S, KV, H // KV, R, T) * hd ** -0.5
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    sinks = st["sinks"].view(1, KV, H // KV, 1, 1) if st["sinks"] is not None else None
    if sinks is not None:
        m = torch.maximum(m, sinks)
    p = (s - m).exp()
    den = p.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + (sinks - m).exp()
    o = ((p.view(S, KV, -1, T) @ v).view(S, KV, H // KV, R, hd) / den).permute(0, 3, 1, 2, 4).reshape(S, R, H * hd)
    return torch.where(real[..., None], o, st["out"].view(S, R, -1)).view(S * R, H * hd)


def _rotated(x, heads, at, c, w):
    """x [n, heads * head_dim] at positions `at` [n]: the per-head norm, then the rotation, angles in 64 bits."""
    n, hd = x.shape[0], c["head_dim"]
    x = x.view(n, heads, hd)
    if w is not None:
        x = x * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt().float() * w
    freq = c["theta"] ** (-torch.arange(0, hd, 2, device=x.device, dtype=torch.float64) / hd)
    a = (at.double()[:, None] * freq)[:, None, :]
    cos, sin = a.cos().float(), a.sin().float()
    if c["neox"]:
        u, v = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat([u * cos - v * sin, u * sin + v * cos], -1).reshape(n, -1)
    u, v = x[..., 0::2], x[..., 1::2]
    return torch.stack([u * cos - v * sin, u * sin + v * cos], -1).reshape(n, -1)


def _plain_append(st):
    c = st["case"]
    S, R, KV, hd, P = c["seqs"], c["rows"], c["kv"], c["head_dim"], c["page"]
    at = (st["lens"][:, None] + torch.arange(R, device="cuda")).view(-1)
    q, k = _rotated(st["q"], c["heads"], at, c, st["q_norm"]), _rotated(st["k"], KV, at, c, st["k_norm"])
    pages = st["table"].long().gather(1, (at.view(S, R) // P).long()).view(-1)
    st["data"][0, pages, 0, :, (at % P).long()] = k.view(-1, KV, hd).to(st["data"].dtype)
    st["data"][0, pages, 1, :, (at % P).long()] = st["v"].view(-1, KV, hd).to(st["data"].dtype)
    return {"q": q, "data": st["data"]}


def _first_free(refs):
    """Page numbers, the free ones first and in ascending order."""
    return torch.sort((refs != 0).int(), stable=True).indices


def _plain_fork(st):
    c, P, table, refs, lens, data = st["case"], st["case"]["page"], st["table"], st["refs"], st["lens"], st["data"]
    src, dst = st["src_dev"], st["dst_dev"]
    # free the losers
    gone = table[dst]
    refs.index_add_(0, gone.clamp(min=0).view(-1).long(), -(gone >= 0).int().view(-1))
    table[dst] = -1
    lens[dst] = 0
    # fork the winners: whole pages shared, the last part copied into the lowest free pages
    n = lens[src]
    full, part = (n // P).long(), (n % P).long()
    col = torch.arange(table.shape[1], device="cuda")
    shared = col < full[:, None]
    rows = table[src]
    refs.index_add_(0, torch.where(shared, rows, 0).view(-1).long(), shared.int().view(-1))
    has = part > 0
    fresh = _first_free(refs)[(has.long().cumsum(0) - 1).clamp(min=0)]
    tail = rows.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    new_row = torch.where(shared, rows, -1)
    new_row = torch.where((col == full[:, None]) & has[:, None], fresh[:, None].int(), new_row)
    table[dst] = new_row
    lens[dst] = n
    refs.index_add_(0, fresh, has.int())
    sp, dp = torch.where(has, tail, rows[:, 0].long()), torch.where(has, fresh, rows[:, 0].long())
    keep = (torch.arange(P, device="cuda") < part[:, None])[:, None, None, :, None]
    data[:, dp] = torch.where(keep, data[:, sp], data[:, dp])
    # room for another page of tokens in every sequence
    have = (lens + P - 1) // P
    want = (lens + c["page"] + P - 1) // P
    missing = (col >= have[:, None]) & (col < want[:, None]) & (table < 0)
    rank = (missing.view(-1).long().cumsum(0) - 1).clamp(min=0)
    page = _first_free(refs)[rank]
    table.copy_(torch.where(missing, page.view(table.shape).int(), table))
    refs.index_add_(0, page, missing.view(-1).int())
    return _state(st)


def _plain_compact(st):
    table, refs, data = st["table"], st["refs"], st["data"]
    table.copy_(st["table0"])
    refs.copy_(st["refs0"])
    used = refs > 0
    n_used = used.sum()
    at = torch.arange(refs.numel(), device="cuda")
    to, frm = (~used & (at < n_used)).nonzero()[:, 0], (used & (at >= n_used)).nonzero()[:, 0]
    data[:, to] = data[:, frm]
    new = at.clone()
    new[frm] = to
    refs[to] = refs[frm]
    refs[frm] = 0
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].int(), table))
    return dict(_state(st), used=n_used.int().view(1))


def _plain_rules(st):
    x, h, pen = st["logits"], st["history"], st["penalties"]
    n, V = x.shape
    ok = (h >= 0) & (h < V)
    count = torch.zeros((n, V), device=x.device).scatter_add_(1, torch.where(ok, h, 0).long(), ok.float())
    rep, freq, pres = pen[:, 0:1], pen[:, 1:2], pen[:, 2:3]
    y = torch.where(x > 0, x / rep, x * rep) - count * freq - pres
    x = torch.where(count > 0, y, x)
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["mask"] is not None:
        v = torch.arange(V, device=x.device)
        x = torch.where((st["mask"][:, v // 32] >> (v % 32)) & 1 != 0, x, float("-inf"))
    best = torch.where(x.isnan(), float("-inf"), x).max(1)
    # the lowest of equal ones; -1 where nothing is allowed
    low = torch.where(x == best.values[:, None], torch.arange(V, device=x.device), V).amin(1)
    return {"logits": x, "tokens": torch.where(best.values > float("-inf"), low, -1).int()}


# ---- bytes and operations ----------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    if op == "rules":
        n, V = c["rows"], c["vocab"]
        return {"bytes": n * (8 * V + 4 * c["history"] + 16) + (4 * V if c["bias"] else 0) + (n * V // 8 if c["mask"] else 0), "flops": n * (2 * V + 4 * c["history"])}
    e, row = SIZE[c["type"]], c["kv"] * c["head_dim"]
    if op == "attend":
        keys = pairs = rows = 0
        for base, n in zip(_lengths(c), _counts(c)):
            if n == 0:
                continue
            rows += n
            lo = max(0, base + 1 - c["window"]) if c["window"] else 0
            keys += base + n - lo + min(c["first"], lo)
            for p in range(base, base + n):
                lo = max(0, p + 1 - c["window"]) if c["window"] else 0
                pairs += p + 1 - lo + min(c["first"], lo)
        q = c["heads"] * c["head_dim"]
        return {"bytes": 2 * keys * row * e + 8 * rows * q, "flops": 4 * pairs * q}
    if op == "append":
        n, q = c["seqs"] * c["rows"], c["heads"] * c["head_dim"]
        return {"bytes": n * (8 * q + 8 * row + 2 * row * e), "flops": 6 * n * (q + row)}
    if op == "fork":
        part = sum(max(1, c["len"] - 2 * i) % c["page"] for i in range(c["forks"]))
        table = c["forks"] * _cdiv(c["len"], c["page"]) * 4
        return {"bytes": 2 * part * c["layers"] * 2 * row * e + 6 * table, "flops": 0}
    moves = min(c["moves"], c["used"], c["pages"] - c["used"])
    return {"bytes": 2 * moves * c["layers"] * 2 * row * c["page"] * e + 16 * c["pages"], "flops": 0}


# ---- the definition in 64 bits --------------------------------------------------------
def exact(case, seed):
    c, op = case, case["op"]
    if op in ("fork", "compact"):
        return None                                                # whole numbers only
    st = prepare(case, seed)
    if op == "rules":
        x = st["logits"].double()
        for r in range(c["rows"]):
            ids = st["history"][r]
            ids = ids[(ids >= 0) & (ids < c["vocab"])].long()
            if ids.numel():
                ids, cnt = torch.unique(ids, return_counts=True)
                rep, freq, pres = (float(v) for v in st["penalties"][r])
                y = x[r, ids]
                x[r, ids] = torch.where(y > 0, y / rep, y * rep) - cnt * freq - pres
            if st["bias"] is not None:
                x[r] += st["bias"].double()
            if st["mask"] is not None:
                bits = (st["mask"][r][:, None] >> torch.arange(32, device="cuda")) & 1
                x[r, bits.view(-1)[:c["vocab"]] == 0] = float("-inf")
        return {"logits": x, "tokens": None}
    S, R, H, KV, hd, P = c["seqs"], c["rows"], c["heads"], c["kv"], c["head_dim"], c["page"]
    if op == "append":
        out, data = torch.zeros((S * R, H * hd), dtype=torch.float64, device="cuda"), st["data"].double()
        a = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
        for s, base in enumerate(_lengths(c)):
            pos = torch.arange(base, base + R, device="cuda")
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None, None] * torch.exp(-2 * a / hd * math.log(c["theta"])))
            done = []
            for x, n, w in ((st["q"], H, st["q_norm"]), (st["k"], KV, st["k_norm"])):
                x = x[s * R:(s + 1) * R].double().view(R, n, hd)
                if w is not None:
                    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
                i, k = (a.long(), a.long() + hd // 2) if c["neox"] else (2 * a.long(), 2 * a.long() + 1)
                z = torch.complex(x[..., i], x[..., k]) * turn
                y = torch.empty_like(x)
                y[..., i], y[..., k] = z.real, z.imag
                done.append(y)
            out[s * R:(s + 1) * R] = done[0].reshape(R, -1)
            page, slot = st["table"][s].long()[pos // P], pos % P
            data[0, page, 0, :, slot] = done[1]
            data[0, page, 1, :, slot] = st["v"][s * R:(s + 1) * R].double().view(R, KV, hd)
        return {"q": out, "data": data}
    out = torch.zeros((S, R, H, hd), dtype=torch.float64, device="cuda")
    for s, (base, n) in enumerate(zip(_lengths(c), _counts(c))):
        if n == 0:
            continue
        T = base + n
        pages = st["table"][s, :_cdiv(T, P)].long()
        p = torch.arange(base, T, device="cuda")[:, None]
        j = torch.arange(T, device="cuda")[None]
        hide = j > p
        if c["window"]:
            hide = hide | ((j <= p - c["window"]) & (j >= c["first"]))
        for h in range(H):
            k, v = (st["data"][0, pages, i, h // (H // KV)].reshape(-1, hd)[:T].double() for i in (0, 1))
            x = st["q"][s * R:s * R + n, h * hd:(h + 1) * hd].double() @ k.T / math.sqrt(hd)
            x[hide] = float("-inf")
            top = x.max(1, keepdim=True).values
            if st["sinks"] is not None:
                top = top.clamp(min=float(st["sinks"][h]))
            x = (x - top).exp_()
            den = x.sum(1, keepdim=True)
            if st["sinks"] is not None:
                den = den + (float(st["sinks"][h]) - top).exp()
            out[s, :n, h] = (x @ v) / den
    return out.view(S * R, H * hd)
