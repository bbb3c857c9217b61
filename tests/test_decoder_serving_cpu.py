"""`Decoder` over pages as a server drives it, on the CPU stand-ins: slots that are idle, freed and filled again, under rules."""
import gc
import weakref

import numpy as np
import pytest
import torch

from frink_b200.decoder import Decoder, LogitRules
from oracle import frink_oracle as fo
from tests import paged_ops
from tests.helpers import tiny_gpt_oss

PRESENCE = (1.0, 0.0, 100.0)       # a token that occurred before is not picked again


def model(**kw):
    cfg, layers, tok, out_norm, head = tiny_gpt_oss()
    return Decoder(cfg, layers, tok, fo.BF16, out_norm, output=head, output_kind=fo.BF16, max_seq=64, ops=paged_ops, device="cpu", **kw)


def ids(n, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 512, n).astype(np.int32))


def alone(prompt, n, **kw):
    """The tokens of a sequence that is the only one, in a cache of its own."""
    dec, rules = model(), LogitRules(1, device="cpu", **kw)
    dec.alloc_pages(1, 4, page=16, dtype=torch.float32)
    cur = dec.prefill_pages(0, prompt, rules)
    out = [int(cur)]
    for _ in range(n - 1):
        cur = dec.step_pages(cur, rules)
        out.append(int(cur))
    return out


def steps(dec, rules, cur, n, slot):
    """n more steps of all slots -> slot's tokens."""
    out = []
    for _ in range(n):
        cur.copy_(dec.step_pages(cur, rules))
        out.append(int(cur[slot]))
    return out


def serving(n_seqs=2, **kw):
    dec, rules = model(), LogitRules(n_seqs, penalties=PRESENCE, device="cpu", **kw)
    dec.alloc_pages(n_seqs, 4 * n_seqs, page=16, dtype=torch.float32)
    return dec, rules, torch.zeros(n_seqs, dtype=torch.int32)


@pytest.mark.parametrize("seed", range(3))
def test_a_slot_that_was_idle_answers_as_a_sequence_alone(seed):
    dec, rules, cur = serving()
    cur[0] = dec.prefill_pages(0, ids(9, seed), rules)
    steps(dec, rules, cur, 12, 0)
    assert rules.history[1].tolist() == [-1] * 64 and int(rules.at[1]) == 0
    prompt = ids(7, 50 + seed)
    cur[1] = dec.prefill_pages(1, prompt, rules)
    assert [int(cur[1])] + steps(dec, rules, cur, 5, 1) == alone(prompt, 6, penalties=PRESENCE)


@pytest.mark.parametrize("forget", [False, True])
def test_a_slot_that_was_freed_and_idle_answers_as_a_sequence_alone(forget):
    dec, rules, cur = serving()
    for s in range(2):
        cur[s] = dec.prefill_pages(s, ids(8 + s, s), rules)
    steps(dec, rules, cur, 6, 1)
    dec.free_pages([1])
    if forget:
        rules.forget(1)
    before = rules.history[1].clone()
    steps(dec, rules, cur, 5, 0)
    assert torch.equal(rules.history[1], before)
    prompt = ids(6, 77)
    cur[1] = dec.prefill_pages(1, prompt, rules)
    assert [int(cur[1])] + steps(dec, rules, cur, 5, 1) == alone(prompt, 6, penalties=PRESENCE)


@pytest.mark.parametrize("last", [3, 64])
def test_a_prompt_in_chunks_is_remembered_whole(last):
    prompt = ids(23, 5)
    dec, rules, cur = serving(last=last)
    dec.forward_pages_seq(1, prompt[:9], rules)
    dec.forward_pages_seq(1, prompt[9:11], rules)
    cur[1] = dec.prefill_pages(1, prompt[11:], rules)
    assert [int(cur[1])] + steps(dec, rules, cur, 4, 1) == alone(prompt, 5, penalties=PRESENCE, last=last)
    assert sorted(rules.history[1].tolist()) == sorted(([-1] * 64 + prompt.tolist() + alone(prompt, 5, penalties=PRESENCE, last=last))[-last:])


def test_a_picked_token_that_begins_the_next_chunk_is_counted_once():
    """A conversation's second turn: its chunk begins with the last token that was picked, which no step has read yet."""
    prompt, turn = ids(9, 6), ids(4, 7)
    dec, rules, cur = serving(last=32)
    cur[0] = dec.prefill_pages(0, prompt, rules)
    said = [int(cur[0])] + steps(dec, rules, cur, 3, 0)
    whole = prompt.tolist() + said + turn.tolist()
    tok = int(dec.prefill_pages(0, torch.tensor(said[-1:] + turn.tolist(), dtype=torch.int32), rules))
    assert sorted(t for t in rules.history[0].tolist() if t >= 0) == sorted(whole + [tok])
    assert tok == alone(torch.tensor(whole, dtype=torch.int32), 1, penalties=PRESENCE, last=32)[0]


def test_generate_starts_a_history_anew_and_goes_on_with_its_own():
    prompt = ids(8, 9)
    dec, rules = model(), LogitRules(1, penalties=PRESENCE, last=32, device="cpu")
    first = dec.generate(prompt, 5, rules=rules)
    dec.reset()
    assert dec.generate(prompt, 5, rules=rules) == first
    more = ids(3, 10)
    dec.generate(more, 1, rules=rules)                            # behind prompt and all but the last token
    held = [t for t in rules.history[0].tolist() if t >= 0]
    assert len(held) == int(rules.at[0]) == 8 + 4 + 3 + 1
    assert sorted(held[:-1]) == sorted(prompt.tolist() + first[:4] + more.tolist())


def test_a_chunk_that_does_not_fit_leaves_the_history_as_it_was():
    dec, rules, cur = serving()
    cur[0] = dec.prefill_pages(0, ids(60, 1), rules)
    kept = rules.history.clone(), rules.at.clone()
    with pytest.raises(ValueError):
        dec.prefill_pages(0, ids(5, 2), rules)
    assert torch.equal(rules.history, kept[0]) and torch.equal(rules.at, kept[1])


def grammar(dec, n_seqs):
    """Rules under which every token may follow, a row of words for each sequence (clear it: nothing may)."""
    words = torch.full((n_seqs, dec.cfg.vocab // 32), -1, dtype=torch.int32)
    return words, LogitRules(n_seqs, penalties=PRESENCE, mask=words, device="cpu")


def test_a_sequence_that_nothing_may_follow_stays_as_it_is():
    dec, _, cur = serving()
    words, rules = grammar(dec, 2)
    for s in range(2):
        cur[s] = dec.prefill_pages(s, ids(8 + s, s), rules)
    before = steps(dec, rules, cur, 2, 0)
    words[1] = 0
    assert steps(dec, rules, cur, 1, 1) == [-1]                  # this step still read the token before
    kept = dec.pages.lens[1].item(), dec.pages.table[1].clone(), rules.history[1].clone(), rules.at[1].item()
    assert kept[0] == kept[3] == 9 + 3
    after, data = steps(dec, rules, cur, 1, 0), dec.pages.data[:, dec.pages.table[1, 0]].clone()
    after += steps(dec, rules, cur, 6, 0)
    assert cur[1] == -1 and kept[0] == dec.pages.lens[1] and torch.equal(kept[1], dec.pages.table[1])
    assert torch.equal(kept[2], rules.history[1]) and kept[3] == rules.at[1] and torch.equal(data, dec.pages.data[:, dec.pages.table[1, 0]])
    first = alone(ids(8, 0), 11, penalties=PRESENCE)
    assert first[1:3] == before and first[4:] == after
    words[1] = -1                                                # the grammar lets it go on, with a token of the caller's
    cur[1] = 7
    cur.copy_(dec.step_pages(cur, rules))
    assert cur[1] >= 0 and dec.pages.lens.tolist() == [8 + 3 + 8, kept[0] + 1]


def test_a_prompt_that_nothing_may_follow():
    dec, _, cur = serving()
    words, rules = grammar(dec, 2)
    words[0] = 0
    cur[0] = dec.prefill_pages(0, ids(8, 1), rules)
    assert cur[0] == -1 and rules.at[0] == 8
    cur[1] = dec.prefill_pages(1, ids(6, 2), rules)
    assert steps(dec, rules, cur, 4, 1) == alone(ids(6, 2), 5, penalties=PRESENCE)[1:] and cur[0] == -1
    assert dec.pages.lens.tolist() == [8, 10]


def test_the_account_follows_sequences_that_have_ended():
    """Pages that an ended sequence would have taken are there for the others; forks take what it holds."""
    dec = model()
    dec.alloc_pages(3, 4, page=16, dtype=torch.float32, max_tokens=48)
    words, rules = grammar(dec, 3)
    cur = torch.zeros(3, dtype=torch.int32)
    words[0] = 0
    cur[0] = dec.prefill_pages(0, ids(16, 1), rules)              # one page, full
    cur[1] = dec.prefill_pages(1, ids(30, 2), rules)              # two pages
    steps(dec, rules, cur, 18, 1)                                 # a third one: the pool is full, and so is sequence 1 with 48 tokens
    assert dec.pages.lens.tolist() == dec._pool.lens == [16, 48, 0] and len(dec._pool.refs) == 4
    with pytest.raises(ValueError):
        dec.step_pages(cur, rules)                                # sequence 1 has a token that does not fit
    words[1] = 0
    cur[1] = -1
    assert dec.step_pages(cur, rules).tolist() == [-1, -1, -1]    # ... and without one the step leaves all of them out
    dec.fork_pages([0], [2])
    assert dec.pages.lens.tolist() == dec._pool.lens == [16, 48, 16]
    dec.free_pages([1, 0])
    assert dec._pool.lens == [0, 0, 16] and len(dec._pool.refs) == 1 and dec.pages.refs.sum() == 1


def test_a_fork_of_an_ended_sequence_takes_what_it_holds():
    dec, _, cur = serving(3)
    words, rules = grammar(dec, 3)
    words[0] = 0
    cur[0] = dec.prefill_pages(0, ids(15, 1), rules)
    cur[1] = dec.prefill_pages(1, ids(15, 2), rules)
    steps(dec, rules, cur, 5, 1)
    with pytest.raises(ValueError, match="holds 15"):
        dec.fork_pages([0], [2], [16])
    dec.fork_pages([0], [2])
    assert dec.pages.lens.tolist() == dec._pool.lens == [15, 20, 15]
    assert len(dec._pool.refs) == int((dec.pages.refs > 0).sum()) == 4
    dec.forward_pages_seq(0, ids(3, 4), rules)                    # it goes on with tokens of the caller's
    assert dec.pages.lens.tolist() == dec._pool.lens and rules.at[0] == 18


def test_negative_tokens_without_rules():
    dec = model()
    dec.alloc_pages(2, 6, page=16, dtype=torch.float32)
    cur = torch.cat([dec.prefill_pages(s, ids(5 + s, s)) for s in range(2)])
    want = dec.step_pages(cur.clone())
    two = model()
    two.alloc_pages(2, 6, page=16, dtype=torch.float32)
    cur = torch.cat([two.prefill_pages(s, ids(5 + s, s)) for s in range(2)])
    cur[0] = -1
    got = two.step_pages(cur)
    assert got.tolist() == [-1, int(want[1])] and two.pages.lens.tolist() == [5, 7]


class _NoGraph:
    """Stands in for a CUDA graph and its capture."""
    inside = False

    def __init__(self, *a):
        pass

    def __enter__(self):
        _NoGraph.inside = True

    def __exit__(self, *a):
        _NoGraph.inside = False


@pytest.mark.parametrize("n", [31, 32])
@pytest.mark.parametrize("n_pages,max_tokens", [(4, 64), (8, 32)])
def test_a_step_is_captured_where_little_or_nothing_fits(monkeypatch, n, n_pages, max_tokens):
    """The pool, or the sequences' table rows, have room for one more token each, or for none (a replay is then refused)."""
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _NoGraph)
    monkeypatch.setattr(torch.cuda, "graph", _NoGraph)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    dec, rules = model(), LogitRules(2, penalties=PRESENCE, device="cpu")
    dec.alloc_pages(2, n_pages, page=16, dtype=torch.float32, max_tokens=max_tokens)
    cur = torch.cat([dec.prefill_pages(s, ids(n, s), rules) for s in range(2)])
    state = lambda: [t.clone() for t in (dec.pages.table, dec.pages.lens, dec.pages.refs, dec.pages.data, rules.history, rules.at)]
    before, seen, run = state(), [], dec._forward_pages_device

    def forward(toks):
        seen.append((toks.tolist(), state()))
        return run(torch.full_like(toks, -1) if _NoGraph.inside else toks)      # a capture runs nothing

    monkeypatch.setattr(dec, "_forward_pages_device", forward)
    dec.capture_pages(cur, rules)
    assert seen[-1][0] == cur.tolist() and dec._pool.lens == dec.pages.lens.tolist() == [n, n]
    for st in [s for _, s in seen] + [state()]:
        assert all(torch.equal(a, b) for a, b in zip(before, st))
    with pytest.raises(ValueError):
        dec.capture_pages(cur[:1], rules)
    if n == 32:
        with pytest.raises(ValueError):
            dec.replay_pages()


def test_a_captured_step_keeps_what_it_reads_and_writes(monkeypatch):
    """The graph holds addresses: the tokens and the rules' tensors live as long as it, whatever becomes of the caller's names."""
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _NoGraph)
    monkeypatch.setattr(torch.cuda, "graph", _NoGraph)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    dec, rules, cur = serving()
    words, rules = grammar(dec, 2)
    rules.bias = torch.zeros(dec.cfg.vocab)
    dec.capture_pages(cur, rules)
    held = [weakref.ref(t) for t in (cur, words, rules.bias, rules.history, rules.at, rules.penalties)]
    rules.bias = rules.mask = None
    del cur, words, rules
    gc.collect()
    assert all(r() is not None for r in held)
    dec.alloc_pages(2, 8)                                         # the graph is gone, and so are they
    gc.collect()
    assert all(r() is None for r in held)


def test_rules_that_do_not_fit_are_refused_before_a_step():
    dec, rules, cur = serving()
    cur[0] = dec.prefill_pages(0, ids(8, 1), rules)
    mask = lambda *shape: torch.full(shape, -1, dtype=torch.int32)
    wrong = [dict(mask=mask(15)), dict(mask=mask(3, 16)), dict(mask=torch.ones(512, dtype=torch.bool)), dict(bias=torch.zeros(511)), dict(bias=torch.zeros(3, 512)),
             dict(bias=torch.zeros(512, dtype=torch.float64))]
    two, one = [LogitRules(2, device="cpu", **kw) for kw in wrong], [LogitRules(1, device="cpu", **kw) for kw in wrong]
    state = lambda: [t.clone() for t in (dec.pages.table, dec.pages.lens, dec.pages.refs, dec.page_live)]
    before, pool = state(), dec._pool.save()
    for r in two + [LogitRules(3, device="cpu"), LogitRules(1, device="cpu")]:
        for call in (dec.step_pages, dec.capture_pages):
            with pytest.raises(ValueError):
                call(cur, r)
    for r in two + [LogitRules(1, device="cpu")]:
        with pytest.raises(ValueError):
            dec.prefill_pages(1, ids(4, 2), r)
    for r in one + [LogitRules(2, device="cpu")]:
        with pytest.raises(ValueError):
            dec.generate(ids(4, 2), 2, rules=r)
    assert all(torch.equal(a, b) for a, b in zip(before, state())) and dec._pool.save() == pool and dec._pos_host == 0
    assert all(int(r.at.sum()) == 0 for r in one + two)
    with pytest.raises(ValueError, match="captured"):
        dec.replay_pages()
    LogitRules(2, bias=torch.zeros(2, 600), mask=mask(20), device="cpu").fits(512, 2)      # longer rows are fine
    for last in (0, 65536):                                       # what the rules' kernel counts in
        with pytest.raises(ValueError, match="65535"):
            LogitRules(2, last=last, device="cpu")
