"""`Decoder` over pages as a server drives it, on the GPU: slots that are idle, freed and filled again, under rules, eagerly and
from a captured step.  A sequence that ran alone is one in a cache of as many slots, so that its rows take the same kernels."""
import numpy as np
import pytest
import torch

from frink_b200.decoder import Decoder, LogitRules
from oracle import frink_oracle as fo
from tests.test_decoder_gpu import small_llama

pytestmark = pytest.mark.gpu

PRESENCE = (1.0, 0.0, 1000.0)      # a token that occurred before is not picked again


def model(**kw):
    cfg, layers, tok, out_norm, head = small_llama(uniform=True)
    return cfg, Decoder(cfg, layers, tok, fo.Q6_K, out_norm, output=head, output_kind=fo.Q6_K, max_seq=96, **kw)


def ids(cfg, n, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, cfg.vocab, n).astype(np.int32)).cuda()


class Server:
    def __init__(self, n_seqs, captured, **kw):
        self.cfg, self.dec = model()
        self.dec.alloc_pages(n_seqs, 6 * n_seqs, page=16, dtype=torch.float32)
        self.rules = LogitRules(n_seqs, **kw)
        self.cur = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
        self.captured = captured
        if captured:
            self.out = self.dec.capture_pages(self.cur, self.rules)[1]

    def prompt(self, s, p):
        self.cur[s:s + 1] = self.dec.prefill_pages(s, p, self.rules)
        return int(self.cur[s])

    def steps(self, n, s):
        got = []
        for _ in range(n):
            if self.captured:
                self.dec.replay_pages()
                self.cur.copy_(self.out)
            else:
                self.cur.copy_(self.dec.step_pages(self.cur, self.rules))
            got.append(int(self.cur[s]))
        return got


@pytest.mark.parametrize("n_seqs", [3, 10])
@pytest.mark.parametrize("captured", [False, True])
def test_idle_and_freed_slots_answer_as_sequences_alone(n_seqs, captured):
    from frink_b200 import device
    one = Server(n_seqs, captured, penalties=PRESENCE)
    first, second, third = (ids(one.cfg, n, n) for n in (9, 7, 12))
    one.prompt(0, first)
    one.steps(8, 0)
    assert one.rules.history[1:].eq(-1).all() and one.rules.at.tolist() == [9 + 1 + 8] + [0] * (n_seqs - 1)
    got = [[one.prompt(1, second)] + one.steps(6, 1)]
    one.dec.free_pages([1])
    one.steps(5, 0)
    got.append([one.prompt(1, third)] + one.steps(6, 1))
    for p, tokens in ((second, got[0]), (third, got[1])):
        solo = Server(n_seqs, False, penalties=PRESENCE)
        assert tokens == [solo.prompt(1, p)] + solo.steps(6, 1)
    assert device.device_error() == 0


def test_chunks_and_generate_keep_the_whole_history():
    from frink_b200 import device
    one, solo = Server(2, False, penalties=PRESENCE, last=20), Server(2, False, penalties=PRESENCE, last=20)
    p = ids(one.cfg, 40, 4)
    one.dec.forward_pages_seq(1, p[:21], one.rules)
    one.dec.forward_pages_seq(1, p[21:24], one.rules)
    a, b = [one.prompt(1, p[24:])], [solo.prompt(1, p)]
    assert torch.equal(one.rules.history, solo.rules.history) and torch.equal(one.rules.at, solo.rules.at)
    assert sorted(one.rules.history[1].tolist()) == sorted((p.tolist() + a)[-20:])
    rules = LogitRules(1, penalties=PRESENCE)
    _, dec = model()
    want = dec.generate(p, 6, rules=rules)
    dec.reset()
    assert dec.generate(p, 6, rules=rules) == want and device.device_error() == 0


@pytest.mark.parametrize("n_seqs", [3, 10])
@pytest.mark.parametrize("captured", [False, True])
def test_a_sequence_that_nothing_may_follow_is_left_out(n_seqs, captured):
    """The grammar of sequence 1 closes, the others go on as if alone; a fork takes what it holds; it opens again."""
    from frink_b200 import device
    words = torch.full((n_seqs, model()[0].vocab // 32), -1, dtype=torch.int32, device="cuda")
    one = Server(n_seqs, captured, penalties=PRESENCE, mask=words)
    dec, rules = one.dec, one.rules
    first, second = ids(one.cfg, 9, 9), ids(one.cfg, 15, 15)
    got = [one.prompt(0, first)]
    one.prompt(1, second)
    got += one.steps(3, 0)
    words[1] = 0
    got += one.steps(1, 0)
    assert one.cur[1] == -1
    kept = dec.pages.lens[1].item(), dec.pages.table[1].clone(), rules.history[1].clone(), rules.at[1].item()
    assert kept[0] == kept[3] == 15 + 4
    data = dec.pages.data[:, dec.pages.table[1, 1]].clone()
    got += one.steps(20, 0)
    assert one.cur[1] == -1 and dec.pages.lens[:2].tolist() == [9 + 24, kept[0]] and rules.at[1] == kept[3]
    assert torch.equal(kept[1], dec.pages.table[1]) and torch.equal(kept[2], rules.history[1]) and torch.equal(data, dec.pages.data[:, dec.pages.table[1, 1]])
    dec.fork_pages([1], [2])
    assert dec._pool.lens[:3] == dec.pages.lens[:3].tolist() == [33, 19, 19] and len(dec._pool.refs) == int((dec.pages.refs > 0).sum())
    words[1] = -1
    one.cur[1] = 7
    one.steps(2, 1)
    assert one.cur[1] >= 0 and dec.pages.lens[:3].tolist() == [35, 21, 19]
    solo = Server(n_seqs, False, penalties=PRESENCE)
    assert got == [solo.prompt(0, first)] + solo.steps(24, 0) and device.device_error() == 0


def test_a_full_sequence_that_has_ended_does_not_stop_the_others():
    from frink_b200 import device
    cfg, dec = model()
    dec.alloc_pages(2, 5, page=16, max_tokens=48)
    words = torch.full((2, cfg.vocab // 32), -1, dtype=torch.int32, device="cuda")
    rules, cur = LogitRules(2, mask=words), torch.zeros(2, dtype=torch.int32, device="cuda")
    cur[1:] = dec.prefill_pages(1, ids(cfg, 48, 1), rules)        # its table row is full
    cur[:1] = dec.prefill_pages(0, ids(cfg, 20, 2), rules)
    g, out = dec.capture_pages(torch.full_like(cur, -1), rules)   # leaves all of them out
    dec.replay_pages()
    assert out.tolist() == [-1, -1] and dec.pages.lens.tolist() == [20, 48]
    with pytest.raises(ValueError):
        dec.step_pages(cur, rules)                                # a token that does not fit
    cur[1] = -1
    for _ in range(12):
        cur.copy_(dec.step_pages(cur, rules))
    assert dec.pages.lens.tolist() == dec._pool.lens == [32, 48] and cur[1] == -1 and device.device_error() == 0


@pytest.mark.parametrize("n", [31, 32])
def test_a_step_is_captured_where_little_or_nothing_fits(n):
    """Room for one more token of each sequence, or for none: the capture moves nothing, a replay is refused where it does not fit."""
    from frink_b200 import device
    cfg, dec = model()
    dec.alloc_pages(2, 4, page=16)
    rules = LogitRules(2, penalties=PRESENCE)
    cur = torch.cat([dec.prefill_pages(s, ids(cfg, n, s), rules) for s in range(2)])
    state = lambda: [t.clone() for t in (dec.pages.table, dec.pages.lens, dec.pages.refs, dec.pages.data, rules.history, rules.at)]
    before = state()
    g, out = dec.capture_pages(cur, rules)
    assert all(torch.equal(a, b) for a, b in zip(before, state())) and dec._pool.lens == [n, n]
    for _ in range(32 - n):
        dec.replay_pages()
        assert dec.pages.lens.tolist() == dec._pool.lens == [32, 32] and min(out.tolist()) >= 0
    with pytest.raises(ValueError):
        dec.replay_pages()
    dec.free_pages([0])
    dec.replay_pages()
    assert dec.pages.lens.tolist() == dec._pool.lens == [0, 33] and device.device_error() == 0
