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
