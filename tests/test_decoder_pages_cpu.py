"""`Decoder` over a paged cache on the CPU stand-ins: the host's account of the pool, refusals, and the same tokens as the
contiguous caches."""
import numpy as np
import pytest
import torch

from frink_b200.decoder import Decoder, LogitRules, _PoolMirror
from oracle import frink_oracle as fo
from tests import paged_ops
from tests.helpers import tiny_gpt_oss


def model(**kw):
    cfg, layers, tok, out_norm, head = tiny_gpt_oss()
    for k, v in kw.items():
        setattr(cfg, k, v)
    return Decoder(cfg, layers, tok, fo.BF16, out_norm, output=head, output_kind=fo.BF16, max_seq=64, ops=paged_ops, device="cpu")


def ids(n, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 512, n).astype(np.int32))


def test_the_mirror_counts_as_the_pool_does():
    m = _PoolMirror(3, 6, 16, 4)
    m.grow([20, 0, 16])
    m.advance([20, 0, 16])
    assert len(m.refs) == 3
    saved = m.save()
    m.fork([0], [1], [20])
    assert len(m.refs) == 4 and m.lens == [20, 20, 16]           # one page shared, one of its own
    with pytest.raises(ValueError, match="free"):
        m.grow([13, 13, 1])                                       # 1 + 1 + 1 pages, 2 free
    with pytest.raises(ValueError, match="free it first"):
        m.fork([0], [2], [1])
    with pytest.raises(ValueError, match="table row"):
        m.grow([45, 0, 0])
    m.free([0])
    assert len(m.refs) == 3 and m.lens == [0, 20, 16]             # the shared page stays
    m.free([1, 2])
    assert not m.refs
    m.restore(saved)
    assert m.lens == [20, 0, 16] and len(m.refs) == 3


def test_paged_tokens_are_the_contiguous_caches_tokens():
    prompt = ids(11, 1)
    want = model().generate(prompt, 5)
    dec = model()
    dec.alloc_pages(2, 6, page=16, dtype=torch.float32)
    tok = dec.prefill_pages(1, prompt)
    got = [int(tok)]
    cur = torch.zeros(2, dtype=torch.int32)
    for _ in range(4):
        cur[1] = tok[-1:]
        tok = dec.step_pages(cur)
        got.append(int(tok[1]))
    assert got == want and dec._pool.lens == dec.pages.lens.tolist() == [0, 15]


def test_chunks_forks_and_frees():
    prompt = ids(21, 2)
    one = model()
    one.alloc_pages(4, 12, page=16, dtype=torch.bfloat16)
    whole = one.forward_pages_seq(0, prompt)
    one.forward_pages_seq(1, prompt[:17])
    assert torch.allclose(one.forward_pages_seq(1, prompt[17:]), whole, rtol=0, atol=2e-2 * float(whole.abs().max()))
    one.fork_pages([0, 0], [2, 3], [None, 17])
    b = one.forward_pages_seq(3, prompt[17:])
    assert torch.allclose(b, whole, rtol=0, atol=2e-2 * float(whole.abs().max()))
    cur = torch.tensor([5, 5, 5, 5], dtype=torch.int32)
    lg = one.forward_pages(cur)
    assert torch.equal(lg[0], lg[2])
    one.free_pages([0, 3])
    assert one.page_live.tolist() == [0, 1, 1, 0]
    lg2 = one.forward_pages(cur)
    assert torch.isfinite(lg2[[1, 2]]).all() and one._pool.lens == one.pages.lens.tolist() == [0, 23, 23, 0]
    for bad in (lambda: one.fork_pages([1], [2]), lambda: one.fork_pages([1, 1], [0, 0]), lambda: one.fork_pages([1], [0], [99]), lambda: one.free_pages([1, 1]),
                lambda: one.forward_pages_seq(0, ids(65, 1)), lambda: one.forward_pages(cur[:3])):
        with pytest.raises(ValueError):
            bad()
    assert one._pool.lens == one.pages.lens.tolist()


def test_first_tokens_need_pages():
    dec = model(first_tokens=2)
    with pytest.raises(ValueError, match="paged"):
        dec.forward(ids(12, 1))
    dec.alloc_pages(1, 4, dtype=torch.float32)
    with_first = dec.forward_pages_seq(0, ids(30, 3))
    dec2 = model()
    dec2.alloc_pages(1, 4, dtype=torch.float32)
    assert not torch.allclose(with_first, dec2.forward_pages_seq(0, ids(30, 3)), atol=1e-3)


def test_rules_pick_and_remember():
    r = LogitRules(2, penalties=(1.0, 0.0, 100.0), last=3, device="cpu")
    r.see(0, torch.tensor([7, 1, 2, 3], dtype=torch.int32))      # only 1, 2, 3 stay
    lg = torch.zeros(2, 8)
    lg[:, [1, 2, 3, 7]] = torch.tensor([5.0, 4.0, 3.0, 2.0])
    assert r.pick(paged_ops, lg).tolist() == [7, 1]
    assert r.pick(paged_ops, lg).tolist() == [1, 2]              # 1 has left row 0's history
    assert sorted(r.history[0].tolist()) == [1, 3, 7] and sorted(r.history[1].tolist()) == [-1, 1, 2]
    r.copy(0, 1)
    assert torch.equal(r.history[0], r.history[1])
    r.forget(1)
    assert r.history[1].tolist() == [-1, -1, -1]
    with pytest.raises(ValueError):
        LogitRules(2, penalties=(1.0, 0.0), device="cpu")


def test_generate_under_a_grammar_ends_where_nothing_may_follow():
    dec = model()
    words = torch.zeros(16, dtype=torch.int32)
    words[3] = 0b1010                                             # tokens 97 and 99 only
    r = LogitRules(1, mask=words, device="cpu")
    assert set(dec.generate(ids(5, 4), 4, rules=r)) <= {97, 99}
    dec.reset()
    words[3] = 0
    assert dec.generate(ids(5, 4), 4, rules=LogitRules(1, mask=words, device="cpu")) == [-1]


def test_sequences_that_are_not_there_are_refused():
    dec = model()
    dec.alloc_pages(3, 8, dtype=torch.float32)
    dec.forward_pages_seq(2, ids(20, 1))
    held = dec._pool.save()
    for call in (lambda: dec.forward_pages_seq(-1, ids(3, 2)), lambda: dec.forward_pages_seq(3, ids(3, 2)), lambda: dec.free_pages([-1]), lambda: dec.fork_pages([-1], [0]),
                 lambda: dec.fork_pages([2], [3]), lambda: dec.fork_pages([2], [0, 1]), lambda: dec.fork_pages([2], [0], [1, 2])):
        with pytest.raises(ValueError):
            call()
    assert dec._pool.save() == held
