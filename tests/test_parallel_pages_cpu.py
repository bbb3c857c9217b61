"""The paged decoder over two gloo ranks on the CPU stand-ins: every rank keeps its own heads' pages (or all of them, where
attention is replicated) and the same account, and takes the same collectives; a left-out sequence too."""
import numpy as np
import pytest
import torch

from oracle import frink_oracle as fo
from tests.helpers import rel_l2, tiny_gpt_oss
from tests.test_parallel_cpu import _tiny_model, spawn


def _case(which, world, n_seqs):
    from frink_b200.decoder import Decoder, LogitRules
    from tests import paged_ops
    if which == "oai":
        (cfg, layers, tok, out_norm, head), kind, dense = tiny_gpt_oss(), fo.BF16, False
    else:
        (cfg, layers, tok, out_norm, head), kind, dense = _tiny_model(which == "moe"), fo.Q8_0, True
    dec = Decoder(cfg, layers, tok, kind, out_norm, output=head, output_kind=kind, max_seq=32, ops=paged_ops, device="cpu", dense_parallel=dense)
    assert dec.world == world
    dec.alloc_pages(n_seqs, 3 * n_seqs, page=16, dtype=torch.float32)
    rules = LogitRules(n_seqs, penalties=(1.1, 0.0, 0.5), device="cpu")
    rng, outs = np.random.default_rng(3), []
    ids = lambda n: torch.from_numpy(rng.integers(0, cfg.vocab, n).astype(np.int32))
    outs.append(dec.forward_pages_seq(0, ids(12), rules).numpy().copy())       # many rows
    outs.append(dec.forward_pages_seq(0, ids(3), rules).numpy().copy())        # a few
    dec.fork_pages([0], [1], [14])
    rules.copy(0, 1)
    for t in ([5, 7] + [0] * (n_seqs - 2), [9, -1] + [0] * (n_seqs - 2), [2, 4] + [0] * (n_seqs - 2)):
        outs.append(dec.forward_pages(torch.tensor(t, dtype=torch.int32))[:2].numpy().copy())
    outs.append(dec.step_pages(torch.tensor([3] * n_seqs, dtype=torch.int32), rules).numpy().copy())
    return outs, dec.pages.lens.tolist(), dec._pool.lens


def _dense3(rank, world):
    return _case("dense", world, 3)


def _moe9(rank, world):
    return _case("moe", world, 9)


def _oai3(rank, world):
    return _case("oai", world, 3)


@pytest.mark.parametrize("case", [_dense3, _moe9, _oai3])
def test_two_ranks_match_one(case):
    """The bound of the contiguous decoder's two-rank tests: the order of the sums of what the ranks split."""
    want, lens, _ = spawn(case, world=1)[0]
    got = spawn(case, world=2)
    assert lens[:2] == [15 + 4, 14 + 3] and got[0][1] == got[1][1] == lens and got[0][2] == got[1][2]
    for outs, _, _ in got:
        for i, (a, b) in enumerate(zip(outs[:-1], want[:-1])):
            rows = slice(0, 1) if i == 3 else slice(None)         # the left-out row of that step means nothing
            assert rel_l2(a[rows], b[rows]) <= 1e-4
        assert np.array_equal(outs[-1][:2], want[-1][:2]) and (outs[-1][2:] == -1).all()
    for i, (a, b) in enumerate(zip(got[0][0], got[1][0])):
        assert np.array_equal(a, b)
