"""Which sequences a decode step moves, and what becomes of its tokens, against a plain restatement; refusals without a GPU."""
import ctypes as C

import pytest
import torch

from frink_b200 import _lib, device

CTX, MEM = C.create_string_buffer(1 << 16), 1 << 20      # a context that no refused call looks into, an address never followed


def test_refusals():
    L = _lib.lib()
    ok = [CTX, None, MEM, MEM, 3, MEM, MEM]
    for at, v in ((0, None), (2, None), (3, None), (4, 0), (4, -1), (5, None), (6, None)):
        assert L.fk_pages_moves(*(ok[:at] + [v] + ok[at + 1:])) == _lib.FK_INVALID
    ok = [CTX, None, MEM, MEM, 3, MEM, 4, MEM]
    for at, v in ((0, None), (2, None), (4, 0), (6, 0), (7, None)):
        assert L.fk_tokens_join(*(ok[:at] + [v] + ok[at + 1:])) == _lib.FK_INVALID
    t = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: device.pages_moves(t, t), lambda: device.tokens_join(t)):
        with pytest.raises(_lib.Invalid):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 256, 257, 4096])
def test_moves(n):
    g = torch.Generator().manual_seed(n)
    toks, live = torch.randint(-3, 5, (n,), generator=g, dtype=torch.int32), torch.randint(0, 2, (n,), generator=g, dtype=torch.int32)
    toks[0] = -2 ** 31
    ids, moves = device.pages_moves(toks.cuda(), live.cuda())
    assert torch.equal(ids.cpu(), toks.clamp(min=0)) and torch.equal(moves.cpu(), ((live != 0) & (toks >= 0)).int())


@pytest.mark.gpu
@pytest.mark.parametrize("n,h", [(1, 1), (3, 7), (300, 64), (5, 65535)])
@pytest.mark.parametrize("all_move", [False, True])
def test_join(n, h, all_move):
    g = torch.Generator().manual_seed(h)
    tok, moves = torch.randint(-1, 9, (n,), generator=g, dtype=torch.int32), torch.randint(0, 2, (n,), generator=g, dtype=torch.int32)
    hist, at = torch.randint(-1, 9, (n, h), generator=g, dtype=torch.int32), torch.randint(0, 2 ** 40, (n,), generator=g)
    dt, dh, da = tok.cuda(), hist.cuda(), at.cuda()
    assert device.tokens_join(dt, None if all_move else moves.cuda(), dh, da) is dt
    for s in range(n):
        if not all_move and not moves[s]:
            tok[s] = -1
        if tok[s] >= 0:
            hist[s, at[s] % h] = tok[s]
            at[s] += 1
    assert torch.equal(dt.cpu(), tok) and torch.equal(dh.cpu(), hist) and torch.equal(da.cpu(), at)
    kept = tok.clone()
    assert torch.equal(device.tokens_join(tok.cuda(), moves.cuda()).cpu(), torch.where(moves > 0, kept, -1))      # no history


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    at = torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (lambda: device.pages_moves(i(3), i(4)), lambda: device.pages_moves(i(3).long(), i(3)), lambda: device.pages_moves(i(6)[::2], i(3)), lambda: device.pages_moves(i(3), i(3).cpu()),
                 lambda: device.tokens_join(i(3), i(2)), lambda: device.tokens_join(i(3), None, i(2, 4), at), lambda: device.tokens_join(i(3), None, i(3, 8)[:, ::2], at),
                 lambda: device.tokens_join(i(3), None, i(3, 4)), lambda: device.tokens_join(i(3), None, i(3, 4), at.int()), lambda: device.tokens_join(i(3), None, i(3, 0), at)):
        with pytest.raises(_lib.Invalid):
            call()
