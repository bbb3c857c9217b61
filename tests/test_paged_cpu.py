"""Refusals of the paged cache's and the logit rules' entry points: what is wrong is said before anything is launched, so the
checks run without a GPU (the context is a block of zeros that no refused call looks into)."""
import ctypes as C
import types

import pytest
import torch

from frink_b200 import _lib, device
from frink_b200.device import _CPages

CTX = C.create_string_buffer(1 << 16)
MEM = 1 << 20          # an address that is never followed


def pool(**kw):
    f = dict(data_dev=MEM, table_dev=MEM, lens_dev=MEM, refs_dev=MEM, ws_dev=MEM, ws_bytes=1 << 30, kind=30, n_layers=2, n_pages=9, page=16, n_kv=2,
             head_dim=64, n_seqs=3, max_pages=4)
    f.update(kw)
    return C.byref(_CPages(*[f[n] for n, _ in _CPages._fields_]))


def ints(*v):
    return (C.c_int * len(v))(*v)


def refused(fn, *args, status=_lib.FK_INVALID, match=""):
    assert getattr(_lib.lib(), fn)(*args) == status
    assert match in _lib.lib().fk_last_error().decode()


POOL_FAULTS = [(dict(data_dev=None), _lib.FK_INVALID), (dict(ws_dev=None), _lib.FK_INVALID), (dict(kind=8), _lib.FK_UNSUPPORTED), (dict(page=48), _lib.FK_UNSUPPORTED),
               (dict(page=256), _lib.FK_UNSUPPORTED), (dict(head_dim=136), _lib.FK_UNSUPPORTED), (dict(head_dim=20), _lib.FK_UNSUPPORTED), (dict(n_seqs=0), _lib.FK_UNSUPPORTED),
               (dict(n_seqs=4097), _lib.FK_UNSUPPORTED), (dict(max_pages=0), _lib.FK_INVALID), (dict(max_pages=1 << 28), _lib.FK_UNSUPPORTED), (dict(n_kv=0), _lib.FK_INVALID),
               (dict(data_dev=MEM + 8), _lib.FK_INVALID), (dict(ws_dev=MEM + 16), _lib.FK_INVALID), (dict(ws_bytes=64), _lib.FK_INVALID)]


@pytest.mark.parametrize("fault,status", POOL_FAULTS)
def test_every_call_refuses_a_wrong_pool(fault, status):
    p, f = pool(**fault), C.c_float
    refused("fk_pages_grow", CTX, None, p, None, 1, status=status)
    refused("fk_pages_advance", CTX, None, p, None, 1, status=status)
    refused("fk_pages_fork", CTX, None, p, ints(0), ints(1), None, 1, status=status)
    refused("fk_pages_free", CTX, None, p, ints(0), 1, status=status)
    refused("fk_pages_compact", CTX, None, p, MEM, status=status)
    refused("fk_rope_kv_paged", CTX, None, p, 0, MEM, MEM, MEM, 256, 128, 128, 1, None, 4, f(1e4), 0, None, None, f(0), MEM, status=status)
    refused("fk_attention_paged", CTX, None, p, 0, MEM, 0, 1, None, 4, f(1), 0, 0, None, MEM, status=status)


def test_lists_are_checked():
    p = pool()
    for ids in ((3,), (-1,), (1, 1)):
        refused("fk_pages_free", CTX, None, p, ints(*ids), len(ids))
    refused("fk_pages_free", CTX, None, p, ints(0), 0)
    refused("fk_pages_free", CTX, None, p, None, 1)
    refused("fk_pages_free", CTX, None, pool(n_seqs=100), ints(*range(65)), 65)
    refused("fk_pages_fork", CTX, None, p, ints(0, 0), ints(1, 1), None, 2, match="twice")
    refused("fk_pages_fork", CTX, None, p, ints(0, 1), ints(1, 2), None, 2, match="source and a destination")
    refused("fk_pages_fork", CTX, None, p, ints(3), ints(1), None, 1)
    refused("fk_pages_fork", CTX, None, p, None, ints(1), None, 1)
    refused("fk_pages_fork", CTX, None, pool(n_layers=65536), ints(0), ints(1), None, 1, status=_lib.FK_UNSUPPORTED)
    refused("fk_pages_grow", CTX, None, p, None, -1)
    refused("fk_pages_advance", CTX, None, p, None, -1)


def test_rope_and_attention_arguments():
    p, f = pool(), C.c_float
    ok = [CTX, None, p, 0, MEM, MEM, MEM, 256, 128, 128, 1, None, 4, f(1e4), 0, None, None, f(0), MEM]
    for at, v in ((3, 2), (3, -1), (4, None), (4, MEM + 4), (7, 252), (7, 258), (8, 64), (10, 0), (12, 0), (13, f(0)), (13, f(float("inf"))), (13, f(float("nan"))), (15, MEM), (18, None), (18, MEM + 8)):
        refused("fk_rope_kv_paged", *(ok[:at] + [v] + ok[at + 1:]))
    refused("fk_rope_kv_paged", *(ok[:7] + [260] + ok[8:]), match="in place")
    ok = [CTX, None, p, 1, MEM, 0, 1, None, 4, f(1), 0, 0, None, MEM]
    for at, v, st in ((3, 2, _lib.FK_INVALID), (4, None, _lib.FK_INVALID), (4, MEM + 4, _lib.FK_INVALID), (5, 200, _lib.FK_INVALID), (5, 258, _lib.FK_INVALID), (6, 0, _lib.FK_UNSUPPORTED),
                      (8, 3, _lib.FK_UNSUPPORTED), (8, 0, _lib.FK_UNSUPPORTED), (10, -1, _lib.FK_INVALID), (11, -1, _lib.FK_INVALID), (13, None, _lib.FK_INVALID)):
        refused("fk_attention_paged", *(ok[:at] + [v] + ok[at + 1:]), status=st)


def test_logit_rule_arguments():
    ok = [CTX, None, MEM, 100, 2, 100, MEM, 5, MEM, MEM, 0, MEM, 0, MEM * 2, MEM]
    for at, v in ((0, None), (2, None), (3, 99), (4, 0), (5, 0), (6, None), (7, -1), (8, None), (10, 99), (12, 3), (13, None)):
        refused("fk_logit_rules", *(ok[:at] + [v] + ok[at + 1:]))
    refused("fk_logit_rules", CTX, None, MEM, 100, 2, 100, MEM, 65536, MEM, None, 0, None, 0, MEM * 2, MEM, status=_lib.FK_UNSUPPORTED)
    refused("fk_logit_rules", CTX, None, MEM, 104, 2, 100, None, 0, None, None, 0, None, 0, MEM, None, match="in place")


def test_python_layer_refuses_tensors_off_the_gpu():
    t = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(_lib.Invalid):
        device.Pages(torch.zeros(1, 4, 2, 2, 16, 64), t(2, 2), t(2), t(4))
    with pytest.raises(_lib.Invalid):
        device.Pages(torch.zeros(1, 4, 2, 2, 16), t(2, 2), t(2), t(4))
    with pytest.raises(_lib.Invalid):
        device.logit_rules(torch.zeros(2, 8))


def test_rows_that_lie_over_one_another_are_refused():
    pg = types.SimpleNamespace(_dev=-1, n_seqs=2)                  # a pool off the GPU, as far as the check of rows looks
    x = torch.zeros(40)
    assert device._rows_of(pg, x[:32].view(4, 8), 8, "x") == (4, 8)
    assert device._rows_of(pg, x.view(4, 10)[:, :8], 8, "x") == (4, 10)
    for rows in (x[:8].expand(4, 8), x.as_strided((4, 8), (4, 1)), x.as_strided((4, 8), (1, 4)), x[:24].view(3, 8), x[:36].view(4, 9), x.double()[:32].view(4, 8)):
        with pytest.raises(_lib.Invalid):
            device._rows_of(pg, rows, 8, "x")
