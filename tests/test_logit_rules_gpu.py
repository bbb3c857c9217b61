"""Rules on logits against a plain restatement in 64 bits.  A changed logit is rounded at most five times (quotient, product,
two differences, the bias' sum), each within half an f32 step of the largest intermediate value: 5 * 2^-24 of 20 (logits
of N(0, 3^2), penalties below 8)."""
import numpy as np
import pytest
import torch

from tests import paged_plain as plain

pytestmark = pytest.mark.gpu


def words(bits):
    n, V = bits.shape
    b = torch.zeros((n, -(-V // 32) * 32), dtype=torch.int64)
    b[:, :V] = bits
    w = (b.view(n, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


@pytest.mark.parametrize("n,V", [(1, 1), (1, 31), (3, 33), (2, 4096), (5, 4097), (64, 1000), (65, 257), (130, 40), (2, 128256), (1, 300007)])
@pytest.mark.parametrize("h,bias,mask", [(0, 0, 0), (1, 0, 0), (40, 1, 1), (300, 2, 2), (0, 2, 1), (5000, 0, 2)])
def test_rules(n, V, h, bias, mask):
    from frink_b200 import device
    g = torch.Generator().manual_seed(n * V + h)
    x = torch.randn((n, V), generator=g) * 3
    hist = torch.randint(-3, V + 3, (n, h), generator=g)
    hist = torch.where(torch.rand((n, h), generator=g) < 0.5, hist % 7, hist).to(torch.int32)
    pen = torch.stack([1 + torch.rand(n, generator=g), torch.rand(n, generator=g) * 0.01, torch.rand(n, generator=g)], 1)
    b = None if not bias else torch.randn(V if bias == 1 else (n, V), generator=g)
    m = None
    if mask:
        bits = torch.rand((1 if mask == 1 else n, V), generator=g) < 0.3
        if mask == 2:
            bits[0] = False                                  # a row that may not go on
        m = words(bits)[0] if mask == 1 else words(bits)
    out, tok = device.logit_rules(x.cuda(), history=hist.cuda(), penalties=pen.cuda(), bias=None if b is None else b.cuda(), mask=None if m is None else m.cuda())
    want, wtok = plain.rules(x, hist, pen, b, m)
    got = out.cpu().double().numpy()
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(got)) and (got[~fin] == -np.inf).all()
    assert np.abs(got[fin] - want[fin]).max(initial=0.0) <= 5 * 2 ** -24 * 80
    # the token is the largest of the logits as they were written, the lowest of equal ones
    for r in range(n):
        assert tok[r].item() == (int(got[r].argmax()) if fin[r].any() else -1)
    if mask == 2:
        assert tok[0].item() == wtok[0] == -1


def test_ties_nan_infinities_and_untouched_logits():
    from frink_b200 import device
    x = torch.zeros((5, 5000))
    x[0, 4500] = x[0, 77] = 2.0                              # ties go to the lower index
    x[1, 10], x[1, 20] = float("nan"), 1.0                   # NaN never wins, and stays
    x[2] = float("nan")
    x[3, 4999] = float("inf")
    x[4] = float("-inf")
    out, tok = device.logit_rules(x.cuda())
    assert tok.tolist() == [77, 20, -1, 4999, -1]
    assert torch.equal(out.cpu().nan_to_num(7.0, 8.0, 9.0), x.nan_to_num(7.0, 8.0, 9.0))


def test_strides_one_row_in_place_and_one_triple():
    from frink_b200 import device
    g = torch.Generator().manual_seed(3)
    wide = torch.randn((4, 900), generator=g)
    hist = torch.randint(0, 700, (4, 50), generator=g).to(torch.int32)
    pen = torch.tensor([[1.2, 0.25, 0.5]]).expand(4, 3)
    want, wtok = plain.rules(wide[:, 100:800], hist, pen, None, None)
    xc = wide.cuda()
    out, tok = device.logit_rules(xc[:, 100:800], history=hist.cuda(), penalties=(1.2, 0.25, 0.5))
    assert np.abs(out.cpu().double().numpy() - want).max() <= 5 * 2 ** -24 * 20 and tok.tolist() == wtok
    assert torch.equal(xc.cpu(), wide)
    row = xc[1, 100:800].contiguous()
    o1, t1 = device.logit_rules(row, history=hist[1].cuda(), penalties=(1.2, 0.25, 0.5), out=row)
    assert o1.data_ptr() == row.data_ptr() and torch.equal(row, out[1]) and t1.tolist() == [wtok[1]]


def test_python_refusals():
    from frink_b200 import _lib, device
    x = torch.zeros((2, 64), device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    bad = [dict(history=i(3, 4), penalties=(1, 0, 0)), dict(history=i(2, 4)), dict(history=i(2, 4).long(), penalties=(1, 0, 0)), dict(history=i(2, 4), penalties=(1, 0)),
           dict(bias=torch.zeros(63, device="cuda")), dict(bias=torch.zeros((3, 64), device="cuda")), dict(mask=i(1)), dict(mask=i(2, 2).long()),
           dict(out=torch.zeros((2, 65), device="cuda")), dict(tokens=i(3)), dict(history=i(2, 8)[:, ::2], penalties=(1, 0, 0))]
    for kw in bad:
        with pytest.raises(_lib.Invalid):
            device.logit_rules(x, **kw)


def test_captured_and_replayed():
    from frink_b200 import device
    g = torch.Generator().manual_seed(5)
    x = torch.randn((3, 5000), generator=g).cuda()
    hist = torch.randint(0, 5000, (3, 20), generator=g).to(torch.int32).cuda()
    pen = torch.tensor([[1.3, 0.1, 0.2]] * 3).cuda()
    device.logit_rules(x, history=hist, penalties=pen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, tok = device.logit_rules(x, history=hist, penalties=pen)
    for s in range(3):
        x.copy_(torch.randn((3, 5000), generator=g))
        graph.replay()
        o, t = device.logit_rules(x, history=hist, penalties=pen)
        assert torch.equal(o, out) and torch.equal(t, tok)


@pytest.mark.parametrize("n,V", [(64, 9 * 24576), (64, 9 * 24480), (64, 9 * 24480 + 1), (64, 10 * 24480), (1, 64 * 24480)])
def test_a_block_takes_as_many_logits_as_it_can(n, V):
    """Vocabularies at which a block's counts are as many as shared memory holds."""
    from frink_b200 import device
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((n, V), generator=g, device="cuda")
    hist = torch.randint(0, V, (n, 300), generator=g, device="cuda", dtype=torch.int32)
    hist[:, 0], hist[:, 1] = V - 1, 0
    pen = torch.tensor([[1.5, 0.25, 0.5]], device="cuda").expand(n, 3).contiguous()
    out, tok = device.logit_rules(x, history=hist, penalties=pen)
    c = torch.zeros((n, V), device="cuda").scatter_add_(1, hist.long(), torch.ones((n, 300), device="cuda"))
    # (divided by a tensor: by a number, torch multiplies with its rounded reciprocal)
    want = torch.where(c > 0, torch.where(x > 0, x / pen[:, :1], x * 1.5) - c * 0.25 - 0.5, x)
    assert torch.equal(out, want) and torch.equal(tok.long(), want.argmax(1))


def test_zeros_of_both_signs_are_ties():
    from frink_b200 import device
    x = torch.full((4, 9000), -1.0)
    x[0, 3], x[0, 7000] = -0.0, 0.0
    x[1, 3], x[1, 7000] = 0.0, -0.0
    x[2, 4], x[2, 5] = -0.0, 0.0
    x[3, 100], x[3, 150] = -0.0, 0.0
    out, tok = device.logit_rules(x.cuda())
    assert tok.tolist() == [3, 3, 4, 100]
    assert torch.equal(torch.signbit(out.cpu()), torch.signbit(x))


def test_one_row_of_a_wide_tensor_is_changed_in_place():
    """A single row is packed, whatever its tensor says about the distance to a next one."""
    from frink_b200 import device
    wide = torch.randn((4, 900), generator=torch.Generator().manual_seed(11)).cuda()
    hist, pen = torch.tensor([[5, 5, 9]], dtype=torch.int32).cuda(), torch.tensor([[1.2, 0.25, 0.5]]).cuda()
    for at in (100, 101):                                         # on and off a 16-byte boundary
        was = wide.clone()
        row = wide[1:2, at:at + 700]
        want, tok = device.logit_rules(row.clone(), history=hist, penalties=pen)
        got, tok2 = device.logit_rules(row, history=hist, penalties=pen, out=row)
        assert got.data_ptr() == row.data_ptr() and torch.equal(row, want) and torch.equal(tok, tok2)
        was[1, at:at + 700] = want[0]
        assert torch.equal(wide, was)
