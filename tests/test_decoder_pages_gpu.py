"""`Decoder` over a paged cache on the GPU: attention, append, bookkeeping and rules as a server uses them together."""
import numpy as np
import pytest
import torch

from oracle import frink_oracle as fo
from tests import paged_ops
from tests.helpers import rel_l2, tiny_gpt_oss
from tests.test_decoder_gpu import small_llama

pytestmark = pytest.mark.gpu


def models(which):
    from frink_b200.decoder import Decoder
    if which == "oai":
        cfg, layers, tok, out_norm, head = tiny_gpt_oss()
        kind = fo.BF16
    elif which == "moe":
        from tests.test_parallel_cpu import _tiny_model
        cfg, layers, tok, out_norm, head = _tiny_model(True)
        kind = fo.Q8_0
    else:
        cfg, layers, tok, out_norm, head = small_llama(uniform=which == "uniform")
        kind = fo.Q6_K
    return cfg, lambda **kw: Decoder(cfg, layers, tok, kind, out_norm, output=head, output_kind=kind, max_seq=96, **kw)


def prompts_of(cfg, n, seed=17):
    rng = np.random.default_rng(seed)
    return [torch.from_numpy(rng.integers(0, cfg.vocab, 5 + 3 * s).astype(np.int32)).cuda() for s in range(n)]


@pytest.mark.parametrize("which", ["uniform", "mixed", "moe", "oai"])
@pytest.mark.parametrize("n_seqs", [3, 11])
def test_paged_batches_match_each_sequence_alone(which, n_seqs):
    """f32 pages.  The bounds of the contiguous batch's test: another summation order in the matvecs of a batch, and re-rounded
    8-bit activations behind it; eleven rows take the GEMMs."""
    from frink_b200 import device
    cfg, mk = models(which)
    prompts, steps = prompts_of(cfg, n_seqs), 6
    solo, want_tok, want_logits = mk(), [], []
    for p in prompts:
        solo.reset()
        t = solo.prefill(p)
        toks, lgs = [int(t)], []
        for _ in range(steps):
            lg = solo.forward(t)
            lgs.append(lg.cpu().numpy()[0])
            t = device.argmax(lg)
            toks.append(int(t))
        want_tok.append(toks)
        want_logits.append(lgs)
    dec = mk()
    dec.alloc_pages(n_seqs, 4 * n_seqs, page=16, dtype=torch.float32)
    cur = torch.cat([dec.prefill_pages(s, p) for s, p in enumerate(prompts)])
    assert cur.tolist() == [t[0] for t in want_tok]
    worst = 0.0
    for i in range(steps):
        # the solo tokens are fed, so that one coin flip does not make the rest incomparable
        cur = torch.tensor([t[i] for t in want_tok], dtype=torch.int32, device="cuda")
        lg = dec.forward_pages(cur)
        worst = max([worst] + [rel_l2(lg[s].cpu().numpy(), want_logits[s][i]) for s in range(n_seqs)])
    assert device.device_error() == 0 and worst <= 2e-2, worst
    assert dec._pool.lens == dec.pages.lens.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_windowed_layers_with_first_tokens_match_the_cpu_decoder(dtype):
    """gpt-oss's layer form over pages, its windowed layer with two first tokens visible: prompt in chunks, a fork, decode steps,
    against the same decoder on the CPU stand-ins (the bound of that form's contiguous test)."""
    cfg, mk = models("oai")
    cfg.first_tokens = 2
    dev, cpu = mk(), mk(ops=paged_ops, device="cpu")
    for d in (dev, cpu):
        d.alloc_pages(3, 14, page=16, dtype=dtype)
    p = prompts_of(cfg, 14, 3)[-1]                                 # 44 tokens
    worst = 0.0
    for a, b in ((0, 30), (30, 31), (31, 44)):
        x, y = dev.forward_pages_seq(0, p[a:b]), cpu.forward_pages_seq(0, p[a:b].cpu())
        worst = max(worst, rel_l2(x.cpu().numpy(), y.numpy()))
    for d in (dev, cpu):
        d.fork_pages([0, 0], [1, 2], [40, None])
        d.free_pages([0])
    dev.compact_pages()
    for t in (3, 99):
        x, y = dev.forward_pages(torch.full((3,), t, dtype=torch.int32, device="cuda")), cpu.forward_pages(torch.full((3,), t, dtype=torch.int32))
        worst = max(worst, rel_l2(x[1:].cpu().numpy(), y[1:].numpy()))
    from frink_b200 import device
    assert device.device_error() == 0 and worst <= 2e-2, worst
    assert dev.pages.lens.tolist() == cpu.pages.lens.tolist() == dev._pool.lens == [0, 42, 46]


def test_a_captured_step_with_rules_follows_the_eager_one_through_frees_and_forks():
    from frink_b200 import device
    from frink_b200.decoder import LogitRules
    cfg, mk = models("uniform")
    prompts = prompts_of(cfg, 4)
    words = torch.full((cfg.vocab // 32,), -1, dtype=torch.int32, device="cuda")

    def start():
        dec = mk()
        dec.alloc_pages(4, 20, page=16, dtype=torch.float16)
        rules = LogitRules(4, penalties=(1.3, 0.1, 0.2), last=8, mask=words)
        cur = torch.cat([dec.prefill_pages(s, p, rules) for s, p in enumerate(prompts)])
        return dec, rules, cur

    words.fill_(-1)
    eager, er, ecur = start()
    graph, gr, gcur = start()
    assert ecur.tolist() == gcur.tolist()
    g, out = graph.capture_pages(gcur, gr)
    assert graph._pool.lens == graph.pages.lens.tolist() and torch.equal(er.history, gr.history)
    for i in range(24):                                            # over page edges
        if i == 7:
            for d, r in ((eager, er), (graph, gr)):
                d.free_pages([1])
                r.forget(1)
                d.fork_pages([2], [1])
                r.copy(2, 1)
            ecur[1], gcur[1] = ecur[2], gcur[2]
        if i == 12:
            words.fill_(0x0f0f0f0f)                                # the grammar changes; both read the same words
        ecur = eager.step_pages(ecur, er)
        graph.replay_pages()
        gcur.copy_(out)
        assert ecur.tolist() == gcur.tolist(), i
        if i >= 12:
            assert all(t % 8 < 4 for t in ecur.tolist())
    assert torch.equal(eager.pages.table, graph.pages.table) and torch.equal(eager.pages.refs, graph.pages.refs)
    assert graph._pool.lens == graph.pages.lens.tolist() and device.device_error() == 0


def test_what_does_not_fit_is_refused_before_anything_is_launched():
    from frink_b200 import device
    cfg, mk = models("uniform")
    dec = mk()
    dec.alloc_pages(3, 4, page=16, max_tokens=48)
    dec.forward_pages_seq(0, torch.zeros(40, dtype=torch.int32, device="cuda"))
    n0 = device.counters(reset=True)
    for bad in (lambda: dec.forward_pages_seq(1, torch.zeros(17, dtype=torch.int32, device="cuda")),
                lambda: dec.forward_pages_seq(0, torch.zeros(9, dtype=torch.int32, device="cuda")), lambda: dec.fork_pages([0], [0]), lambda: dec.fork_pages([0], [1], [41])):
        with pytest.raises(ValueError):
            bad()
    assert device.counters()["launches"] == 0 and n0 is not None
    dec.fork_pages([0], [1])
    with pytest.raises(ValueError):
        dec.fork_pages([0], [2], [7])                              # the pool is full
    dec.fork_pages([0], [2], [32])                                 # whole pages only
    dec.free_pages([2])
    for _ in range(8):
        dec.forward_pages(torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        dec.forward_pages(torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert device.device_error() == 0 and dec.pages.lens.tolist() == [48, 48, 0]


def test_generate_with_rules_and_seventy_sequences():
    from frink_b200 import device
    from frink_b200.decoder import LogitRules
    cfg, mk = models("uniform")
    dec = mk()
    p = prompts_of(cfg, 1)[0]
    plainly = dec.generate(p, 12)
    dec.reset()
    assert dec.generate(p, 12, rules=LogitRules(1)) == plainly
    dec.reset()
    no_repeats = dec.generate(p, 12, rules=LogitRules(1, penalties=(1.0, 0.0, 1000.0), last=64))
    assert len(set(no_repeats)) == 12 and not set(no_repeats) & set(p.tolist())
    many = mk()
    many.alloc_pages(70, 150, page=16, max_tokens=32)
    one = many.prefill_pages(0, p)
    many.fork_pages([0] * 69, list(range(1, 70)))
    toks = many.step_pages(one.expand(70).contiguous())
    assert len(set(toks.tolist())) == 1 and device.device_error() == 0
