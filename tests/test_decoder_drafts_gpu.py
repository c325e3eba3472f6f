"""The decoder on a 4-bit cache, and drafted: kv_append, prefix_attention and verify_drafts as a program uses them together, every call against its definition."""

import numpy as np
import pytest
import torch

from oracle import paged as P
from oracle import verify as V

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def make():
    from velox_voice_b200 import decoder as D

    cfg = D.DecoderConfig(blocks=2, positions=600, cache="fp4")
    weights = D.make_weights(cfg)
    return lambda **kw: D.HypothesisDecoder(D.DecoderConfig(**{**vars(cfg), **kw}), weights, pages=200)


def host(t):
    return t.detach().cpu().numpy()


def check_append(call, k, v, k_pages, v_pages, page_table, lengths, *, q=None, rotary=None, row_offsets=None, starts=None):
    before = host(k_pages), host(v_pages)
    out = call(k, v, k_pages, v_pages, page_table, lengths, q=q, rotary=rotary, row_offsets=row_offsets, starts=starts)
    want = P.kv_append_fp4_ref(host(k.float()), host(v.float()), *before, host(page_table), host(lengths), host(rotary), False, None if row_offsets is None else host(row_offsets),
                               None if starts is None else host(starts))
    for got, w in zip((k_pages, v_pages), want):
        assert (P.fp4_values(host(got)) == P.fp4_values(w)).all()
    return out


def check_attention(call, q, k_pages, v_pages, page_table, lengths, prefix_table=None, prefix_lengths=None, *, row_offsets=None):
    """2^-11 of each probability and 2^-8 of the result, as the tests of the operator."""
    out = call(q, k_pages, v_pages, page_table, lengths, prefix_table, prefix_lengths, row_offsets=row_offsets)
    want, spread = P.prefix_attention_ref(host(q.double()), P.fp4_values(host(k_pages)), P.fp4_values(host(v_pages)), host(page_table), host(lengths),
                                          None if prefix_table is None else host(prefix_table), None if prefix_lengths is None else host(prefix_lengths),
                                          None if row_offsets is None else host(row_offsets))
    most = np.abs(P.fp4_values(host(v_pages))).max()
    assert (np.abs(host(out.double()) - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -10.5) * spread + 2.0 ** -25 * 700 * most).all()
    return out


def check_verify(call, logits, ids, uniforms, *, draft_logits=None, row_offsets=None, temperature=1.0):
    accepted, following = call(logits, ids, uniforms, draft_logits=draft_logits, row_offsets=row_offsets, temperature=temperature)
    want = V.verify_ref(host(logits.double()), host(ids), host(uniforms.double()), None if draft_logits is None else host(draft_logits.double()), host(row_offsets), temperature)
    assert [(int(a), int(b)) for a, b in zip(accepted, following)] == [w[:2] for w in want]
    return accepted, following


def test_every_call_of_a_drafted_decode_is_right(make, monkeypatch):
    from velox_voice_b200 import ops

    calls = []
    for name, check in (("kv_append", check_append), ("prefix_attention", check_attention), ("verify_drafts", check_verify)):
        monkeypatch.setattr(ops, name, lambda *a, _c=getattr(ops, name), _k=check, _n=name, **k: (calls.append(_n), _k(_c, *a, **k))[1])
    torch.manual_seed(0)
    dec, counts, beams = make(), [40, 75], 3
    dec.k_pages.random_()  # whatever was there before
    dec.v_pages.random_()
    utt = dec.read(torch.randn(sum(counts), dec.cfg.d_model, device="cuda").bfloat16(), counts)
    hyp = dec.begin(utt, beams, 30)
    ids = dec.step(hyp, torch.arange(6, device="cuda") * 37).long()
    hyp.lengths[4] = -1
    for temperature in (1.0, 0.0):
        rows = [5, 1, 4, 5, 2, 0]
        given = torch.randint(0, dec.cfg.vocab, (sum(rows),), device="cuda")
        first = np.cumsum([0] + rows)[:-1]
        given[first[:5].tolist()] = ids[:5]
        before = hyp.lengths.tolist()
        accepted, following = dec.verify(hyp, given, rows, torch.rand(sum(rows), 2, device="cuda"), temperature=temperature)
        assert hyp.lengths.tolist() == [b + a + 1 if b >= 0 and r else b for b, a, r in zip(before, accepted.tolist(), rows)]
        ids = following.long().clamp_min(0)
    dec.settle(hyp)
    assert hyp.tokens[0] == hyp.lengths[0] and calls.count("verify_drafts") == 2 and calls.count("prefix_attention") == 2 * 4


def test_drafts_that_are_what_the_decoder_says_stand(make):
    """Greedy drafts of the decoder itself, taken from score() of the same ids, all stand, and the cache goes on as without drafts."""
    torch.manual_seed(1)
    dec = make()
    utt = dec.read(torch.randn(60, dec.cfg.d_model, device="cuda").bfloat16(), [60])
    a, b = dec.begin(utt, 2, 40), dec.begin(utt, 2, 40)
    n, ids = 4, torch.tensor([5, 9], device="cuda")
    given = torch.randint(0, dec.cfg.vocab, (2, n), device="cuda")
    given[:, 0] = ids
    for i in range(1, n):  # each draft by the logits of the same call, whose rows do not depend on later ids
        logits = dec.score(a, given.flatten(), [n, n]).view(2, n, -1)
        a.lengths.sub_(n)
        a.tokens = [0, 0]
        given[:, i] = logits[:, i - 1].argmax(-1)
    accepted, following = dec.verify(a, given.flatten(), [n, n], torch.rand(2 * n, 2, device="cuda"), temperature=0.0)
    logits = dec.score(b, given.flatten(), [n, n]).view(2, n, -1)
    assert accepted.tolist() == [n - 1] * 2 and following.tolist() == logits[:, -1].argmax(-1).tolist()
    assert torch.equal(a.lengths, b.lengths)


def test_a_captured_step_gives_the_same_tokens(make):
    torch.manual_seed(2)
    dec = make()
    utt = dec.read(torch.randn(100, dec.cfg.d_model, device="cuda").bfloat16(), [100])
    hyp, again = dec.begin(utt, 4, 20), dec.begin(utt, 4, 20)
    step = dec.compile_step(again)
    a = b = torch.arange(4, device="cuda")
    for _ in range(20):
        a, b = dec.step(hyp, a).long(), step(b).long()
        assert torch.equal(a, b)


@pytest.mark.parametrize("args", [["--cache", "fp4"], ["--cache", "fp4", "--drafts", "3"], ["--drafts", "2", "--utterances", "2"]])
def test_the_example_runs(args, monkeypatch, capsys):
    from velox_voice_b200 import decoder as D

    monkeypatch.setattr("sys.argv", ["decoder", "--frames", "60", "--beams", "3", "--tokens", "8", *args])
    D.main()
    assert "hypotheses over 60 frames" in capsys.readouterr().out
