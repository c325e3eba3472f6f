"""The decoder of velox_voice_b200/decoder.py: the operators of the paged cache as a program uses them together."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    from velox_voice_b200 import decoder as D

    cfg = D.DecoderConfig(blocks=2, positions=600)
    return D.HypothesisDecoder(cfg, D.make_weights(cfg), pages=400)


def check_append(call, k, v, k_pages, v_pages, page_table, lengths, *, q=None, rotary=None, row_offsets=None, starts=None):
    """The call, and its results against the rotation in fp64 for its own arguments: half a unit in the last of 8 bits."""
    seen = k_pages.clone(), v_pages.clone()
    out = call(k, v, k_pages, v_pages, page_table, lengths, q=q, rotary=rotary, row_offsets=row_offsets, starts=starts)
    n, ps, half = page_table.shape[0], k_pages.shape[1], rotary.shape[1] // 2
    off = list(range(n + 1)) if row_offsets is None else row_offsets.tolist()
    for s in range(n):
        for i, r in enumerate(range(off[s], off[s + 1])):
            if int(lengths[s]) < 0:
                assert not out[r].any()
                continue
            t = int(lengths[s]) + i
            c = rotary[t + (0 if starts is None else int(starts[s]))].double()

            def near(got, x):
                a, b = x[:, :half].double(), x[:, half:].double()
                want = torch.cat([a * c[:half] - b * c[half:], b * c[:half] + a * c[half:]], -1)
                return ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * x.abs().amax().double()).all()

            page = int(page_table[s, t // ps])
            assert near(k_pages[page, t % ps], k[r]) and near(out[r], q[r]) and torch.equal(v_pages[page, t % ps], v[r])
            seen[0][page, t % ps], seen[1][page, t % ps] = k_pages[page, t % ps], v_pages[page, t % ps]
    assert torch.equal(seen[0].view(torch.int16), k_pages.view(torch.int16)) and torch.equal(seen[1].view(torch.int16), v_pages.view(torch.int16))
    return out


def check_attention(call, q, k_pages, v_pages, page_table, lengths, prefix_table=None, prefix_lengths=None, *, row_offsets=None):
    """The call, and its result against a softmax in fp64 over its own arguments: one rounding of the result, one of each probability."""
    out = call(q, k_pages, v_pages, page_table, lengths, prefix_table, prefix_lengths, row_offsets=row_offsets)
    n, ps = page_table.shape[0], k_pages.shape[1]
    off = list(range(n + 1)) if row_offsets is None else row_offsets.tolist()
    for s in range(n):
        for i, r in enumerate(range(off[s], off[s + 1])):
            if int(lengths[s]) < 0:
                assert not out[r].any()
                continue
            j = torch.arange(int(lengths[s]) + i + 1, device=q.device)
            k, v = (c[page_table[s].long()[j // ps], j % ps] for c in (k_pages, v_pages))
            if prefix_table is not None:
                g = s // (n // prefix_table.shape[0])
                j = torch.arange(int(prefix_lengths[g]), device=q.device)
                k, v = (torch.cat([c[prefix_table[g].long()[j // ps], j % ps], x]) for c, x in ((k_pages, k), (v_pages, v)))
            w = torch.softmax(torch.einsum("hd,jhd->hj", q[r].double(), k.double()) * q.shape[2] ** -0.5, -1)
            want, spread = torch.einsum("hj,jhd->hd", w, v.double()), torch.einsum("hj,jhd->hd", w, v.double().abs())
            assert ((out[r].double() - want).abs() <= 2.0 ** -8 * (want.abs() + spread) + 2.0 ** -13 * spread).all()
    return out


def test_every_call_of_reading_stepping_and_scoring_is_right(dec, monkeypatch):
    """Frames of two utterances, steps of their hypotheses (one of which has finished) and whole continuations.  (Tokens or logits of
    whole decodes say little: four-bit linears make a code step of a last bit.)"""
    from velox_voice_b200 import ops

    calls = []
    append, attend = ops.kv_append, ops.prefix_attention
    monkeypatch.setattr(ops, "kv_append", lambda *a, **k: (calls.append("append"), check_append(append, *a, **k))[1])
    monkeypatch.setattr(ops, "prefix_attention", lambda *a, **k: (calls.append("attend"), check_attention(attend, *a, **k))[1])
    torch.manual_seed(0)
    counts, beams, tokens = [40, 75], 3, 6
    frames = torch.randn(sum(counts), dec.cfg.d_model, device="cuda").bfloat16()
    dec.k_pages.fill_(float("nan"))
    dec.v_pages.fill_(float("nan"))
    utt = dec.read(frames, counts)
    hyp = dec.begin(utt, beams, 3 + tokens)
    ids = torch.arange(6, device="cuda") * 37
    for step in range(3):
        if step == 2:
            hyp.lengths[4] = -1
        ids = dec.step(hyp, ids).long()
    assert hyp.lengths.tolist() == [3, 3, 3, 3, -1, 3]
    rows = [tokens, 1, 3, tokens, 2, 4]
    logits = dec.score(hyp, torch.randint(0, dec.cfg.vocab, (sum(rows),), device="cuda"), rows)
    live = [r for i, r in enumerate(torch.split(logits, rows)) if i != 4]
    assert logits.shape == (sum(rows), dec.cfg.vocab) and all(torch.isfinite(x.float()).all() for x in live)
    assert hyp.lengths.tolist() == [9, 4, 6, 9, -1, 7]
    assert calls == ["append", "attend"] * (dec.cfg.blocks * 5)
    dec.release(hyp)
    dec.release(utt)


def test_a_captured_step_gives_the_same_tokens(dec):
    torch.manual_seed(2)
    frames = torch.randn(100, dec.cfg.d_model, device="cuda").bfloat16()
    utt = dec.read(frames, [100])
    hyp, again = dec.begin(utt, 4, 20), dec.begin(utt, 4, 20)
    step = dec.compile_step(again)
    a = b = torch.arange(4, device="cuda")
    for _ in range(20):
        a, b = dec.step(hyp, a).long(), step(b).long()
        assert torch.equal(a, b)
    free = len(dec._free)
    for x in (hyp, again, utt):
        dec.release(x)
    assert len(dec._free) == free + 4 * 2 * 2 + 7


def test_finished_hypotheses_and_a_pool_that_is_too_small(dec):
    torch.manual_seed(3)
    frames = torch.randn(50, dec.cfg.d_model, device="cuda").bfloat16()
    utt = dec.read(frames, [50])
    hyp, alone = dec.begin(utt, 3, 8), dec.begin(utt, 1, 8)
    hyp.lengths[1] = -1
    ids = torch.tensor([5, 6, 7], device="cuda")
    for _ in range(3):
        nxt = dec.step(hyp, ids)
        one = dec.step(alone, ids[2:])
        assert nxt[2] == one[0]  # the rows of others change nothing
        ids = nxt.long()
    assert hyp.lengths.tolist() == [3, -1, 3]
    with pytest.raises(RuntimeError, match="pages wanted"):
        dec.begin(utt, 1000, 100)
    with pytest.raises(ValueError):
        dec.read(frames, [20, 20])
    for x in (hyp, alone, utt):
        dec.release(x)
