"""Drafted decoding over a cache held in 4 bits, as cases that can be timed: `kv_append` into 4-bit pages (rotation and
quantization on the way), `prefix_attention` over them, and `verify_drafts` (drafted tokens against the target's
probabilities), each in a plain form and through the public entry points.

A page of 4-bit keys or values is u8 [kv_heads, page_size / 16, 9 head_dim]: of every 16 tokens of a head first the
codes, head_dim / 2 bytes a token (E2M1, the even value in the low half), then the scales, head_dim / 16 bytes a token
(E4M3, one for 16 values).

What the sizes stand for: the hypotheses of an utterance share its encoder frames (40 ms each: 375 for a quarter of a
minute, 3,750 for a full span of long audio, 89,999 for an hour); heads are the encoder's (8 of 64) or grouped ones of a
larger decoder (32 query heads on 8 key heads of 128); 5,538 is the vocabulary."""

import math
import random

import torch

own = False

NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decoding step of the ten hypotheses of one utterance: launches and host time
        _append("append4_beam_step", seqs=10, tokens=1, history=40, heads=8, kv_heads=8, dim=64, rot=64, page=16),
        # the frames of one span of long audio become the prefix; rows in fp32 as a linear can leave them
        _append("append4_span", seqs=1, tokens=3750, history=0, heads=8, kv_heads=8, dim=64, rot=64, page=16, dtype="float32",
                interleaved=True),
        # prompts of a batch, together an hour of audio, half of each head rotated
        _append("append4_hour", seqs=24, tokens=5000, history=0, heads=32, kv_heads=8, dim=128, rot=64, page=32),
        # one decoding step of ten hypotheses over a short utterance
        _attention("attend4_utterance", groups=1, beams=10, tokens=1, prefix=375, history=24, heads=8, kv_heads=8, dim=64, page=16),
        # four drafts and the token before them, for the ten hypotheses of each of sixteen spans
        _attention("attend4_drafts", groups=16, beams=10, tokens=5, prefix=3750, history=90, heads=8, kv_heads=8, dim=64, page=16),
        # a server's step: long answers of their own, some finished, the middle of some dropped
        _attention("attend4_serve", groups=64, beams=1, tokens=1, prefix=0, history=8000, heads=32, kv_heads=8, dim=128, page=64,
                   ragged=True, dropped=True),
        # 32 hypotheses over an hour of audio
        _attention("attend4_hour", groups=1, beams=32, tokens=1, prefix=89999, history=300, heads=32, kv_heads=8, dim=128, page=32),
        # eight prompts with 16 answers each
        _attention("attend4_prompts", groups=8, beams=16, tokens=1, prefix=8190, history=1024, heads=32, kv_heads=8, dim=128, page=64,
                   ragged=True),
        # a chunk of two prompts behind a shared one
        _attention("attend4_chunk", groups=1, beams=2, tokens=1500, prefix=8192, history=500, heads=32, kv_heads=8, dim=128, page=64),
        # ten hypotheses with four greedy drafts each
        _verify("verify_beam", seqs=10, drafts=4, vocab=5538, drafter=False),
        # a batch of hypotheses with a drafter's probabilities, not the same number of drafts for each
        _verify("verify_batch", seqs=160, drafts=7, vocab=5538, drafter=True, ragged=True, temperature=0.8),
        # a large vocabulary, rows in fp32
        _verify("verify_wide", seqs=64, drafts=5, vocab=131071, drafter=True, dtype="float32"),
    ]


def _append(name, **kw):
    return {"name": name, "kind": "append", "dtype": "bfloat16", "interleaved": False, "ragged": True, **kw}


def _attention(name, **kw):
    return {"name": name, "kind": "attention", "ragged": False, "dropped": False, **kw}


def _verify(name, **kw):
    return {"name": name, "kind": "verify", "ragged": False, "temperature": 1.0, "dtype": "bfloat16", **kw}


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "drafts", "drafts", "chunk", "verify", "verify"))
    if kind == "verify":
        vocab = _log_size(rng, 1000, 131072)
        seqs = _log_size(rng, 1, min(512, max(2, 40000000 // (9 * vocab))))
        return {"kind": "verify", "seqs": seqs, "drafts": rng.choice((0, 1, 2, 3, 4, 5, 6, 7, 8)), "vocab": vocab, "drafter": rng.random() < 0.6,
                "ragged": rng.random() < 0.5, "temperature": rng.choice((1.0, 0.7, 1.3, 0.0)), "dtype": rng.choice(("bfloat16", "bfloat16", "float32"))}
    heads, kv_heads, dim = rng.choice(((8, 8, 64), (8, 8, 64), (16, 4, 64), (32, 8, 128), (32, 8, 128), (12, 4, 128), (20, 2, 128)))
    common = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice((16, 16, 32, 48, 64, 128)), "ragged": rng.random() < 0.5}
    if kind == "append":
        tokens = rng.choice((1, _log_size(rng, 2, 6000)))
        seqs = _log_size(rng, 1, min(512, max(2, 90000 // tokens)))
        return {"kind": "append", "seqs": seqs, "tokens": tokens, "history": rng.randrange(0, 500), "rot": rng.choice((dim, dim // 2, dim)),
                "dtype": rng.choice(("bfloat16", "bfloat16", "float32")), "interleaved": rng.random() < 0.4, **common}
    groups = _log_size(rng, 1, 16)
    case = {"kind": "attention", "groups": groups, "dropped": rng.random() < 0.25, **common}
    if kind == "decode":
        case.update(beams=_log_size(rng, 1, 256 // groups), tokens=1, prefix=rng.choice((0, _log_size(rng, 16, 90000 // groups))),
                    history=_log_size(rng, 1, 2000))
    elif kind == "drafts":
        case.update(beams=_log_size(rng, 1, 160 // groups), tokens=rng.randrange(2, 9), prefix=rng.choice((0, _log_size(rng, 64, 4000))),
                    history=_log_size(rng, 1, 1000))
    else:
        case.update(groups=1, beams=rng.randrange(1, 4), tokens=_log_size(rng, 100, 1000), prefix=rng.choice((0, _log_size(rng, 100, 8192))),
                    history=rng.randrange(0, 500))
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _sizes(case):
    """Rows, lengths and prefixes of a case: host numbers, the same whatever the seed of the values.  Where a case is ragged,
    sequences are between half and all of its sizes long and a few of many have finished (length -1)."""
    rng = random.Random(23)

    def around(n):
        return rng.randint((n + 1) // 2, n) if case["ragged"] and n > 1 else n

    if case["kind"] == "verify":
        return {"tokens": [around(case["drafts"]) + 1 for _ in range(case["seqs"])]}
    groups = case.get("groups", 1)
    n = case["seqs"] if case["kind"] == "append" else groups * case["beams"]
    tokens = [around(case["tokens"]) for _ in range(n)]
    lengths = [around(case["history"]) for _ in range(n)]
    if case["ragged"] and n >= 32 and case["kind"] == "attention":
        lengths = [-1 if rng.random() < 0.04 else l for l in lengths]
    return {"tokens": tokens, "lengths": lengths, "prefix": [around(case.get("prefix", 0)) for _ in range(groups)]}


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    z = _sizes(case)
    n, rows = len(z["tokens"]), sum(z["tokens"])

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    offsets = _offsets(z["tokens"])
    s = {"case": case, "host": z, "row_offsets": ints(offsets)}
    if case["kind"] == "verify":
        # logits as a trained head leaves them: a few likely tokens, a long tail; the drafter's are near the target's, and its
        # drafts are drawn from them
        vocab, kind = case["vocab"], NAMES[case["dtype"]]
        logits = torch.randn(rows, vocab, generator=g, device=dev) * 2.0
        logits.scatter_add_(1, torch.randint(vocab, (rows, 6), generator=g, device=dev), 8.0 + 3.0 * torch.randn(rows, 6, generator=g, device=dev))
        s["logits"] = logits.to(kind)
        s["draft_logits"] = None
        if case["drafter"]:
            s["draft_logits"] = (logits + 0.3 * torch.randn(rows, vocab, generator=g, device=dev)).to(kind)
            noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device=dev, dtype=torch.float64).clamp(1e-300, 1.0 - 1e-16)))
            near = s["draft_logits"].double() / case["temperature"] + noise if case["temperature"] else s["draft_logits"]
        else:
            near = logits + torch.randn(rows, vocab, generator=g, device=dev)
        ids = torch.randint(vocab, (rows,), generator=g, device=dev)
        ids[1:] = near.argmax(1)[:-1]
        s["ids"] = ids
        s["uniforms"] = torch.rand(rows, 2, generator=g, device=dev)
        return s
    ps, h, kv, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    groups = len(z["prefix"])
    # pages: those of the prefixes, then those of the sequences, in the order in which a long-running pool hands them out;
    # they hold what was there before
    prefix_pages = [-(-p // ps) for p in z["prefix"]]
    own_pages = [-(-(max(l, 0) + t) // ps) for l, t in zip(z["lengths"], z["tokens"])]
    total = sum(prefix_pages) + sum(own_pages) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    rng = random.Random(seed)

    def table(counts, at):
        first, width = ints(_offsets(counts)[:-1]) + at, max(counts) + 1
        col = torch.arange(width, dtype=torch.int32, device=dev)
        there = col < ints(counts)[:, None]
        return torch.where(there, order[(first[:, None] + col).clamp_max(total - 1).long()], -1)

    s["prefix_table"] = table(prefix_pages, 0) if max(z["prefix"]) > 0 else None
    s["prefix_lengths"] = ints(z["prefix"]) if max(z["prefix"]) > 0 else None
    s["page_table"] = table(own_pages, sum(prefix_pages))
    if case.get("dropped"):
        # the middle pages of a third of the longer sequences have been dropped
        drop = [i for i, c in enumerate(own_pages) if c >= 6 and rng.random() < 0.34]
        col = torch.arange(s["page_table"].shape[1], dtype=torch.int32, device=dev)
        of = torch.zeros(n, dtype=torch.bool, device=dev)
        of[drop] = True
        s["page_table"].masked_fill_(of[:, None] & (col >= 2) & (col < ints(own_pages)[:, None] - 3), -1)
    for name in ("k_pages", "v_pages"):
        pages = torch.randint(0, 256, (total, kv, ps // 16, 9 * d), generator=g, device=dev, dtype=torch.uint8)
        # scales from 1/16 to 1/2: values of variance one, more or less
        pages[..., 8 * d:] = torch.randint(0x18, 0x31, pages[..., 8 * d:].shape, generator=g, device=dev, dtype=torch.uint8)
        s[name] = pages
    s["lengths"] = ints(z["lengths"])
    if case["kind"] == "attention":
        # queries as the rotation leaves them: some rows look at a few keys, others at many
        sharp = 0.5 + 1.5 * torch.rand(rows, h, 1, generator=g, device=dev)
        s["q"] = (torch.randn(rows, h, d, generator=g, device=dev) * sharp).bfloat16()
    else:
        # one fused projection's output, rows of q | k | v
        rot = case["rot"]
        last = max(max(l, 0) + t for l, t in zip(z["lengths"], z["tokens"]))
        angle = torch.arange(last, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
            -torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        s["rotary"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["qkv"] = torch.randn(rows, (h + 2 * kv) * d, generator=g, device=dev).to(NAMES[case["dtype"]])
    if case["tokens"] == 1:
        s["row_offsets"] = None
    return s


# ------------------------------------------------------------------------------------------------ plain form


def _split(s):
    """q, k and v of the fused rows, as views"""
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"]
    return (x[:, :h * d].unflatten(1, (h, d)), x[:, h * d:(h + kv) * d].unflatten(1, (kv, d)),
            x[:, (h + kv) * d:].unflatten(1, (kv, d)))


def _row_tokens(s):
    """sequence and index among its own tokens of every row"""
    counts = torch.tensor(s["host"]["tokens"], device=s["row_offsets"].device if s["row_offsets"] is not None else s["lengths"].device)
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    first = counts.cumsum(0) - counts
    return seq, torch.arange(seq.numel(), device=seq.device) - first[seq]


def _e4m3_values(dev):
    """the value of each of the 127 scale bytes 0 .. 0x7e, fp32"""
    b = torch.arange(127, device=dev)
    e, m = b >> 3, (b & 7).float()
    return torch.where(e > 0, torch.exp2(e.float() - 7) * (1 + m / 8), m * 2.0 ** -9)


def _values(pages):
    """u8 [..., 9 D] -> fp32 [..., 16, D]"""
    d = pages.shape[-1] // 9
    codes = pages[..., :8 * d].unflatten(-1, (16, d // 2))
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=pages.device)
    scale = _e4m3_values(pages.device)[pages[..., 8 * d:].unflatten(-1, (16, d // 16)).int()]
    return lut[codes.int()] * scale.repeat_interleave(16, -1)


def _rotate(x, cos, sin, interleaved):
    """x [rows, heads, d] in 32 bits; cos, sin [rows, rot / 2].  Products and sums are rounded one by one."""
    half = cos.shape[1]
    c, n = cos[:, None], sin[:, None]
    y = x.float().clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * c - b * n
    y[..., second] = b * c + a * n
    return y


def _quantize(x):
    """fp32 [rows, heads, d] -> codes u8 [rows, heads, d / 2], scales u8 [rows, heads, d / 16]: the scale nearest to a sixth of
    the largest of 16 values, then the values nearest to their quotients by it, ties to the even code"""
    blocks = x.unflatten(-1, (-1, 16))
    byte_values = _e4m3_values(x.device)
    t = blocks.abs().amax(-1)
    t = (t / torch.full_like(t, 6.0)).clamp_max(448.0)
    up = torch.bucketize(t, (byte_values[:-1] + byte_values[1:]) / 2)  # (a tie goes down)
    below = up.clamp_max(125)
    even = (t == (byte_values[below] + byte_values[below + 1]) / 2) & (up % 2 == 1) & (up < 126)
    byte = up + even.int()
    scale = byte_values[byte]
    q = (blocks / torch.where(scale > 0, scale, 1.0)[..., None]) * (scale > 0)[..., None]
    a = q.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = (code | ((q < 0).int() << 3)).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def _plain_append(s):
    case, ps, d = s["case"], s["case"]["page"], s["case"]["dim"]
    q, k, v = _split(s)
    seq, i = _row_tokens(s)
    t = s["lengths"].long()[seq] + i
    cs = s["rotary"][t.clamp_min(0)]
    half = cs.shape[1] // 2
    active = s["lengths"][seq] >= 0
    q_out = (_rotate(q, cs[:, :half], cs[:, half:], case["interleaved"]) * active[:, None, None]).bfloat16()
    page = s["page_table"][seq, t.clamp_min(0) // ps].long()
    keep = (active & (page >= 0)).nonzero()[:, 0]
    page, unit, at = page[keep], t[keep] % ps // 16, t[keep] % 16
    for pages, x in ((s["k_pages"], _rotate(k, cs[:, :half], cs[:, half:], case["interleaved"])), (s["v_pages"], v.float())):
        codes, scales = _quantize(x[keep])
        pages[..., :8 * d].unflatten(-1, (16, d // 2))[page, :, unit, at] = codes
        pages[..., 8 * d:].unflatten(-1, (16, d // 16))[page, :, unit, at] = scales
    return q_out


def _plain_values(pages):
    """as the cache's bf16 form has them: [pages, page_size, kv_heads, head_dim]"""
    return _values(pages).flatten(2, 3).transpose(1, 2).bfloat16()


def _run_of(pages, table):
    """keys or values of the pages of each row of a table: fp32 [rows, kv_heads, tokens, d]"""
    x = _values(pages[table.clamp_min(0).long()])  # [rows, table, kv, units, 16, d]
    return x.flatten(3, 4).permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    h, kv, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    per, groups, beams = h // kv, case["groups"], case["beams"]
    dev, lens = q.device, s["lengths"].long()
    tmax = max(s["host"]["tokens"])
    seq, i = _row_tokens(s)
    qp = torch.zeros(lens.numel(), tmax, kv, per, d, device=dev)
    qp[seq, i] = q.float().unflatten(1, (kv, per))
    qp = qp.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [sequences, kv, tmax per, d]
    # own tokens
    k, v = _run_of(s["k_pages"], s["page_table"]), _run_of(s["v_pages"], s["page_table"])
    j = torch.arange(k.shape[2], device=dev)
    last = torch.where(lens[:, None] >= 0, lens[:, None] + torch.arange(tmax, device=dev), -1)  # that row i sees
    seen = (j <= last[..., None]) & (s["page_table"] >= 0).repeat_interleave(ps, 1)[:, None]
    x = torch.matmul(qp, k.transpose(2, 3)) * d ** -0.5
    x.masked_fill_(~seen.repeat_interleave(per, 1)[:, None], float("-inf"))
    m = x.amax(-1)
    if s["prefix_table"] is not None:
        # the rows of a group together
        qg = qp.unflatten(0, (groups, beams)).transpose(1, 2).flatten(2, 3)  # [groups, kv, beams tmax per, d]
        kp, vp = _run_of(s["k_pages"], s["prefix_table"]), _run_of(s["v_pages"], s["prefix_table"])
        xp = torch.matmul(qg, kp.transpose(2, 3)) * d ** -0.5
        xp.masked_fill_((torch.arange(kp.shape[2], device=dev) >= s["prefix_lengths"].long()[:, None])[:, None, None], float("-inf"))
        m = torch.maximum(m, xp.amax(-1).unflatten(2, (beams, -1)).transpose(1, 2).flatten(0, 1))
    m = m.clamp_min(-1e30)
    w = torch.exp(x.sub_(m[..., None]))
    total, o = w.sum(-1), torch.matmul(w, v)
    if s["prefix_table"] is not None:
        w = torch.exp(xp.sub_(m.unflatten(0, (groups, beams)).transpose(1, 2).flatten(2, 3)[..., None]))
        total = total + w.sum(-1).unflatten(2, (beams, -1)).transpose(1, 2).flatten(0, 1)
        o = o + torch.matmul(w, vp).unflatten(2, (beams, -1)).transpose(1, 2).flatten(0, 1)
    o = o / total.clamp_min(1e-30)[..., None] * (lens >= 0)[:, None, None, None]
    return o.unflatten(2, (tmax, per)).transpose(1, 2)[seq, i].flatten(1, 2).bfloat16()


def _plain_verify(s):
    """in 64 bits: a draft stands or falls by one comparison, a token by where a sum passes a number"""
    case = s["case"]
    t, ids, off = case["temperature"], s["ids"], s["row_offsets"].long()
    n, rows = off.numel() - 1, ids.numel()
    r = torch.arange(rows, device=ids.device)
    seq, i = _row_tokens(s)
    last = r == off[1:][seq] - 1
    drafted = torch.roll(ids, -1)[:, None]
    if t == 0.0:
        best = s["logits"].argmax(1)  # (the first of equals)
        stands = best == drafted[:, 0]
    else:
        def likely(x):
            e = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / t)
            return e / e.sum(1, keepdim=True)

        p = likely(s["logits"])
        q = torch.zeros_like(p).scatter_(1, drafted, 1.0) if s["draft_logits"] is None else likely(s["draft_logits"])
        stands = s["uniforms"][:, 0].double() * q.gather(1, drafted)[:, 0] < p.gather(1, drafted)[:, 0]
    stands = stands & ~last
    # rows up to the first draft that falls
    falls = torch.where(stands, rows, i)
    accepted = torch.full((n,), rows, device=ids.device).scatter_reduce_(0, seq, falls, "amin")
    end = off[:-1] + accepted
    if t == 0.0:
        return accepted.int(), best[end].int()
    rest = torch.where(last[end, None], p[end], (p[end] - q[end]).clamp_min(0.0))
    rest = torch.where((rest.sum(1, keepdim=True) > 0), rest, p[end])
    sums = rest.cumsum(1)
    passed = sums > s["uniforms"][end, 1].double()[:, None] * sums[:, -1:]
    return accepted.int(), passed.int().argmax(1).int()


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from velox_voice_b200 import ops

        if kind == "verify":
            accepted, follows = ops.verify_drafts(s["logits"], s["ids"], s["uniforms"], draft_logits=s["draft_logits"], row_offsets=s["row_offsets"],
                                                  temperature=case["temperature"])
            return {"accepted": accepted, "next": follows}
        if kind == "attention":
            return ops.prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["prefix_table"], s["prefix_lengths"],
                                        row_offsets=s["row_offsets"])
        q, k, v = _split(s)
        q = ops.kv_append(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], q=q, rotary=s["rotary"], interleaved=case["interleaved"],
                          row_offsets=s["row_offsets"])
        return {"q": q, "k": ops.kv_values(s["k_pages"]), "v": ops.kv_values(s["v_pages"])}
    if kind == "verify":
        accepted, follows = _plain_verify(s)
        return {"accepted": accepted, "next": follows}
    if kind == "attention":
        return _plain_attention(s)
    return {"q": _plain_append(s), "k": _plain_values(s["k_pages"]), "v": _plain_values(s["v_pages"])}


def work(case):
    """Bytes and operations of one pass: sequences that take part and their keys (dropped pages count as read); of an
    appended cache also its values, which a pass returns."""
    z = _sizes(case)
    rows = sum(z["tokens"])
    if case["kind"] == "verify":
        cells = (rows + (rows - len(z["tokens"]) if case["drafter"] and case["temperature"] else 0)) * case["vocab"]
        return {"bytes": cells * (4 if case["dtype"] == "float32" else 2) + rows * 16, "flops": 4 * cells}
    h, kv, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "float32" else 2
        positions = min(rows, max(l + t for l, t in zip(z["lengths"], z["tokens"])))
        places = ps * (sum(-(-(l + t) // ps) for l, t in zip(z["lengths"], z["tokens"])) + 3)
        nbytes = rows * ((h + 2 * kv) * d * size + h * d * 2 + kv * d * 9 // 8) + positions * case["rot"] * 4
        return {"bytes": nbytes + places * kv * d * (4 + 9 / 8), "flops": rows * ((h + kv) * case["rot"] * 3 + 2 * kv * d * 4)}
    nbytes, flops = 2 * rows * h * d * 2 + sum(z["prefix"]) * kv * d * 9 / 8, 0
    for at, (l, t) in enumerate(zip(z["lengths"], z["tokens"])):
        if l >= 0:
            nbytes += (l + t) * kv * d * 9 / 8
            flops += 4 * h * d * (t * z["prefix"][at // case["beams"]] + t * l + t * (t + 1) // 2)
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------ 64 bits


def _exact_values(pages):
    """u8 [n, 9 D] units -> fp64 [n, 16, D]: a code is sign, two bits of exponent and one of significand; a scale four and three"""
    d = pages.shape[1] // 9
    codes = pages[:, :8 * d].long().view(-1, 16, d // 2, 1) >> torch.tensor([0, 4], device=pages.device) & 15
    e, m = codes >> 1 & 3, (codes & 1).double()
    mag = torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1).double(), m / 2) * (1 - 2 * (codes >> 3)).double()
    b = pages[:, 8 * d:].long().view(-1, 16, d // 16, 1)
    be, bm = b >> 3, (b & 7).double() / 8
    scale = torch.where(be > 0, (1 + bm) * 2.0 ** (be - 7).double(), bm * 2.0 ** -6)
    return (mag.flatten(2).view(-1, 16, d // 16, 16) * scale).flatten(2)


def _exact_nearest(x, grid):
    """index of the nearest number of an ascending grid, ties to the even index"""
    up = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    down, a, b = up - 1, x - grid[up - 1], grid[up] - x
    return torch.where((a < b) | ((a == b) & (down % 2 == 0)), down, up)


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence.  What is quantized is the rotated value in 32 bits, each product and sum
    rounded; from there on everything is exact."""
    if case["kind"] == "verify":
        return None
    s = prepare(case, seed)
    z, ps = s["host"], case["page"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    dev = s["lengths"].device
    row_at = _offsets(z["tokens"])
    table = s["page_table"].cpu().tolist()
    if case["kind"] == "append":
        b = torch.arange(127, device=dev).double()
        grid8 = torch.where(b >= 8, (1 + b % 8 / 8) * 2.0 ** (b // 8 - 7), b * 2.0 ** -9)
        grid4 = torch.tensor(E2M1, device=dev, dtype=torch.float64)
        half = case["rot"] // 2
        units = {name: _exact_values(s[name].reshape(-1, 9 * d)).view(-1, kv, ps // 16, 16, d) for name in ("k_pages", "v_pages")}
        x32 = s["qkv"].float().view(-1, h + 2 * kv, d)
        x = x32.double()
        q_out = torch.zeros(x.shape[0], h, d, dtype=torch.float64, device=dev)
        first = torch.arange(half, device=dev) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        for n, (l, t) in enumerate(zip(z["lengths"], z["tokens"])):
            rows = slice(row_at[n], row_at[n + 1])
            cs = s["rotary"][l:l + t, None]
            c, e = cs[..., :half], cs[..., half:]
            y = x[rows, :h].clone()
            y[..., first], y[..., second] = (x[rows, :h][..., first] * c - x[rows, :h][..., second] * e,
                                             x[rows, :h][..., second] * c + x[rows, :h][..., first] * e)
            q_out[rows] = y
            k32 = x32[rows, h:h + kv].clone()
            a, b2 = k32[..., first].clone(), k32[..., second].clone()
            k32[..., first], k32[..., second] = a.mul(c).sub(b2.mul(e)), b2.mul(c).add(a.mul(e))
            where = torch.arange(l, l + t, device=dev)
            pages = torch.tensor(table[n], device=dev)[where // ps]
            for name, v in (("k_pages", k32), ("v_pages", x32[rows, h + kv:])):
                v = v.double().unflatten(-1, (-1, 16))
                # (a sixth of the largest as 32 bits hold it, as the operator says)
                byte = _exact_nearest((v.abs().amax(-1) / 6.0).float().double().clamp_max(448.0), grid8)
                scale = grid8[byte][..., None]
                code = _exact_nearest((v.abs() / scale.clamp_min(1e-30)).clamp_max(6.0), grid4)
                v = (grid4[code] * torch.sign(v) * scale).flatten(-2)
                units[name][pages, :, where % ps // 16, where % 16] = v
        values = {n: u.flatten(2, 3).transpose(1, 2) for n, u in units.items()}
        return {"q": q_out, "k": values["k_pages"], "v": values["v_pages"]}
    q = s["q"].double()
    out = torch.zeros_like(q)

    def run_of(name, row, index):
        pages = torch.tensor(row, device=dev)[index // ps]
        index, pages = index[pages >= 0], pages[pages >= 0]
        unit = s[name][pages, :, index % ps // 16].flatten(0, 1)  # [tokens kv, 9 d]
        at = (index % 16).repeat_interleave(kv)
        return torch.cat([_exact_values(u)[torch.arange(u.shape[0], device=dev), a] for u, a in zip(unit.split(65536), at.split(65536))]).view(-1, kv, d), index

    if s["prefix_table"] is not None:
        prefix = s["prefix_table"].cpu().tolist()
    for n, (l, t) in enumerate(zip(z["lengths"], z["tokens"])):
        g = n // case["beams"]
        if n % case["beams"] == 0 and z["prefix"][g]:
            shared = [run_of(name, prefix[g], torch.arange(z["prefix"][g], device=dev))[0] for name in ("k_pages", "v_pages")]
        if l < 0:
            continue
        k, place = run_of("k_pages", table[n], torch.arange(l + t, device=dev))
        v, _ = run_of("v_pages", table[n], torch.arange(l + t, device=dev))
        if z["prefix"][g]:
            k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
            place = torch.cat([torch.full((z["prefix"][g],), -1, device=dev), place])
        rows = slice(row_at[n], row_at[n + 1])
        late = place > l + torch.arange(t, device=dev)[:, None]
        for e in range(h):
            x = (q[rows, e] @ k[:, e // (h // kv)].t() / math.sqrt(d)).masked_fill(late, float("-inf"))
            out[rows, e] = torch.softmax(x, -1) @ v[:, e // (h // kv)]
    return out
