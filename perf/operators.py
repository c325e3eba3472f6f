"""The paged cache of keys and values and the attention that reads it, as cases that can be timed: `kv_append` (new
keys and values into their pages, rotated by position on the way) and `prefix_attention` (sequences that share a
long prefix, which is read once for all of them), each in a plain form and through the public entry points.

What the sizes stand for: the hypotheses of an utterance share its encoder frames (40 ms each: 375 for a quarter of a
minute, 3,750 for a full span of long audio, 89,999 for an hour) and differ in the tokens they have decoded; ten are
rescored or decoded together.  Heads are the encoder's (8 of 64) or grouped ones of a larger decoder (32 query heads on
8 key heads of 128)."""

import math
import random

import torch

own = False

NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one decoding step of the ten hypotheses of one utterance: launches and host time only
        _append("append_beam_step", seqs=10, tokens=1, history=40, heads=8, kv_heads=8, dim=64, rot=64, page=16),
        # one step of a busy server: 256 sequences, grouped heads
        _append("append_serve_step", seqs=256, tokens=1, history=700, heads=32, kv_heads=8, dim=128, rot=128, page=64),
        # the frames of one span of long audio become the prefix; rows in fp32 as a linear leaves them by default
        _append("append_span", seqs=1, tokens=3750, history=0, heads=8, kv_heads=8, dim=64, rot=64, page=16,
                dtype="float32", interleaved=True),
        # prompts of a batch, together an hour of audio, half of each head rotated
        _append("append_hour", seqs=24, tokens=5000, history=0, heads=32, kv_heads=8, dim=128, rot=64, page=32),
        # one decoding step of ten hypotheses over a short utterance
        _attention("beam_utterance", groups=1, beams=10, tokens=1, prefix=375, history=24, heads=8, kv_heads=8, dim=64, page=16),
        # the same for a batch of sixteen spans
        _attention("beam_batch", groups=16, beams=10, tokens=1, prefix=3750, history=90, heads=8, kv_heads=8, dim=64, page=16),
        # rescoring: every hypothesis whole, of utterances of a minute and less, not the same number for each
        _attention("rescore_batch", groups=16, beams=10, tokens=60, prefix=1537, history=0, heads=8, kv_heads=8, dim=64, page=16,
                   ragged=True),
        # 64 answers to one long prompt
        _attention("shared_prompt", groups=1, beams=64, tokens=1, prefix=8191, history=512, heads=32, kv_heads=8, dim=128, page=64),
        # 32 hypotheses over an hour of audio
        _attention("shared_hour", groups=1, beams=32, tokens=1, prefix=89999, history=300, heads=32, kv_heads=8, dim=128, page=32),
        # eight prompts with their sequences, some pages of long sequences dropped, some sequences finished
        _attention("several_prompts", groups=8, beams=24, tokens=1, prefix=4096, history=1024, heads=32, kv_heads=8, dim=128, page=32,
                   ragged=True, dropped=True),
        # prompt chunks of four sequences behind a shared prompt
        _attention("prompt_chunks", groups=1, beams=4, tokens=2048, prefix=16384, history=500, heads=32, kv_heads=8, dim=128, page=64),
        # a whole step of a decoder layer: rotate and append, then attend
        _attention("decode_step", groups=4, beams=16, tokens=1, prefix=2000, history=200, heads=16, kv_heads=16, dim=64, page=16,
                   kind="step"),
    ]


def _append(name, **kw):
    return {"name": name, "kind": "append", "dtype": "bfloat16", "interleaved": False, **kw}


def _attention(name, **kw):
    return {"name": name, "kind": "attention", "ragged": False, "dropped": False, **kw}


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice(((8, 8, 64), (8, 8, 64), (16, 4, 64), (32, 8, 128), (32, 8, 128), (12, 4, 128), (20, 2, 128)))
    page = rng.choice((16, 16, 32, 64, 24, 128))
    common = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    kind = rng.choice(("append", "append", "step", "decode", "decode", "rescore", "chunks"))
    if kind == "append":
        tokens = rng.choice((1, _log_size(rng, 2, 6000)))
        seqs = _log_size(rng, 1, min(512, max(2, 90000 // tokens)))
        return {"kind": "append", "seqs": seqs, "tokens": tokens, "history": rng.randrange(0, 500), "rot": rng.choice((dim, dim // 2, dim)),
                "dtype": rng.choice(("bfloat16", "bfloat16", "float32")), "interleaved": rng.random() < 0.4, **common}
    groups = _log_size(rng, 1, 16)
    case = {"kind": "step" if kind == "step" else "attention", "groups": groups, "ragged": groups > 1 and rng.random() < 0.5,
            "dropped": rng.random() < 0.25, **common}
    if kind in ("step", "decode"):
        case.update(beams=_log_size(rng, 1, 512 // groups), tokens=1, prefix=rng.choice((0, _log_size(rng, 16, 90000 // groups))),
                    history=_log_size(rng, 1, 2000))
    elif kind == "rescore":
        case.update(beams=_log_size(rng, 2, 16), tokens=_log_size(rng, 2, 100), prefix=_log_size(rng, 64, 4000), history=0)
    else:
        case.update(groups=1, ragged=False, beams=rng.randrange(1, 5), tokens=_log_size(rng, 200, 2048), prefix=rng.choice((0, _log_size(rng, 100, 16384))),
                    history=rng.randrange(0, 500))
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _sizes(case):
    """Rows, lengths and groups of a case: host numbers, the same whatever the seed of the values.  Sequences are between half
    and all of the case's sizes long; a few of a large ragged batch have finished (length -1)."""
    rng = random.Random(17)

    def around(n):
        return n if n <= 1 else rng.randint((n + 1) // 2, n)

    if case["kind"] == "append":
        groups, sizes = 1, [case["seqs"]]
    else:
        groups = case["groups"]
        sizes = [around(case["beams"]) if case["ragged"] else case["beams"] for _ in range(groups)]
    n = sum(sizes)
    tokens = [around(case["tokens"]) for _ in range(n)]
    lengths = [around(case["history"]) for _ in range(n)]
    if case.get("ragged") and n >= 32:
        for i in range(n):
            if rng.random() < 0.04:
                lengths[i] = -1
    prefix = [around(case.get("prefix", 0)) if groups > 1 else case.get("prefix", 0) for _ in range(groups)]
    return {"sizes": sizes, "tokens": tokens, "lengths": lengths, "prefix": prefix}


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    z = _sizes(case)
    ps, h, kv, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    n, rows = len(z["tokens"]), sum(z["tokens"])
    groups = len(z["sizes"])

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    # pages: those of the prefixes, then those of the sequences, in the order in which a long-running pool hands them out;
    # they hold what was there before
    prefix_pages = [-(-p // ps) for p in z["prefix"]]
    own_pages = [-(-(max(l, 0) + t) // ps) for l, t in zip(z["lengths"], z["tokens"])]
    total = sum(prefix_pages) + sum(own_pages) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    rng = random.Random(seed)
    at = 0

    def table(counts):
        nonlocal at
        t = torch.full((len(counts), max(counts) + 1), -1, dtype=torch.int32, device=dev)
        for i, c in enumerate(counts):
            t[i, :c] = order[at:at + c]
            at += c
        return t

    prefix_table = table(prefix_pages) if max(z["prefix"]) > 0 else None
    page_table = table(own_pages)
    if case.get("dropped"):
        # the middle pages of a third of the longer sequences have been dropped
        for i, c in enumerate(own_pages):
            if c >= 6 and rng.random() < 0.34:
                page_table[i, 2:c - 3] = -1
    k_pages = torch.randn(total, ps, kv, d, generator=g, device=dev, dtype=torch.bfloat16)
    v_pages = torch.randn(total, ps, kv, d, generator=g, device=dev, dtype=torch.bfloat16)
    s = {"case": case, "host": z, "k_pages": k_pages, "v_pages": v_pages, "page_table": page_table, "lengths": ints(z["lengths"]),
         "row_offsets": None if case["tokens"] == 1 else ints(_offsets(z["tokens"])),
         "prefix_table": prefix_table, "prefix_lengths": None if prefix_table is None else ints(z["prefix"]),
         "group_offsets": ints(_offsets(z["sizes"])) if case.get("ragged") else None}
    if case["kind"] == "attention":
        # queries as the rotation leaves them: some rows look at a few keys, others at many
        sharp = 0.5 + 1.5 * torch.rand(rows, h, 1, generator=g, device=dev)
        s["q"] = (torch.randn(rows, h, d, generator=g, device=dev) * sharp).bfloat16()
    else:
        # one fused projection's output, rows of q | k | v
        rot = case.get("rot", d)
        start = [p for p, c in zip(z["prefix"], z["sizes"]) for _ in range(c)]
        last = max(a + max(l, 0) + t for a, l, t in zip(start, z["lengths"], z["tokens"]))
        angle = torch.arange(last, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
            -torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        s["rotary"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["starts"] = ints(start)
        s["qkv"] = torch.randn(rows, (h + 2 * kv) * d, generator=g, device=dev).to(NAMES[case.get("dtype", "bfloat16")])
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
    counts = s["host"]["tokens"]
    n = len(counts)
    dev = s["lengths"].device
    if s["row_offsets"] is None:
        seq = torch.arange(n, device=dev)
        return seq, s["lengths"].long()
    off = s["row_offsets"].long()
    seq = torch.repeat_interleave(torch.arange(n, device=dev), off[1:] - off[:-1], output_size=sum(counts))
    return seq, s["lengths"].long()[seq] + torch.arange(sum(counts), device=dev) - off[seq]


def _rotate(x, cos, sin, interleaved):
    """x [rows, heads, d] in 32 bits; cos, sin [rows, rot / 2]"""
    half = cos.shape[1]
    c, n = cos[:, None], sin[:, None]
    y = x.float().clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2].float(), x[..., 1:2 * half:2].float()
        y[..., 0:2 * half:2] = a * c - b * n
        y[..., 1:2 * half:2] = b * c + a * n
    else:
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        y[..., :half] = a * c - b * n
        y[..., half:2 * half] = b * c + a * n
    return y


def _plain_append(s):
    case, ps = s["case"], s["case"]["page"]
    q, k, v = _split(s)
    seq, t = _row_tokens(s)
    active = s["lengths"][seq] >= 0
    pos = (s["starts"][seq] + t).clamp_min(0)
    cs = s["rotary"][pos]
    half = cs.shape[1] // 2
    inter = case.get("interleaved", False)
    q_out = (_rotate(q, cs[:, :half], cs[:, half:], inter) * active[:, None, None]).bfloat16()
    page = s["page_table"][seq, t.clamp_min(0) // ps].long()
    keep = (active & (page >= 0)).nonzero()[:, 0]
    page, slot = page[keep], t[keep] % ps
    s["k_pages"][page, slot] = _rotate(k, cs[:, :half], cs[:, half:], inter)[keep].bfloat16()
    s["v_pages"][page, slot] = v[keep].bfloat16()
    return q_out


def _plain_attention(s, q):
    case, z = s["case"], s["host"]
    h, kv, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    per = h // kv
    dev = q.device
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    seq_at, row_at = _offsets(z["sizes"]), _offsets(z["tokens"])
    for g, size in enumerate(z["sizes"]):
        s0, s1 = seq_at[g], seq_at[g + 1]
        r0, r1 = row_at[s0], row_at[s1]
        tmax = max(z["tokens"][s0:s1])
        lens = s["lengths"][s0:s1].long()
        # queries of the group's sequences, padded to the longest: [size, tmax, h, d]
        if tmax == 1:
            qp, rows = q[r0:r1, None].float(), None
        else:
            index = torch.arange(tmax, device=dev)
            count = s["row_offsets"][s0 + 1:s1 + 1] - s["row_offsets"][s0:s1]
            rows = index < count[:, None]
            qp = torch.zeros(size, tmax, h, d, device=dev)
            qp[rows] = q[r0:r1].float()
        qp = qp.view(size, tmax, kv, per, d).permute(2, 0, 1, 3, 4)  # [kv, size, tmax, per, d]
        # own keys: [size, width]
        width = max(max(l, 0) + t for l, t in zip(z["lengths"][s0:s1], z["tokens"][s0:s1]))
        j = torch.arange(width, device=dev)
        table = s["page_table"][s0:s1, :-(-width // ps)].long()
        page = table[:, j // ps]
        limit = lens[:, None] + torch.arange(1, tmax + 1, device=dev)  # keys of row i
        limit = torch.where(lens[:, None] >= 0, limit, 0)
        seen = (j < limit[..., None]) & (page >= 0)[:, None]           # [size, tmax, width]
        slot = j % ps
        there = (page >= 0)[..., None] & (j < (lens + tmax)[:, None])[..., None]
        n_prefix = z["prefix"][g]
        if n_prefix:
            jp = torch.arange(n_prefix, device=dev)
            pp = s["prefix_table"][g].long()[jp // ps]
        acc = torch.empty(kv, size, tmax, per, d, device=dev)
        # as many key heads at a time as keep the scores within a few GB
        step = max(1, min(kv, 2 ** 29 // (size * tmax * per * (width + n_prefix) + size * width * d)))
        for e in range(0, kv, step):
            qe = qp[e:e + step]
            b = qe.shape[0]
            ke, ve = ((c[page.clamp_min(0), slot, e:e + step].float() * there[..., None]).permute(2, 0, 1, 3)
                      for c in (s["k_pages"], s["v_pages"]))  # [b, size, width, d]
            x = torch.matmul(qe.reshape(b, size, tmax * per, d), ke.transpose(2, 3)).view(b, size, tmax, per, width) * d ** -0.5
            x = torch.where(seen[:, :, None], x, float("-inf"))
            m = x.amax(-1)
            if n_prefix:
                kp, vp = (c[pp, jp % ps, e:e + step].float().transpose(0, 1) for c in (s["k_pages"], s["v_pages"]))  # [b, keys, d]
                xp = torch.matmul(qe.reshape(b, size * tmax * per, d), kp.transpose(1, 2)) * d ** -0.5
                m = torch.maximum(m, xp.amax(-1).view(m.shape))
            m = m.clamp_min(-1e30)
            w = torch.exp(x - m[..., None])
            total = w.sum(-1)
            o = torch.matmul(w.view(b, size, tmax * per, width), ve).view(b, size, tmax, per, d)
            if n_prefix:
                w = torch.exp(xp - m.view(b, -1, 1))
                total = total + w.sum(-1).view(total.shape)
                o = o + torch.matmul(w, vp).view(o.shape)
                del xp
            acc[e:e + step] = o / total.clamp_min(1e-30)[..., None]
            del x, w
        acc = acc * (lens >= 0).view(1, size, 1, 1, 1)
        acc = acc.permute(1, 2, 0, 3, 4).reshape(size, tmax, h, d)
        out[r0:r1] = (acc[:, 0] if rows is None else acc[rows]).bfloat16()
    return out


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        from velox_voice_b200 import ops

        if kind != "attention":
            q, k, v = _split(s)
            q = ops.kv_append(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], q=q, rotary=s["rotary"],
                              interleaved=s["case"].get("interleaved", False), row_offsets=s["row_offsets"], starts=s["starts"])
        else:
            q = s["q"]
        if kind != "append":
            out = ops.prefix_attention(q, s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["prefix_table"],
                                       s["prefix_lengths"], row_offsets=s["row_offsets"], group_offsets=s["group_offsets"])
    else:
        q = s["q"] if kind == "attention" else _plain_append(s)
        if kind != "append":
            out = _plain_attention(s, q)
    if kind == "attention":
        return out
    done = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if kind == "step":
        done["out"] = out
    return done


def _distinct_positions(z):
    spans = [(p + max(l, 0), p + max(l, 0) + t) for p, c in zip(z["prefix"], z["sizes"])
             for l, t in list(zip(z["lengths"], z["tokens"]))[:c]]
    return max(b for _, b in spans) - min(a for a, _ in spans)


def work(case):
    """Bytes and operations of one pass: sequences that take part and their keys (dropped pages count as read)."""
    z = _sizes(case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    nbytes = flops = 0
    rows = sum(z["tokens"])
    if case["kind"] != "attention":
        size = 4 if case.get("dtype") == "float32" else 2
        rot = case.get("rot", d)
        positions = min(rows, _distinct_positions(z))
        nbytes += rows * (h + 2 * kv) * d * size + rows * (h + 2 * kv) * d * 2 + positions * rot * 4
        flops += rows * (h + kv) * rot * 3
    if case["kind"] != "append":
        if case["kind"] == "attention":
            nbytes += rows * h * d * 2
        nbytes += rows * h * d * 2 + sum(z["prefix"]) * kv * d * 4
        at = 0
        for p, c in zip(z["prefix"], z["sizes"]):
            for l, t in zip(z["lengths"][at:at + c], z["tokens"][at:at + c]):
                if l < 0:
                    continue
                keys = l + t
                nbytes += keys * kv * d * 4
                flops += 4 * h * d * (t * p + t * l + t * (t + 1) // 2)
            at += c
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    """The definition, sequence by sequence, in 64 bits: rotation as a product of complex numbers, attention over the list of
    the sequence's keys."""
    s = prepare(case, seed)
    z, ps = s["host"], case["page"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    dev = s["k_pages"].device
    kp, vp = s["k_pages"], s["v_pages"]
    row_at = _offsets(z["tokens"])
    table = s["page_table"].cpu().tolist()
    done = {}
    q_all = s.get("q")
    if case["kind"] != "attention":
        kp, vp = kp.double(), vp.double()
        x = s["qkv"].double()
        starts = s["starts"].cpu().tolist()
        rot = s["rotary"].shape[1]
        turn = torch.complex(s["rotary"][:, :rot // 2].double(), s["rotary"][:, rot // 2:].double())
        q_all = torch.zeros(x.shape[0], h, d, dtype=torch.float64, device=dev)

        def turned(y, p):
            first, rest = y[..., :rot], y[..., rot:]
            if case.get("interleaved"):
                w = torch.view_as_complex(first.reshape(*first.shape[:-1], rot // 2, 2).contiguous()) * p[:, None]
                first = torch.view_as_real(w).flatten(-2)
            else:
                w = torch.complex(first[..., :rot // 2].contiguous(), first[..., rot // 2:].contiguous()) * p[:, None]
                first = torch.cat([w.real, w.imag], -1)
            return torch.cat([first, rest], -1)

        for i, (l, t) in enumerate(zip(z["lengths"], z["tokens"])):
            if l < 0:
                continue
            rows = slice(row_at[i], row_at[i + 1])
            p = turn[starts[i] + l:starts[i] + l + t]
            y = x[rows].view(t, h + 2 * kv, d)
            q_all[rows] = turned(y[:, :h], p)
            pages = torch.tensor([table[i][j // ps] for j in range(l, l + t)], device=dev)
            slots = torch.arange(l, l + t, device=dev) % ps
            there = pages >= 0
            kp[pages[there], slots[there]] = turned(y[:, h:h + kv], p)[there]
            vp[pages[there], slots[there]] = y[:, h + kv:][there]
        done = {"q": q_all, "k_pages": kp, "v_pages": vp}
        if case["kind"] == "append":
            return done
        # attention reads what the cache and the rotated queries hold: bf16
        kp, vp, q_all = kp.bfloat16(), vp.bfloat16(), q_all.bfloat16()
    out = torch.zeros(q_all.shape[0], h, d, dtype=torch.float64, device=dev)
    at = 0
    for g, size in enumerate(z["sizes"]):
        n = z["prefix"][g]
        if n:
            pages = s["prefix_table"][g].long().repeat_interleave(ps)[:n]
            slots = torch.arange(n, device=dev) % ps
            prefix_k, prefix_v = (c[pages, slots].double().transpose(0, 1) for c in (kp, vp))  # [kv, n, d]
        for i in range(at, at + size):
            l, t = z["lengths"][i], z["tokens"][i]
            if l < 0:
                continue
            index = [j for j in range(l + t) if table[i][j // ps] >= 0]
            pages = torch.tensor([table[i][j // ps] for j in index], device=dev, dtype=torch.long)
            number = torch.tensor(index, device=dev, dtype=torch.long)
            k, v = (c[pages, number % ps].double().transpose(0, 1) for c in (kp, vp))
            if n:
                k, v = torch.cat([prefix_k, k], 1), torch.cat([prefix_v, v], 1)
            place = torch.cat([torch.full((n,), -1, device=dev, dtype=torch.long), number])
            rows = slice(row_at[i], row_at[i + 1])
            late = place > l + torch.arange(t, device=dev)[:, None]  # [t, keys]
            for e in range(kv):
                qe = q_all[rows, e * (h // kv):(e + 1) * (h // kv)].double().transpose(0, 1)  # [per, t, d]
                x = (qe @ k[e].t() / math.sqrt(d)).masked_fill(late, float("-inf"))
                out[rows, e * (h // kv):(e + 1) * (h // kv)] = (torch.softmax(x, -1) @ v[e]).transpose(0, 1)
        at += size
    if case["kind"] == "attention":
        return out
    done["out"] = out
    return done
