"""The operators that answer in 4 bits, as measurable cases:

  append   new keys (rotated) and values into a paged cache that holds them in 4
           bits, and the new tokens' values read back from it
  read     cached tokens read back
  attend   attention of each sequence's new tokens over its cached keys
  project  products of a few tokens (or a prompt's chunk) with base weights held
           in 4 bits, with their biases and adapters

A case is a dict of plain values.  The lengths of a batch are drawn from the
case's own values, so that every seed of a case does the same work.

Pages.  A page holds, for every KV head, 16 G P bytes of 4-bit numbers n and then
2 G P bytes of fp16 scales s (P tokens a page, G groups of 32 columns); a number
stands for (n - 8) s of its group.  A 32-bit word has columns 8 x + 2 j in its bits
4 j and 8 x + 2 j + 1 in its bits 16 + 4 j.  Keys: word (row 4 + c) G + i holds
columns 32 i + 8 c .., scale row G + i is group i's.  Values: word (row / 4 4 G + r)
4 + row % 4 holds columns 8 r .., scale (row / 4 G + i) 4 + row % 4 is group i's.

Weights.  [out / 16][in / 128][64] times four words: word i of entry 16 c + r holds
row r's columns 32 i + 8 c .. of the block; then the scales [out / 16][in / 128][16]
[128 / group] in fp16, then, where there are any, the offsets alike: a weight is
(n - 8) s + offset.
Rows and columns are padded with zeros.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST = 2688.0  # of the cache's scales
_engine = None


def _lib():
    """The framework's engine (own only)."""
    global _engine
    if _engine is None:
        sys.path.insert(0, os.path.abspath("glacier.tune_amd"))
        import glacier_attn as ga

        _engine = ga.GpuAttentionEngine(torch.cuda.current_device(), ga.PREC_BF16)
    return _engine


def _batch(kind, seqs, new_lo, new_hi, kv_lo, kv, heads_q, heads_kv, head_dim, page, dtype="bf16",
           theta=1.0e6, pad=0):
    """seqs sequences of new_lo .. new_hi new tokens (all of them for read), kv_lo .. kv
    tokens each with them; pad: rows behind the last sequence."""
    return {"kind": kind, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "kv_lo": kv_lo, "kv": kv,
            "heads_q": heads_q, "heads_kv": heads_kv, "head_dim": head_dim, "page": page,
            "dtype": dtype, "theta": theta, "pad": pad}


def _project(tokens, width, outs, group, rank=0, mins=False, bias=False, dtype="bf16"):
    """outs: the projections' widths, joined by commas."""
    return {"kind": "project", "tokens": tokens, "width": width, "outs": outs, "group": group,
            "rank": rank, "mins": mins, "bias": bias, "dtype": dtype}


def listed():
    named = {
        # a step of 64 answers at once
        "append_tokens_64": _batch("append", 64, 1, 1, 1, 1024, 28, 4, 128, 16),
        # a packed batch of prompts of ragged lengths
        "append_prompts_16": _batch("append", 16, 64, 512, 64, 512, 32, 8, 128, 64, theta=5.0e5),
        # a short shared beginning, looked at in the checking mode
        "read_prefix_200_fp32": _batch("read", 1, 200, 200, 200, 200, 14, 2, 64, 16, dtype="fp32"),
        # whole sequences taken out of the cache, to be kept elsewhere
        "read_sequences_16": _batch("read", 16, 300, 4096, 300, 4096, 32, 8, 128, 64),
        # the first words of a single short answer
        "attend_token_512": _batch("attend", 1, 1, 1, 512, 512, 14, 2, 64, 16),
        # a serving step: 32 answers, contexts short to long
        "attend_tokens_32": _batch("attend", 32, 1, 1, 64, 8192, 28, 4, 128, 16),
        # one answer over a document
        "attend_token_65536": _batch("attend", 1, 1, 1, 65536, 65536, 32, 8, 128, 64),
        # a long prompt's chunk over what is cached of it already
        "attend_chunk_2048": _batch("attend", 1, 2048, 2048, 8192, 8192, 28, 4, 128, 64),
        # the checking mode: short chunks of ragged lengths, a head size between the usual ones
        "attend_chunks_3_fp32": _batch("attend", 3, 17, 120, 200, 1001, 8, 2, 96, 32, dtype="fp32", pad=5),
        # queries, keys and values of one token of an answer, with the tuned adapters
        "project_qkv_token": _project(1, 3584, "3584,512,512", 32, rank=16, bias=True),
        # the first half of the feed-forward for 16 answers at once, offsets among the weights
        "project_ffn_tokens_16": _project(16, 3584, "18944,18944", 128, mins=True),
        # a small model's prompt, of odd length
        "project_qkv_prompt_333": _project(333, 896, "896,128,128", 32, rank=16, bias=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "project", "project"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "project":
        width, outs = rng.choice([(3584, "3584,512,512"), (3584, "18944,18944"), (18944, "3584"),
                                  (4096, "4096,1024,1024"), (4096, "4096"), (896, "896,128,128"),
                                  (896, "4864"), (4864, "896"), (2048, "2048,256"), (1120, "1000,36")])
        group = rng.choice([g for g in (32, 32, 64, 128) if width % g == 0])
        return _project(_log(rng, 1, 512), width, outs, group, rng.choice([0, 0, 8, 16, 64]),
                        rng.random() < 0.4, rng.random() < 0.5, dtype)
    hq, hkv, d = rng.choice([(28, 4, 128), (32, 8, 128), (14, 2, 64), (12, 2, 128), (8, 8, 64),
                             (8, 2, 96), (5, 1, 80), (8, 2, 256), (16, 4, 32), (40, 8, 128)])
    page = rng.choice([16, 32, 64, 128])
    seqs = _log(rng, 1, 64)
    theta = rng.choice([1.0e4, 5.0e5, 1.0e6])
    if kind == "append":
        new = _log(rng, 1, 512)
        return _batch(kind, seqs, max(1, new // 4), new, max(1, new // 4), new + _log(rng, 1, 512), hq, hkv, d,
                      page, dtype, theta)
    if kind == "read":
        kv = min(_log(rng, 1, 4096), max(1, 2 ** 19 // (seqs * hkv)))
        return _batch(kind, seqs, max(1, kv // 8), kv, max(1, kv // 8), kv, hq, hkv, d, page, dtype)
    kv = _log(rng, 32, 16384)
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 1024)
    new = min(new, kv, max(1, 2 ** 31 // (seqs * hq * kv * 8)))  # the plain form's scores
    kv = min(kv, max(new, 2 ** 20 // (seqs * hkv)))
    return _batch(kind, seqs, new // 3 if seqs > 1 else new, new, max(new, kv // 8), kv, hq, hkv, d, page,
                  dtype, pad=rng.choice([0, 0, 5]))


def _lengths(case):
    """(new tokens, cached tokens with them) of every sequence."""
    r = random.Random(",".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    new[r.randrange(len(new))] = case["new_hi"]
    if case["kind"] == "read":
        return new, list(new)
    kv = [max(n, r.randint(case["kv_lo"], case["kv"])) for n in new]
    if case["kind"] == "attend":
        kv[r.randrange(len(kv))] = case["kv"]
    return new, kv


# ---- the formats ----------------------------------------------------------
def _groups(d):
    g = -(-d // 32)
    return g + (g in (5, 7))


def _wide(x, d):
    """x [..., D] with its columns padded to whole groups."""
    return torch.nn.functional.pad(x, (0, 32 * _groups(d) - d))


def _five_bits(s):
    """s (fp32) rounded to five significant bits, ties to even."""
    u = s.contiguous().view(torch.int32)
    return ((u + 0x3ffff + ((u >> 19) & 1)) & ~0x7ffff).view(torch.float32)


def _quantise(x):
    """x [..., 32 G] in fp32: numbers [..., 32 G] (int32) and scales [..., G] (fp16)."""
    g = x.unflatten(-1, (-1, 32))
    top, low = g.amax(-1), g.amin(-1)
    m = torch.where(top >= -low, top, low)
    s = _five_bits(m / -8.0).clamp(-LARGEST, LARGEST).half()
    at = torch.floor(g.double() / s.double()[..., None] + 0.5) + 8.0
    n = torch.where(s[..., None] == 0, torch.full_like(at, 8.0), at.clamp(0.0, 15.0))
    return n.to(torch.int32).flatten(-2), s


def _words(n):
    """Numbers [..., 8 x] as 32-bit words [..., x]."""
    n = n.unflatten(-1, (-1, 4, 2)).long()
    shift = torch.arange(4, device=n.device) * 4
    w = ((n[..., 0] << shift) | (n[..., 1] << (shift + 16))).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _numbers(w):
    """_words back: [..., x] to [..., 8 x], as fp32 of n - 8."""
    shift = torch.arange(4, device=w.device, dtype=torch.int32) * 4
    lo, hi = (w[..., None] >> shift) & 15, (w[..., None] >> (shift + 16)) & 15
    return (torch.stack([lo, hi], -1).flatten(-3) - 8).float()


def _parts(pages, page, g, keys):
    """The words and scales of pages [n, Hkv, bytes] as views: keys [n, Hkv, P, 4, G]
    and [n, Hkv, P, G], values [n, Hkv, P / 4, 4 G, 4] and [n, Hkv, P / 4, G, 4]."""
    words = pages[..., :16 * g * page].view(torch.int32)
    scales = pages[..., 16 * g * page:].view(torch.float16)
    if keys:
        return words.unflatten(-1, (page, 4, g)), scales.unflatten(-1, (page, g))
    return words.unflatten(-1, (page // 4, 4 * g, 4)), scales.unflatten(-1, (page // 4, g, 4))


def _held(pages, page, d, keys):
    """What pages [n, Hkv, bytes] stand for: [n, Hkv, P, D] in fp32."""
    g = _groups(d)
    words, scales = _parts(pages, page, g, keys)
    if keys:
        n = _numbers(words.transpose(-1, -2))
    else:
        n = _numbers(words.movedim(-1, -2).flatten(-3, -2))
        scales = scales.movedim(-1, -2).flatten(-3, -2)
    n = n.reshape(*scales.shape, 32)
    return (n * scales.float()[..., None]).flatten(-2)[..., :d]


def _store(s, side, page, row, x):
    """x [T, Hkv, D] (fp32) to rows of pages, in 4 bits."""
    d, g = x.shape[-1], _groups(x.shape[-1])
    n, scale = _quantise(_wide(x, d))
    words, scales = _parts(s[side + "_pages"], s["case"]["page"], g, side == "k")
    if side == "k":
        words[page, :, row] = _words(n).unflatten(-1, (g, 4)).transpose(-1, -2)
        scales[page, :, row] = scale
    else:
        words[page, :, row // 4, :, row % 4] = _words(n)
        scales[page, :, row // 4, :, row % 4] = scale


def _packed(n, scales, mins, group):
    """Weights' numbers [out, in] (int), scales and mins [out, in / group] as bytes."""
    rows, cols = n.shape
    n = torch.nn.functional.pad(n, (0, -cols % 128, 0, -rows % 16), value=8)
    w = _words(n).unflatten(1, (-1, 4, 4)).unflatten(0, (-1, 16))  # [tiles, 16, blocks, i, c]
    found = [w.permute(0, 2, 4, 1, 3).reshape(-1).view(torch.uint8)]
    for t in (scales, mins):
        if t is not None:
            t = torch.nn.functional.pad(t, (0, n.shape[1] // group - t.shape[1], 0, -rows % 16))
            t = t.unflatten(1, (-1, 128 // group)).unflatten(0, (-1, 16)).transpose(1, 2)
            found.append(t.reshape(-1).view(torch.uint8))
    return torch.cat(found)


def _weights(packed, rows, cols, group, mins):
    """_packed back, as [out, in] in fp32."""
    tiles, blocks = -(-rows // 16), -(-cols // 128)
    size, groups = tiles * blocks * 1024, blocks * 128 // group
    n = _numbers(packed[:size].view(torch.int32).view(tiles, blocks, 4, 16, 4).permute(0, 3, 1, 4, 2))
    n = n.reshape(tiles * 16, groups, group)
    rest = packed[size:].view(torch.float16).view(-1, tiles, blocks, 16, 128 // group)
    rest = rest.transpose(2, 3).reshape(-1, tiles * 16, groups)
    w = n * rest[0].float()[..., None]
    if mins:
        w += rest[1].float()[..., None]
    return w.flatten(1)[:rows, :cols]


# ---- what a program has in hand -------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    s = {"case": case}
    if case["kind"] == "project":
        t, cols, group, rank = case["tokens"], case["width"], case["group"], case["rank"]
        s["x"], s["projs"] = normal(t, cols), []
        for rows in map(int, case["outs"].split(",")):
            n = torch.round(normal(rows, cols, scale=2.8, dtype=torch.float32)).clamp(-8, 7).to(torch.int32) + 8
            scales = (0.02 * (0.5 + torch.rand(rows, cols // group, device="cuda", generator=g))).half()
            mins = normal(rows, cols // group, scale=0.01, dtype=torch.float16) if case["mins"] else None
            p = {"w": _packed(n, scales, mins, group), "out": rows}
            if case["bias"]:
                p["bias"] = normal(rows, scale=0.5, dtype=torch.float32)
            if rank:
                p["a"] = normal(cols, rank, scale=cols ** -0.5, dtype=torch.float32)
                p["b"] = normal(rank, rows, scale=0.5, dtype=torch.float32)
                p["scaling"] = 2.0
            s["projs"].append(p)
        return s
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    new, kv = _lengths(case)
    tokens, page, groups = sum(new) + case["pad"], case["page"], _groups(d)
    pages = [-(-n // page) for n in kv]
    widest = -(-case["kv"] // page)
    order = torch.randperm(sum(pages), device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(kv), widest), -1, device="cuda", dtype=torch.int32)
    held = torch.arange(widest, device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    table[held] = order
    s["page_table"], s["tokens"] = table, tokens
    s["kv_lens"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
    s["cu_tokens"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    places = torch.arange(sum(pages) * page, device="cuda")
    for side in "kv":
        s[side + "_pages"] = torch.empty(sum(pages), hkv, 18 * groups * page, device="cuda", dtype=torch.uint8)
        _store(s, side, places // page, places % page, normal(len(places), hkv, d).float())
    if case["kind"] == "append":
        s["q"], s["k"], s["v"] = normal(tokens, hq, d), normal(tokens, hkv, d), normal(tokens, hkv, d)
    if case["kind"] == "attend":
        s["q"] = normal(tokens, hq, d)
        s["out"] = torch.full_like(s["q"], 0.5)
        s["lse"] = torch.full((hq, tokens), 0.5, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------
def _turn(x, positions, theta):
    """x [T, H, D] rotated by its positions, pairs (i, i + D / 2), in 64 bits: where a
    quantised value lies between two numbers decides which one is held."""
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                                                    -2.0 * i / x.shape[-1])[None, :]
    c, s = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _places(s, tokens):
    """Of every row: its sequence, its place among that one's new tokens, its
    position, and whether a sequence has it."""
    cu, t = s["cu_tokens"].long(), torch.arange(tokens, device="cuda")
    seq = (cu[None, 1:] <= t[:, None]).sum(1)
    live = seq < len(cu) - 1
    seq = seq.clamp(max=len(cu) - 2)
    at = t - cu[seq]
    return seq, at, s["kv_lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + at, live


def _plain_read(s, page, row):
    """Rows of pages as the program's type: keys and values [T, Hkv, D]."""
    case, found = s["case"], []
    dt, d, g = DTYPES[case["dtype"]], case["head_dim"], _groups(case["head_dim"])
    kw, ks = _parts(s["k_pages"], case["page"], g, True)
    vw, vs = _parts(s["v_pages"], case["page"], g, False)
    for n, scale in ((_numbers(kw[page, :, row].transpose(-1, -2)), ks[page, :, row]),
                     (_numbers(vw[page, :, row // 4, :, row % 4]), vs[page, :, row // 4, :, row % 4])):
        n = n.reshape(*scale.shape, 32)
        found.append((n * scale.float()[..., None]).flatten(-2)[..., :d].to(dt))
    return found


def _plain_append(s):
    case = s["case"]
    seq, _, pos, _ = _places(s, s["tokens"])
    page, row = s["page_table"][seq, pos // case["page"]].long(), pos % case["page"]
    _store(s, "k", page, row, _turn(s["k"], pos, case["theta"]).float())
    _store(s, "v", page, row, s["v"].float())
    return (_turn(s["q"], pos, case["theta"]).to(s["q"].dtype), *_plain_read(s, page, row))


def _plain_attend(s):
    case = s["case"]
    hq, hkv, d, dt = case["heads_q"], case["heads_kv"], case["head_dim"], s["q"].dtype
    group, tokens = hq // hkv, s["q"].shape[0]
    table = s["page_table"].long().clamp(min=0)
    seqs, keys, most = table.shape[0], table.shape[1] * case["page"], case["new_hi"]
    # [seqs, kv heads, keys, D]
    k, v = (_held(s[side + "_pages"], case["page"], d, side == "k")[table].permute(0, 2, 1, 3, 4).reshape(seqs, hkv, keys, d)
            for side in "kv")
    seq, at, pos, live = _places(s, tokens)
    cu = s["cu_tokens"].long()
    rows = (cu[:-1, None] + torch.arange(most, device="cuda")).clamp(max=tokens - 1)
    q = s["q"][rows].float().reshape(seqs, most, hkv, group, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, hkv, group * most, d), k.transpose(2, 3).contiguous())
    score = score.mul_(1.0 / math.sqrt(d)).view(seqs, hkv, group, most, keys)
    last = (s["kv_lens"].long() - (cu[1:] - cu[:-1]))[:, None] + torch.arange(most, device="cuda")
    seen = torch.arange(keys, device="cuda") <= last[..., None]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, hkv, group * most, keys), v).view(seqs, hkv, group, most, d) / total
    lse = (top + total.log())[..., 0]  # [seqs, kv heads, group, most]
    at = at.clamp(max=most - 1)
    out = out[seq, :, :, at].reshape(tokens, hq, d).to(dt)
    lse = lse[seq, :, :, at].reshape(tokens, hq)
    return (torch.where(live[:, None, None], out, s["out"]),
            torch.where(live[None, :], lse.t(), s["lse"]))


def _plain_project(x, p, case):
    y = x.float() @ _weights(p["w"], p["out"], case["width"], case["group"], case["mins"]).t()
    if case["rank"]:
        y += p["scaling"] * (x.float() @ p["a"]) @ p["b"]
    if case["bias"]:
        y += p["bias"]
    return y.to(x.dtype)


def run(s):
    case = s["case"]
    if own:
        eng = _lib()
        if case["kind"] == "project":
            return eng.proj_quant_forward(s["x"], [dict(p) for p in s["projs"]], rank=case["rank"],
                                          group=case["group"], mins=case["mins"])
        index = (s["k_pages"], s["v_pages"], s["cu_tokens"], s["kv_lens"], s["page_table"])
        if case["kind"] == "attend":
            return eng.qcache_forward(s["q"], *index, max_new=case["new_hi"], max_kv=case["kv"],
                                      out=s["out"], lse=s["lse"])
        found = ()
        if case["kind"] == "append":
            found = (eng.qcache_append(s["k"], s["v"], *index, rope_freq_base=case["theta"], q=s["q"]),)
        return (*found, *eng.qcache_read(*index, s["tokens"], case["head_dim"], DTYPES[case["dtype"]]))
    if case["kind"] == "project":
        return [_plain_project(s["x"], p, case) for p in s["projs"]]
    if case["kind"] == "attend":
        return _plain_attend(s)
    if case["kind"] == "append":
        return _plain_append(s)
    seq, _, pos, _ = _places(s, s["tokens"])
    return tuple(_plain_read(s, s["page_table"][seq, pos // case["page"]].long(), pos % case["page"]))


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "project":
        t, cols, outs = case["tokens"], case["width"], list(map(int, case["outs"].split(",")))
        held = cols / 2 + (4 if case["mins"] else 2) * cols / case["group"]
        adapters = 4 * case["rank"] * (cols * len(outs) + sum(outs))
        return {"bytes": sum(outs) * held + adapters + size * t * (cols + sum(outs)),
                "flops": 2 * t * cols * sum(outs) + 2 * t * case["rank"] * (cols * len(outs) + sum(outs))}
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    new, kv = _lengths(case)
    held = d / 2 + 2 * -(-d // 32)  # bytes of a token's head
    if case["kind"] == "append":  # written, and read back
        return {"bytes": sum(new) * (2 * hq * d * size + 2 * hkv * (2 * d * size + 2 * held)),
                "flops": sum(new) * d * (6 * hq + 14 * hkv)}
    if case["kind"] == "read":
        return {"bytes": 2 * sum(new) * hkv * (held + d * size), "flops": 2 * sum(new) * hkv * d}
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, kv))
    read = sum(c for n, c in zip(new, kv) if n)
    return {"bytes": 2 * sum(new) * hq * d * size + 2 * read * hkv * held + 4 * sum(new) * hq,
            "flops": 4 * d * hq * pairs}


# ---- in 64 bits, from the definitions -------------------------------------
def _nibble(flat, word, column):
    """The number of a column in 32-bit word `word` of flat bytes."""
    bit = column % 8 // 2 * 4 + column % 2 * 16
    return (flat[word * 4 + bit // 8].long() >> (bit % 8)) & 15


def _half(flat, at):
    """The fp16 number `at` of flat bytes."""
    return torch.stack([flat[2 * at], flat[2 * at + 1]], -1).view(torch.float16)[..., 0].double()


def _sequence(case, s, side, pages, tokens):
    """The first `tokens` tokens of the sequence with these pages: [Hkv, tokens, D]."""
    g, p, hkv = _groups(case["head_dim"]), case["page"], case["heads_kv"]
    got, rows = s[side + "_pages"][pages], torch.arange(p, device="cuda")
    # a page's head's rows, for all pages and heads at once: bytes along the first axis
    flat = got.flatten(0, 1).t()
    col = torch.arange(case["head_dim"], device="cuda")
    i, r, scales = col // 32, col // 8, flat[16 * g * p:]
    row = rows[:, None]
    if side == "k":
        word, at = (row * 4 + r % 4) * g + i, row * g + i
    else:
        word, at = (row // 4 * 4 * g + r) * 4 + row % 4, (row // 4 * g + i) * 4 + row % 4
    bit = (col % 8 // 2 * 4 + col % 2 * 16).expand_as(word)
    n = (flat[word * 4 + bit // 8].long() >> (bit % 8)[..., None]) & 15
    scale = torch.stack([scales[2 * at], scales[2 * at + 1]], -1).view(torch.float16)[..., 0].double()
    x = (n - 8).double() * scale  # [P, D, pages heads]
    return x.unflatten(2, (-1, hkv)).permute(3, 2, 0, 1).flatten(1, 2)[:, :tokens]


def _rounded(x):
    """x [..., 32] (64 bits) as a group of the cache stands for it."""
    at = x.abs().argmax(-1, keepdim=True)
    most = x.abs().amax(-1, keepdim=True)
    step = torch.where((x == most).any(-1, keepdim=True), most, x.gather(-1, at)) / -8.0
    unit = torch.exp2(torch.floor(torch.log2(step.abs())) - 4)
    step = (torch.round(step / unit) * unit).clamp(-LARGEST, LARGEST)
    return torch.nan_to_num(torch.floor(x / step + 0.5).clamp(-8, 7) * step)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "project":
        x, found = s["x"].double(), []
        blocks, group = -(-case["width"] // 128), case["group"]
        col = torch.arange(case["width"], device="cuda")
        for p in s["projs"]:
            y = torch.empty(x.shape[0], p["out"], device="cuda", dtype=torch.float64)
            tiles = -(-p["out"] // 16)
            for r0 in range(0, p["out"], 2048):
                row = torch.arange(r0, min(p["out"], r0 + 2048), device="cuda")[:, None]
                word = (((row // 16) * blocks + col // 128) * 64 + col % 32 // 8 * 16 + row % 16) * 4 + col % 128 // 32
                at = (((row // 16) * blocks + col // 128) * 16 + row % 16) * (128 // group) + col % 128 // group
                scales = p["w"][tiles * blocks * 1024:]
                w = (_nibble(p["w"], word, col) - 8).double() * _half(scales, at)
                if case["mins"]:
                    w += _half(scales[tiles * blocks * 4096 // group:], at)
                y[:, r0:r0 + 2048] = x @ w.t()
            if case["rank"]:
                y += p["scaling"] * ((x @ p["a"].double()) @ p["b"].double())
            found.append(y + p["bias"].double() if case["bias"] else y)
        return found
    new, kv = _lengths(case)
    starts = [sum(new[:b]) for b in range(len(new))]
    page, table, d = case["page"], s["page_table"].cpu(), case["head_dim"]
    if case["kind"] == "append":
        spot = torch.cat([torch.arange(c - n, c) for n, c in zip(new, kv)]).cuda()
        j = torch.arange(d // 2, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64),
                           spot.double().view(-1, 1, 1) * torch.exp(-2.0 * j / d * math.log(case["theta"])))
        found = []
        for x in (s["q"], s["k"]):
            z = torch.complex(x[..., :d // 2].double(), x[..., d // 2:].double()) * turn
            found.append(torch.cat([z.real, z.imag], -1))
        kept = [_rounded(_wide(x, d).unflatten(-1, (-1, 32))).flatten(-2)[..., :d]
                for x in (found[1].float().double(), s["v"].double())]
        return (found[0], *kept)
    whole = [[_sequence(case, s, side, table[b, :-(-c // page)].long().cuda(), c) for side in "kv"]
             for b, c in enumerate(kv)] if case["kind"] == "read" else []
    if whole:
        return tuple(torch.cat([w[x].transpose(0, 1) for w in whole]) for x in (0, 1))
    hq, group = case["heads_q"], case["heads_q"] // case["heads_kv"]
    out, lse = s["out"].double(), s["lse"].double()
    for b, (n, c) in enumerate(zip(new, kv)):
        if n == 0:
            continue
        k, v = (_sequence(case, s, side, table[b, :-(-c // page)].long().cuda(), c) for side in "kv")
        rows = slice(starts[b], starts[b] + n)
        hidden = torch.ones(n, c, device="cuda", dtype=torch.bool).triu(c - n + 1)
        for h in range(hq):
            z = (s["q"][rows, h].double() @ k[h // group].t() / math.sqrt(d)).masked_fill(hidden, -math.inf)
            lse[h, rows] = torch.logsumexp(z, -1)
            out[rows, h] = torch.softmax(z, -1) @ v[h // group]
    return out, lse
