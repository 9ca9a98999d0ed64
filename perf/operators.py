"""The operators that a decoder runs between its q/k/v projections and its O
projection when it answers, as measurable cases:

  qknorm  per-head RMS norms of the queries and keys with the position rotation
          in the same pass, forward, or backward with both weights' gradients
  append  new keys and values into a paged cache, keys and queries rotated on
          the way
  attend  attention of each sequence's new tokens over its cached keys

A case is a dict of plain values.  The lengths of a batch are drawn from the
case's own values, so that every seed of a case does the same work.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1.0e-6
_engine = None


def _lib():
    """The framework's engine (own only)."""
    global _engine
    if _engine is None:
        sys.path.insert(0, os.path.abspath("glacier.tune_amd"))
        import glacier_attn as ga

        _engine = ga.GpuAttentionEngine(torch.cuda.current_device(), ga.PREC_BF16)
    return _engine


def _qknorm(tokens, heads_q, heads_kv, head_dim, dtype="bf16", grad=False, theta=1.0e6, far=4096):
    """far: positions lie below it."""
    return {"kind": "qknorm", "tokens": tokens, "heads_q": heads_q, "heads_kv": heads_kv,
            "head_dim": head_dim, "dtype": dtype, "grad": grad, "theta": theta, "far": far}


def _append(seqs, new_lo, new_hi, kv, heads_q, heads_kv, head_dim, page, dtype="bf16",
            theta=1.0e6):
    """seqs sequences of new_lo .. new_hi new tokens, at most kv tokens each afterwards."""
    return {"kind": "append", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "kv": kv,
            "heads_q": heads_q, "heads_kv": heads_kv, "head_dim": head_dim, "page": page,
            "dtype": dtype, "theta": theta, "pad": 0}


def _attend(seqs, new_lo, new_hi, kv_lo, kv, heads_q, heads_kv, head_dim, page, dtype="bf16",
            pad=0):
    """As append, of kv_lo .. kv tokens a sequence; pad: rows behind the last sequence."""
    return {"kind": "attend", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "kv_lo": kv_lo,
            "kv": kv, "heads_q": heads_q, "heads_kv": heads_kv, "head_dim": head_dim,
            "page": page, "dtype": dtype, "pad": pad}


def listed():
    named = {
        # one token of each of a few answers: what counts is the call itself
        "qknorm_tokens_8": _qknorm(8, 28, 4, 128),
        # a prompt of ordinary length
        "qknorm_prompt_4096": _qknorm(4096, 32, 8, 128, theta=5.0e5),
        # a training batch's backward pass, weights' gradients among it
        "qknorm_grad_4096": _qknorm(4096, 28, 4, 128, grad=True),
        # the same on few tokens of a small model, in the fp32 mode that results are checked in
        "qknorm_grad_333_fp32": _qknorm(333, 14, 2, 64, dtype="fp32", grad=True, far=70000),
        # a step of 64 answers at once
        "append_tokens_64": _append(64, 1, 1, 1024, 28, 4, 128, 16),
        # a packed batch of prompts of ragged lengths
        "append_prompts_16": _append(16, 64, 512, 512, 32, 8, 128, 64, theta=5.0e5),
        # the first words of a single short answer
        "attend_token_512": _attend(1, 1, 1, 512, 512, 14, 2, 64, 16),
        # a serving step: 32 answers, contexts short to long
        "attend_tokens_32": _attend(32, 1, 1, 64, 8192, 28, 4, 128, 16),
        # one answer over a document
        "attend_token_65536": _attend(1, 1, 1, 65536, 65536, 32, 8, 128, 64),
        # a long prompt's chunk over what is cached of it already
        "attend_chunk_2048": _attend(1, 2048, 2048, 8192, 8192, 28, 4, 128, 64),
        # prompts' chunks of ragged lengths, some idle sequences, a padded batch
        "attend_chunks_8": _attend(8, 0, 256, 300, 4096, 32, 8, 128, 16, pad=19),
        # the checking mode on a head size between the usual ones
        "attend_chunks_3_fp32": _attend(3, 17, 120, 200, 1001, 8, 2, 96, 32, dtype="fp32"),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qknorm", "append", "attend", "attend"])
    hq, hkv, d = rng.choice([(28, 4, 128), (32, 8, 128), (14, 2, 64), (12, 2, 128), (8, 8, 64),
                             (8, 2, 96), (5, 1, 80), (8, 2, 256), (16, 4, 32), (40, 8, 128)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    theta = rng.choice([1.0e4, 5.0e5, 1.0e6])
    if kind == "qknorm":
        return _qknorm(_log(rng, 1, 8192), hq, hkv, d, dtype, rng.random() < 0.5, theta,
                       _log(rng, 512, 131072))
    page = rng.choice([16, 32, 64, 128])
    seqs = _log(rng, 1, 64)
    if kind == "append":
        new = _log(rng, 1, 512)
        return _append(seqs, max(1, new // 4), new, new + _log(rng, 1, 512), hq, hkv, d, page,
                       dtype, theta)
    kv = _log(rng, 32, 16384)
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 1024)
    new = min(new, kv, max(1, 2 ** 31 // (seqs * hq * kv * 8)))  # the plain form's scores
    kv = min(kv, max(new, 2 ** 26 // (seqs * hkv)))
    return _attend(seqs, new // 3 if seqs > 1 else new, new, max(new, kv // 8), kv, hq, hkv, d,
                   page, dtype, rng.choice([0, 0, 5]))


def _lengths(case):
    """(new tokens, cached tokens afterwards) of every sequence."""
    r = random.Random(",".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    new[r.randrange(len(new))] = case["new_hi"]
    if case["kind"] == "append":
        return new, [r.randint(n, case["kv"]) for n in new]
    kv = [max(n, r.randint(case["kv_lo"], case["kv"])) for n in new]
    kv[r.randrange(len(kv))] = case["kv"]
    return new, kv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)

    s = {"case": case}
    if case["kind"] == "qknorm":
        t = case["tokens"]
        s["q"], s["k"] = normal(t, hq, d, scale=2.0), normal(t, hkv, d, scale=2.0)
        for w in ("q_weight", "k_weight"):
            s[w] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
        s["positions"] = torch.randint(0, case["far"], (t,), device="cuda", generator=g,
                                       dtype=torch.int32)
        if case["grad"]:
            s["dq_out"], s["dk_out"] = normal(t, hq, d, scale=0.1), normal(t, hkv, d, scale=0.1)
        return s
    new, kv = _lengths(case)
    tokens, page = sum(new) + case["pad"], case["page"]
    pages = [-(-n // page) for n in kv]
    widest = -(-case["kv"] // page)
    order = torch.randperm(sum(pages), device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(kv), widest), -1, device="cuda", dtype=torch.int32)
    held = torch.arange(widest, device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    table[held] = order
    s["page_table"] = table
    s["kv_lens"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
    s["cu_tokens"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["k_pages"] = normal(sum(pages), hkv, page, d)
    s["v_pages"] = normal(sum(pages), hkv, page, d)
    s["q"] = normal(tokens, hq, d)
    if case["kind"] == "append":
        s["k"], s["v"] = normal(tokens, hkv, d), normal(tokens, hkv, d)
    else:
        s["out"] = torch.full_like(s["q"], 0.5)
        s["lse"] = torch.full((hq, tokens), 0.5, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------
def _turn(x, positions, theta, sign):
    """x [T, H, D] rotated by sign * its position: pairs (i, i + D / 2)."""
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                                                    -2.0 * i / x.shape[-1])[None, :]
    c, s = torch.cos(angle).float()[:, None, :], sign * torch.sin(angle).float()[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _norm_turn(x, w, positions, theta):
    f = x.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    return _turn(f * r * w, positions, theta, 1.0).to(x.dtype)


def _norm_turn_grad(dy, x, w, positions, theta):
    f, g = x.float(), _turn(dy.float(), positions, theta, -1.0)
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    wg = w * g
    dx = r * wg - r ** 3 * f * (wg * f).mean(-1, keepdim=True)
    return dx.to(x.dtype), (g * f * r).sum((0, 1))


def _places(s, tokens):
    """Of every row of q: its sequence, its place among that one's new tokens,
    its position, and whether a sequence has it."""
    cu, t = s["cu_tokens"].long(), torch.arange(tokens, device="cuda")
    seq = (cu[None, 1:] <= t[:, None]).sum(1)
    live = seq < len(cu) - 1
    seq = seq.clamp(max=len(cu) - 2)
    at = t - cu[seq]
    return seq, at, s["kv_lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + at, live


def _plain_append(s):
    case = s["case"]
    seq, _, pos, _ = _places(s, s["q"].shape[0])
    page = s["page_table"][seq, pos // case["page"]].long()
    s["k_pages"][page, :, pos % case["page"]] = _turn(s["k"].float(), pos, case["theta"], 1.0).to(s["k"].dtype)
    s["v_pages"][page, :, pos % case["page"]] = s["v"]
    return _turn(s["q"].float(), pos, case["theta"], 1.0).to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _plain_attend(s):
    case = s["case"]
    hq, hkv, d, dt = case["heads_q"], case["heads_kv"], case["head_dim"], s["q"].dtype
    group, tokens = hq // hkv, s["q"].shape[0]
    table = s["page_table"].long().clamp(min=0)
    seqs, keys, most = table.shape[0], table.shape[1] * case["page"], case["new_hi"]
    # [seqs, kv heads, keys, D]
    k, v = (x[table].permute(0, 2, 1, 3, 4).reshape(seqs, hkv, keys, d).float()
            for x in (s["k_pages"], s["v_pages"]))
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


def run(s):
    case = s["case"]
    if own:
        eng = _lib()
        if case["kind"] == "append":
            q_rot = eng.cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["cu_tokens"],
                                     s["kv_lens"], s["page_table"], rope_freq_base=case["theta"],
                                     q=s["q"])
            return q_rot, s["k_pages"], s["v_pages"]
        if case["kind"] == "attend":
            return eng.cache_forward(s["q"], s["k_pages"], s["v_pages"], s["cu_tokens"],
                                     s["kv_lens"], s["page_table"], max_new=case["new_hi"],
                                     max_kv=case["kv"], out=s["out"], lse=s["lse"])
        if not case["grad"]:
            return eng.qk_norm_forward(s["q"], s["k"], s["q_weight"], s["k_weight"], EPS,
                                       rope_freq_base=case["theta"], positions=s["positions"])
        dwq, dwk = torch.zeros_like(s["q_weight"]), torch.zeros_like(s["k_weight"])
        dq, dk = eng.qk_norm_backward(s["dq_out"], s["dk_out"], s["q"], s["k"], s["q_weight"],
                                      s["k_weight"], EPS, rope_freq_base=case["theta"],
                                      positions=s["positions"], dq_weight=dwq, dk_weight=dwk)
        return dq, dk, dwq, dwk
    if case["kind"] == "append":
        return _plain_append(s)
    if case["kind"] == "attend":
        return _plain_attend(s)
    if not case["grad"]:
        return (_norm_turn(s["q"], s["q_weight"], s["positions"], case["theta"]),
                _norm_turn(s["k"], s["k_weight"], s["positions"], case["theta"]))
    dq, dwq = _norm_turn_grad(s["dq_out"], s["q"], s["q_weight"], s["positions"], case["theta"])
    dk, dwk = _norm_turn_grad(s["dk_out"], s["k"], s["k_weight"], s["positions"], case["theta"])
    return dq, dk, dwq, dwk


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    if case["kind"] == "qknorm":
        t = case["tokens"]
        return {"bytes": (3 if case["grad"] else 2) * t * (hq + hkv) * d * size + 4 * t,
                "flops": (20 if case["grad"] else 8) * t * (hq + hkv) * d}
    new, kv = _lengths(case)
    if case["kind"] == "append":
        return {"bytes": 2 * sum(new) * (hq + 2 * hkv) * d * size,
                "flops": 3 * sum(new) * (hq + hkv) * d}
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, kv))
    read = sum(c for n, c in zip(new, kv) if n)
    return {"bytes": 2 * sum(new) * hq * d * size + 2 * read * hkv * d * size + 4 * sum(new) * hq,
            "flops": 4 * d * hq * pairs}


# ---- in 64 bits, from the definitions -------------------------------------
def _rotation(positions, theta, d):
    """[T, D, D]'s action as complex numbers: e^{i pos theta^(-2j/D)}, j < D / 2."""
    j = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    return torch.polar(torch.ones(1, device="cuda", dtype=torch.float64),
                       positions.double().view(-1, 1, 1) * torch.exp(-2.0 * j / d * math.log(theta)))


def _pairs(x):
    half = x.shape[-1] // 2
    return torch.complex(x[..., :half].double(), x[..., half:].double())


def _flat(z):
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "qknorm":
        turn, d, got = _rotation(s["positions"], case["theta"], case["head_dim"]), case["head_dim"], []
        for side in "qk":
            x, w = s[side].double(), s[side + "_weight"].double()
            size = (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
            if not case["grad"]:
                got.append(_flat(_pairs(x / size * w) * turn))
                continue
            g = _flat(_pairs(s[f"d{side}_out"]) * turn.conj())
            unit = x / size
            gw = g * w
            got.append((gw - unit * (gw * unit).sum(-1, keepdim=True) / d) / size)
            got.append((g * unit).flatten(0, 1).sum(0))
        return tuple(got) if not case["grad"] else (got[0], got[2], got[1], got[3])
    new, kv = _lengths(case)
    starts = [sum(new[:b]) for b in range(len(new))]
    page, table = case["page"], s["page_table"].cpu()
    if case["kind"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        spot = torch.cat([torch.arange(c - n, c) for n, c in zip(new, kv)])
        turn = _rotation(spot.cuda(), case["theta"], case["head_dim"])
        k, q, v = _flat(_pairs(s["k"]) * turn), _flat(_pairs(s["q"]) * turn), s["v"].double()
        for b, (n, c) in enumerate(zip(new, kv)):
            where = torch.arange(c - n, c)
            to, off = table[b, where // page].long().cuda(), (where % page).cuda()
            kp[to, :, off] = k[starts[b]:starts[b] + n]
            vp[to, :, off] = v[starts[b]:starts[b] + n]
        return q, kp, vp
    hq, hkv = case["heads_q"], case["heads_kv"]
    group = hq // hkv
    out, lse = s["out"].double(), s["lse"].double()
    for b, (n, c) in enumerate(zip(new, kv)):
        if n == 0:
            continue
        of = table[b, :-(-c // page)].long().cuda()
        rows = slice(starts[b], starts[b] + n)
        hidden = torch.ones(n, c, device="cuda", dtype=torch.bool).triu(c - n + 1)
        for h in range(hq):
            kh, vh = (x[of, h // group].reshape(-1, x.shape[-1])[:c].double() for x in (s["k_pages"], s["v_pages"]))
            z = (s["q"][rows, h].double() @ kh.t() / math.sqrt(case["head_dim"])).masked_fill(hidden, -math.inf)
            lse[h, rows] = torch.logsumexp(z, -1)
            out[rows, h] = torch.softmax(z, -1) @ vh
    return out, lse
