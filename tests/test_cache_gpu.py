"""The paged key/value cache (glacier_attn_cache_*), through the Python front
end, against its definition in 64 bits."""
import math
import threading

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


# (new tokens, tokens with them) per sequence; hq, hkv, D, page, rows behind
BATCHES = {
    "one_key": ([(1, 1)], 1, 1, 8, 16, 0),
    "one_token": ([(1, 512)], 14, 2, 64, 16, 0),
    "tokens": ([(1, 17), (1, 1), (1, 300), (1, 64), (1, 65)], 28, 4, 128, 16, 3),
    "idle_among_them": ([(0, 40), (1, 33), (0, 0), (2, 2), (0, 7)], 8, 2, 96, 32, 1),
    "whole_prompt": ([(77, 77)], 8, 8, 64, 64, 0),
    "chunk": ([(50, 190)], 28, 4, 128, 32, 0),
    "ragged_chunks": ([(5, 5), (130, 300), (1, 1000), (64, 64), (0, 10), (33, 97)], 32, 8, 128, 16, 19),
    "odd_head": ([(3, 40), (20, 21)], 5, 1, 80, 128, 2),
    "narrow_head": ([(9, 70), (1, 129)], 16, 4, 32, 16, 0),
    "wide_head": ([(6, 50), (1, 200)], 8, 2, 256, 16, 0),
    "between_heads": ([(4, 90)], 6, 3, 200, 64, 0),
    "many_heads": ([(3, 50)], 40, 1, 64, 16, 0),
    "long": ([(1, 9000), (2, 300)], 16, 4, 128, 256, 0),
    "long_chunk": ([(40, 5000)], 14, 2, 64, 1024, 0),
    "many_sequences": ([(1, 20 + i % 50) for i in range(150)], 4, 2, 64, 16, 5),
}


# The layout of the work follows from how many keys the page table or max_kv
# allow: a table for 2^17 of them takes 128-row tiles (bf16, heads up to 128) and
# many splits; the lengths themselves, mostly 16-row tiles.
WIDE = 2 ** 17


@pytest.mark.parametrize("columns", [0, WIDE])
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_attention(eng, name, dt, columns):
    seqs, hq, hkv, d, page, pad = BATCHES[name]
    p = ch.Paged(seqs, hq, hkv, d, page, DTYPES[dt], 5, pad, columns=columns // page)
    q = p.q.cuda()
    out = torch.full_like(q, 7.0)
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = ch.attend_ref(p)
    hints = dict(max_new=max(n for n, _ in seqs), max_kv=max(kv for _, kv in seqs))
    few = dict(max_kv=20000)  # fewer splits than for 2^17 keys
    for kw in (hints, few, {}):
        eng.cache_forward(q, *p.arrays(), out=out, lse=lse, **kw)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
    if pad:  # rows behind the last sequence stay as they were
        assert (out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all()
    again, none = eng.cache_forward(q, *p.arrays())
    live = slice(0, p.tokens - pad)
    assert none is None and torch.equal(again[live], out[live])
    eng.cache_forward(q, *p.arrays(), out=q)  # over its own queries
    assert torch.equal(q[live], out[live])


CHUNKS = {  # more than 16 rows a KV head: 128-row tiles where the table is wide
    "d40": ([(30, 31), (129, 500), (0, 90)], 8, 2, 40, 16, 4),
    "d64": ([(200, 900), (1, 3), (64, 64)], 14, 2, 64, 32, 0),
    "d72": ([(65, 700)], 6, 2, 72, 64, 1),
    "d8": ([(70, 200), (33, 40)], 8, 1, 8, 16, 0),
    "d128_one_head_groups": ([(128, 128), (129, 130), (127, 1000)], 4, 4, 128, 16, 7),
    "d128_group_of_40": ([(9, 3000), (5, 5)], 40, 1, 128, 128, 0),
    "d128_many": ([(3 + i, 40 + 13 * i) for i in range(70)], 16, 2, 128, 16, 2),
    "d256": ([(60, 61), (129, 700), (1, 90)], 8, 2, 256, 16, 3),
    "d136": ([(50, 900)], 6, 3, 136, 32, 0),
    "d248_group_of_16": ([(17, 400), (40, 41)], 16, 1, 248, 64, 0),
    "d120_long": ([(20, 6000)], 10, 2, 120, 512, 0),
    "d64_group_of_130": ([(3, 700), (1, 40)], 130, 1, 64, 16, 2),  # a token's heads in two tiles
}


@pytest.mark.parametrize("keys", [512, 1500, 3000, 9000, WIDE])
@pytest.mark.parametrize("name", sorted(CHUNKS))
def test_chunks_in_every_layout(eng, name, keys):
    # max_kv only lays the work out: few or many splits, narrow or wide tiles
    seqs, hq, hkv, d, page, pad = CHUNKS[name]
    p = ch.Paged(seqs, hq, hkv, d, page, torch.bfloat16, 15, pad, columns=WIDE // page)
    out = torch.full((p.tokens, hq, d), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = ch.attend_ref(p)
    eng.cache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, out=out, lse=lse)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    assert not pad or ((out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all())


@pytest.mark.parametrize("keys", [800, 1500, WIDE])
@pytest.mark.parametrize("name", sorted(CHUNKS))
def test_fp32_chunks_in_every_layout(eng, name, keys):
    # tiles of 16 and of 32 rows, whole and in splits, in order and longest first
    seqs, hq, hkv, d, page, pad = CHUNKS[name]
    p = ch.Paged(seqs, hq, hkv, d, page, torch.float32, 16, pad, columns=WIDE // page)
    out = torch.full((p.tokens, hq, d), 7.0, device="cuda")
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = ch.attend_ref(p)
    eng.cache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, out=out, lse=lse)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    assert not pad or ((out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all())


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_wrong_hints_change_nothing_but_the_layout(eng, dt):
    p = ch.Paged([(70, 400), (1, 2500)], 8, 2, 128, 16, DTYPES[dt], 6)
    ref = ch.attend_ref(p)
    for kw in (dict(max_new=1, max_kv=1), dict(max_new=70, max_kv=300), dict(max_new=10 ** 6, max_kv=10 ** 9)):
        out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), save=True, **kw)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_rows_without_a_key(eng, dt, columns):
    # a length below the number of new tokens leaves the first rows at negative
    # positions: they see nothing, get 0 and -inf, and append nothing
    p = ch.Paged([(6, 9), (3, 3)], 16, 2, 64, 16, DTYPES[dt], 7, columns=columns)
    p.kv_lens[1] = 1
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), save=True)
    assert not out[6:8].any() and (lse[:, 6:8] == -math.inf).all()
    q = ch.Paged([(6, 9), (3, 3)], 16, 2, 64, 16, DTYPES[dt], 7)
    q.seqs = [(6, 9), (1, 1)]
    q.q = torch.cat([p.q[:6], p.q[8:9]])
    q.tokens = 7
    q.k[1], q.v[1] = q.k[1][:1], q.v[1][:1]
    ref = ch.attend_ref(q)
    ch.check("out", torch.cat([out[:6], out[8:]]), ref[0], ref[1])
    ch.check("lse", torch.cat([lse[:, :6], lse[:, 8:]], 1), ref[2], ref[3])
    before = p.both.clone()
    k = torch.ones(9, 2, 64, device="cuda", dtype=DTYPES[dt])
    eng.cache_append(k, 2 * k, *p.arrays())
    same = torch.eq(before, p.both) | (before.isnan() & p.both.isnan())
    changed = (~same).any(-1).nonzero()  # page, k or v, head, row
    last = int(p.table[1, 0])
    assert {(int(r[0]), int(r[3])) for r in changed} == \
        {(int(p.table[0, 0]), i) for i in range(3, 9)} | {(last, 0)}


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_bad_pages_hold_no_keys(eng, dt, columns):
    p = ch.Paged([(4, 150), (1, 64), (1, 5)], 16, 2, 64, 16, DTYPES[dt], 8, columns=columns)
    bad = {(0, 2): -1, (0, 9): p.n_pages, (1, 0): 2 ** 31 - 1, (2, 0): -2 ** 31}
    hidden = [(b, i) for (b, pg) in bad for i in range(16 * pg, min(16 * pg + 16, p.seqs[b][1]))]
    for (b, pg), to in bad.items():
        p.table[b, pg] = to
    ref = ch.attend_ref(p, hidden)
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), save=True)
    assert (lse[:, 5] == -math.inf).all() and not out[5].any()
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    before = p.both.clone()
    k = torch.ones(6, 2, 64, device="cuda", dtype=DTYPES[dt])
    eng.cache_append(k, k, *p.arrays())  # sequences 0 and 2 end in a bad page
    same = torch.eq(before, p.both) | (before.isnan() & p.both.isnan())
    changed = {(int(r[0]), int(r[3])) for r in (~same).any(-1).nonzero()}
    assert changed == {(int(p.table[1, 3]), 15)}


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("hq,d", [(8, 64), (16, 128), (4, 96), (6, 256)])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_not_finite_keys_reach_only_rows_that_see_them(eng, dt, hq, d, columns):
    # NaN and infinities in K and V of late tokens of a chunk: rows before them are
    # those of the same chunk without them, rows from them on are not finite
    seqs, bad = [(90, 130), (20, 20), (1, 70)], {0: (100, 117), 1: (9, 9)}
    p = ch.Paged(seqs, hq, 2, d, 16, DTYPES[dt], 16, columns=columns)
    ref = ch.attend_ref(p)
    for what in (math.nan, math.inf, -math.inf):
        for side in (0, 1):
            both = p.both.clone()
            for b, (first, last) in bad.items():
                for pos in (first, last):
                    both[p.table[b, pos // 16], side, :, pos % 16, 3::7] = what
            arrays = (both[:, 0], both[:, 1], p.cu, p.kv_lens, p.table)
            out, lse = eng.cache_forward(p.q.cuda(), *arrays, save=True)
            clean = torch.ones(p.tokens, dtype=torch.bool)
            clean[100 - 40:90] = False  # positions 100 .. 129 of the first sequence
            clean[90 + 9:90 + 20] = False
            ch.check("out", out[clean.cuda()], ref[0][clean], ref[1][clean])
            ch.check("lse", lse[:, clean.cuda()], ref[2][:, clean], ref[3][:, clean])
            rest = out[~clean.cuda()].float().cpu()
            if side == 1:  # V: its columns, in every row that sees it
                assert not torch.isfinite(rest[..., 3::7]).any()
                others = torch.ones(d, dtype=torch.bool)
                others[3::7] = False
                want, bound = ref[0].clone(), ref[1]
                ch.check("out", rest[..., others], want[~clean][..., others], bound[~clean][..., others])
                if what != what or what > 0:
                    assert (rest[..., 3::7] == what).all() or what != what
            elif what != what:
                assert rest.isnan().all()


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("power", [0, 12, 17, 54])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_scores_far_from_zero(eng, dt, power, columns):
    # q and k times 2^power: but for near ties a row is its best key's value
    seqs, hq, hkv, d = [(40, 300), (3, 900), (1, 50), (60, 60)], 8, 2, 128
    p = ch.Paged(seqs, hq, hkv, d, 16, DTYPES[dt], 21, columns=columns)
    p.k_pages.mul_(2.0 ** power)
    out, lse = eng.cache_forward((p.q * 2.0 ** power).cuda(), *p.arrays(), save=True)
    if power == 0:
        ref = ch.attend_ref(p)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
        return
    at, sure = 0, 0
    for b, (n, kv) in enumerate(seqs):
        for h in range(hq):
            q, k = p.q[at:at + n, h].double() * 2.0 ** power, p.k[b][:, h // (hq // hkv)].double() * 2.0 ** power
            hidden = torch.arange(kv)[None, :] > torch.arange(kv - n, kv)[:, None]
            score = ((q @ k.T) / math.sqrt(d)).masked_fill(hidden, -math.inf)
            # an fp32 sum of d products and its scaling, at their largest
            off = ((q.abs() @ k.abs().T) / math.sqrt(d) * (d + 4) * ch.F).masked_fill(hidden, 0).amax(-1)
            top = torch.cat([score, torch.full((n, 1), -math.inf)], -1).topk(2, -1)
            ok = top.values[:, 0] - top.values[:, 1] > 2 * off + 40
            best = p.v[b][top.indices[:, 0], h // (hq // hkv)].double()
            # the weight's rounding and the result's
            ch.check("out", out[at:at + n, h][ok.cuda()], best[ok],
                     (2 if dt == "bf16" else 4) * ch.half_step(DTYPES[dt]) * best[ok].abs())
            ch.check("lse", lse[h, at:at + n], top.values[:, 0], off + 4 * ch.F * top.values[:, 0].abs() + 40)
            sure += int(ok.sum())
        at += n
    assert sure >= 0.9 * at * hq


def test_lengths_past_the_table(eng):
    # positions the table has no column for hold no key
    p = ch.Paged([(1, 64)], 4, 1, 64, 16, torch.bfloat16, 9)
    table = p.table[:, :2]  # a view: rows further apart than they are long
    ref = ch.attend_ref(p, [(0, j) for j in range(32, 64)])
    out, lse = eng.cache_forward(p.q.cuda(), p.k_pages, p.v_pages, p.cu, p.kv_lens, table, save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    before = p.both.clone()
    k = torch.ones(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    eng.cache_append(k, k, p.k_pages, p.v_pages, p.cu, p.kv_lens, table)
    assert torch.equal(before.nan_to_num(9.0), p.both.nan_to_num(9.0))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_append(eng, name, dt):
    seqs, hq, hkv, d, page, pad = BATCHES[name]
    p = ch.Paged(seqs, hq, hkv, d, page, DTYPES[dt], 11, pad)
    k, v = (torch.randn(p.tokens, hkv, d).to(DTYPES[dt]) for _ in range(2))
    for theta in (None, 5e5):
        q, q_rot = p.q.cuda(), torch.full((p.tokens, hq, d), 7.0, device="cuda", dtype=DTYPES[dt])
        before = p.both.clone()
        got = eng.cache_append(k.cuda(), v.cuda(), *p.arrays(), rope_freq_base=theta,
                               **({} if theta is None else dict(q=q, q_rot=q_rot)))
        assert (got is None) == (theta is None)
        pos = p.positions()
        turned = ch.rotate(k.double(), pos, theta)
        bound = (ch.half_step(DTYPES[dt]) * turned.abs() + 8 * ch.F * ch.pair_size(k.double())
                 if theta else torch.zeros_like(turned))
        kp, vp = p.k_pages.cpu(), p.v_pages.cpu()
        was = before.cpu().nan_to_num(9.0)
        t = 0
        for b, (n, kv) in enumerate(seqs):
            for i in range(n):
                at, row = int(p.table[b, (kv - n + i) // page]), (kv - n + i) % page
                ch.check("k", kp[at, :, row], turned[t], bound[t])
                assert torch.equal(vp[at, :, row], v[t])
                was[at, 0, :, row], was[at, 1, :, row] = kp[at, :, row], vp[at, :, row]
                t += 1
        assert torch.equal(was, p.both.cpu().nan_to_num(9.0)), "no other row changes"
        if theta:
            live = slice(0, p.tokens - pad)
            want = ch.rotate(p.q.double(), pos, theta)
            b = ch.half_step(DTYPES[dt]) * want.abs() + 8 * ch.F * ch.pair_size(p.q.double())
            ch.check("q", q_rot[live], want[live], b[live])
            assert (q_rot[p.tokens - pad:] == 7.0).all()
            eng.cache_append(k.cuda(), v.cuda(), *p.arrays(), rope_freq_base=theta, q=q, q_rot=q)
            assert torch.equal(q[live], q_rot[live])


def test_empty_calls(eng):
    p = ch.Paged([(0, 20), (0, 0)], 4, 2, 64, 16, torch.bfloat16, 12)
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), save=True)  # no rows
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    eng.cache_append(none, none, *p.arrays())
    # rows, but no sequence
    q = torch.full((3, 4, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    zero = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = eng.cache_forward(q, p.k_pages, p.v_pages, zero, zero[:0], p.table[:0], out=q.clone())[0]
    assert torch.equal(out, q)


def test_refusals(eng):
    p = ch.Paged([(1, 20)], 4, 2, 64, 16, torch.bfloat16, 13)
    q = p.q.cuda()
    k = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    for change in (dict(cu_tokens=p.cu.long()), dict(kv_lens=p.kv_lens.float()), dict(page_table=p.table.cpu()),
                   dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(k_pages=p.k_pages.float()),
                   dict(v_pages=p.v_pages[:-1]), dict(k_pages=p.k_pages.transpose(1, 2)),
                   dict(v_pages=p.v_pages.contiguous()), dict(lse=torch.zeros(4, 2, device="cuda"))):
        args = dict(q=q, k_pages=p.k_pages, v_pages=p.v_pages, cu_tokens=p.cu, kv_lens=p.kv_lens,
                    page_table=p.table)
        args.update(change)
        with pytest.raises(TypeError):
            eng.cache_forward(**args)
    with pytest.raises(ga.InvalidArgument):  # q without a rotation
        eng.cache_append(k, k, *p.arrays(), q=q)
    with pytest.raises(ga.InvalidArgument):
        eng.cache_append(k, k, *p.arrays(), rope_freq_base=-1.0)
    with pytest.raises(ga.InvalidArgument):  # 3 query heads for 2 of the cache
        eng.cache_forward(q[:, :3].contiguous(), *p.arrays())


@pytest.mark.parametrize("normed", [False, True])
def test_a_prompt_and_its_answer_as_one_sequence(eng, normed):
    """A sequence given chunk by chunk and then token by token, through norms,
    append and attention, has the rows that the whole sequence has in
    glacier_attn_forward, which the training path uses."""
    T, hq, hkv, d, page, theta = 150, 14, 2, 64, 16, 1.0e6
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(T, h, d, device="cuda", generator=g).bfloat16() for h in (hq, hkv, hkv))
    wq, wk = (1 + 0.1 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    qn, kn = eng.qk_norm_forward(q, k, wq, wk, 1e-6) if normed else (q, k)
    want = eng.forward(qn, kn, v, theta, save=False)[0].float()
    pages = torch.zeros(2, 12, hkv, page, d, device="cuda", dtype=torch.bfloat16)
    table = torch.randperm(12, device="cuda", generator=g).to(torch.int32)[None]
    at = 0
    for n in [64, 1, 37, 40] + [1] * 8:
        rows = slice(at, at + n)
        at += n
        cu = torch.tensor([0, n], device="cuda", dtype=torch.int32)
        lens = torch.tensor([at], device="cuda", dtype=torch.int32)
        arrays = (pages[0], pages[1], cu, lens, table)
        if normed:  # norms and rotation in one pass, keys appended as they are
            pos = torch.arange(at - n, at, device="cuda", dtype=torch.int32)
            q_rot, k_rot = eng.qk_norm_forward(q[rows].contiguous(), k[rows].contiguous(), wq, wk, 1e-6,
                                               rope_freq_base=theta, positions=pos)
            eng.cache_append(k_rot, v[rows], *arrays)
        else:
            q_rot = eng.cache_append(k[rows], v[rows], *arrays, rope_freq_base=theta, q=q[rows])
        out = eng.cache_forward(q_rot, *arrays)[0].float()
        # both sides hold bf16 weights, queries and outputs: the path's bf16 gate
        assert (out - want[rows]).abs().max() <= 2e-2 * want.abs().max()
    assert at == T


def test_a_captured_step_follows_its_arrays(eng):
    """One captured step of append and attention, replayed for growing
    sequences by changing the device arrays only, between eager calls."""
    hq, hkv, d, page, theta, B = 8, 2, 128, 16, 5e5, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    pages = n(2, 200, hkv, page, d)
    mirror = pages.clone()
    table = torch.randperm(200, device="cuda", generator=g)[:B * 60].view(B, 60).to(torch.int32)
    q, k, v = n(B + 2, hq, d), n(B + 2, hkv, d), n(B + 2, hkv, d)
    cu = torch.arange(B + 1, device="cuda", dtype=torch.int32)
    lens = torch.tensor([1, 500, 900], device="cuda", dtype=torch.int32)
    out, q_rot = torch.zeros_like(q), torch.zeros_like(q)

    def step(store, to, rot):
        eng.cache_append(k, v, store[0], store[1], cu, lens, table, rope_freq_base=theta, q=q, q_rot=rot)
        eng.cache_forward(rot, store[0], store[1], cu, lens, table, max_new=1, max_kv=960, out=to)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pages, out, q_rot)
    for turn in range(4):
        for t in (q, k, v):
            t.copy_(n(*t.shape))
        # rows behind the last sequence keep what the replay before left there
        want, rot = out.clone(), torch.zeros_like(q)
        step(mirror, want, rot)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pages, mirror)
        lens += 1
        if turn == 1:  # one sequence rests
            cu.copy_(torch.tensor([0, 1, 1, 2], dtype=torch.int32))


def test_another_stream(eng):
    p = ch.Paged([(20, 300), (1, 700)], 8, 2, 128, 16, torch.bfloat16, 14)
    q = p.q.cuda()
    want = eng.cache_forward(q, *p.arrays())[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eng.cache_forward(q, *p.arrays())[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_offsets_past_32_bits(eng, dt):
    # pages whose elements lie past 2^31 (and bytes past 2^32) of one allocation
    d, page, hkv, hq = 128, 256, 8, 16
    size = hkv * page * d
    n = 2 ** 31 // size + 40
    p = ch.Paged([(3, 700), (1, 300)], hq, hkv, d, page, DTYPES[dt], 17, spare=0)
    far = torch.arange(n - p.n_pages, n, device="cuda")
    pages = []
    for x in (p.k_pages, p.v_pages):
        big = torch.empty(n, hkv, page, d, device="cuda", dtype=DTYPES[dt])
        big[far] = x
        pages.append(big)
    table = torch.where(p.table >= 0, p.table + n - p.n_pages, p.table)
    ref = ch.attend_ref(p)
    out, lse = eng.cache_forward(p.q.cuda(), *pages, p.cu, p.kv_lens, table, save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    k = torch.randn(4, hkv, d, device="cuda").to(DTYPES[dt])
    eng.cache_append(k, 2 * k, *pages, p.cu, p.kv_lens, table)
    for t, (b, pos) in enumerate([(0, 697), (0, 698), (0, 699), (1, 299)]):
        at = int(table[b, pos // page])
        assert torch.equal(pages[0][at, :, pos % page], k[t])
        assert torch.equal(pages[1][at, :, pos % page], 2 * k[t])


def test_two_graphs_of_one_engine_run_side_by_side(eng):
    # each captured call has a workspace of its own, so graphs of one engine may
    # run at the same time; every replay is checked against the eager result
    g = torch.Generator(device="cuda").manual_seed(5)
    runs = []
    for seqs, hq, hkv, d in (([(1, 6000), (1, 3000)], 28, 4, 128), ([(150, 5000)], 16, 4, 128)):
        p = ch.Paged(seqs, hq, hkv, d, 64, torch.bfloat16, 18)
        q = p.q.cuda()
        w = torch.ones(d, device="cuda")
        dw = torch.zeros(2, d, device="cuda")
        out, lse = torch.empty_like(q), torch.empty(hq, p.tokens, device="cuda")
        x = torch.randn(400, hq, d, device="cuda", generator=g).bfloat16()
        dx = torch.empty_like(x), torch.empty_like(x)

        def step(p=p, q=q, w=w, dw=dw, out=out, lse=lse, x=x, dx=dx):
            dw.zero_()
            eng.cache_forward(q, *p.arrays(), out=out, lse=lse)
            eng.qk_norm_backward(x, x, x, x, w, w, 1e-6, rope_freq_base=1e6, dq=dx[0], dk=dx[1],
                                 dq_weight=dw[0], dk_weight=dw[1])

        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (out, lse, dw, *dx)]
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, stream, (out, lse, dw, *dx), want, p, q, w, x))
    for _ in range(4):
        for _, _, got, _, *_ in runs:
            for t in got:
                t.fill_(5.0)
        torch.cuda.synchronize()
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, got, want, *_ in runs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_sequences_that_share_a_prefix(eng, dt, columns):
    # the first 64 tokens of both are one set of pages
    p = ch.Paged([(9, 100), (20, 130)], 8, 2, 64, 16, DTYPES[dt], 23, columns=columns)
    p.table[1, :4] = p.table[0, :4]
    for x in (p.k, p.v):
        x[1][:64] = x[0][:64]
    ref = ch.attend_ref(p)
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("cu", [[0, 9, 200], [0, 60, 20], [-7, 9, 29], [29, 29, 29], [5, 4, 3]])
def test_wrong_offsets_stay_in_their_rows(eng, cu, columns):
    # cu_tokens that no batch has: wrong rows at most, none outside the tensors
    p = ch.Paged([(9, 100), (20, 130)], 8, 2, 64, 16, torch.bfloat16, 24, columns=columns)
    bad = torch.tensor(cu, dtype=torch.int32, device="cuda")
    args = (p.k_pages, p.v_pages, bad, p.kv_lens, p.table)
    rows = torch.full((3 * p.tokens, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((3, 8, p.tokens), 7.0, device="cuda")
    own = slice(p.tokens, 2 * p.tokens)
    q, used = p.q.cuda(), p.both.clone()
    eng.cache_forward(q, *args, out=rows[own], lse=lse[1])
    eng.cache_append(q[:, :2].contiguous(), q[:, 2:4].contiguous(), *args, rope_freq_base=1e4, q=q,
                     q_rot=rows[own])
    assert (rows[:p.tokens] == 7.0).all() and (rows[2 * p.tokens:] == 7.0).all()
    assert (lse[0] == 7.0).all() and (lse[2] == 7.0).all()
    # appended rows lie in the sequences' pages
    free = torch.ones(p.n_pages, dtype=torch.bool, device="cuda")
    free[p.table[p.table >= 0].long()] = False
    assert torch.equal(p.both[free].view(torch.int16), used[free].view(torch.int16))


def test_two_engines_from_two_threads():
    runs, failed = [], []
    for seed, (seqs, hq, hkv, d) in enumerate((([(1, 4000), (1, 900)], 28, 4, 128), ([(100, 900)], 8, 2, 64))):
        p = ch.Paged(seqs, hq, hkv, d, 16, torch.bfloat16, 25 + seed)
        runs.append((ga.GpuAttentionEngine(0, ga.PREC_BF16), torch.cuda.Stream(), p, p.q.cuda()))
    want = [e.cache_forward(q, *p.arrays())[0] for e, _, p, q in runs]
    torch.cuda.synchronize()

    def work(i):
        e, stream, p, q = runs[i]
        try:
            with torch.cuda.stream(stream):
                got = [e.cache_forward(q, *p.arrays())[0] for _ in range(20)]
                stream.synchronize()
            assert all(torch.equal(x, want[i]) for x in got)
        except BaseException as x:  # noqa: BLE001
            failed.append(x)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for e, *_ in runs:
        e.close()
    assert not failed, failed
