"""The paged key/value cache (glacier_attn_cache_*) where its layouts of the work
could differ from each other: bits of the weights, sizes of the sums, tiles
without a key, calls without hints."""
import math

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402
from test_cache_gpu import CHUNKS, WIDE  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LAYOUTS = [512, 3000, WIDE]  # max_kv: 16-row tiles, 128-row tiles in few and in many splits


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


@pytest.mark.parametrize("keys", LAYOUTS)
@pytest.mark.parametrize("name", ["d40", "d64", "d128_one_head_groups", "d120_long", "d256"])
def test_weights_reach_v_with_16_bits(eng, name, keys):
    # A weight multiplies V as two bf16 terms: off by 2^-8 of the first one's
    # rounding, itself 2^-8 of the weight.  The sums are off as in fp32.
    seqs, hq, hkv, d, page, pad = CHUNKS[name]
    p = ch.Paged(seqs, hq, hkv, d, page, BF16, 31, pad, columns=WIDE // page)
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, save=True)
    ref = ch.attend_ref(p)
    p.v = [v.abs() for v in p.v]
    size = ch.attend_ref(p)[0]  # weights times |V|
    ch.check("out", out, ref[0], ref[1] - (ch.half_step(BF16) - 2.0 ** -16) * size)
    ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("keys", LAYOUTS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_that_all_round_one_way(eng, d, keys):
    # V is 1, so the result is 1.  Of every 128 keys one has the weight 1 and the
    # others 0.5 (1 + 0.88 / 256), which bf16 rounds to 0.5: one term would give
    # 0.9965.  Two are off by 2^-16 and the sums by 2^-14, less than 2^-9, half a step below 1.
    n, kv, hq, hkv = 140, 1500, 4, 1
    p = ch.Paged([(n, kv)], hq, hkv, d, 16, BF16, 32, columns=WIDE // 16)
    low = math.log(0.5 * (1 + 0.88 / 256)) * math.sqrt(d)
    first = torch.tensor(low).to(BF16)
    k = torch.zeros(kv, d, dtype=BF16)
    k[:, 0], k[:, 1] = first, torch.tensor(low - float(first)).to(BF16)
    k[::128] = 0.0
    pages = p.table[0, :-(-kv // 16)].long()
    rows = torch.zeros(len(pages) * 16, d, dtype=BF16)
    rows[:kv] = k
    p.k_pages[pages, 0] = rows.view(len(pages), 16, d).cuda()
    p.v_pages.fill_(1.0)
    q = torch.zeros(n, hq, d, device="cuda", dtype=BF16)
    q[..., :2] = 1.0
    out = eng.cache_forward(q, *p.arrays(), max_kv=keys)[0]
    assert (out == 1.0).all(), (out.min(), out.max())


# layouts: dtype, hq, hkv, D, max_kv
NO_KEY_LAYOUTS = {
    "bf16 16 rows": ("bf16", 8, 2, 64, 300), "bf16 16 rows, splits": ("bf16", 8, 2, 64, 2000),
    "bf16 128 rows": ("bf16", 320, 20, 128, 512), "bf16 128 rows, splits": ("bf16", 8, 2, 64, WIDE),
    "bf16 128 rows, wide heads": ("bf16", 8, 2, 256, WIDE), "fp32 16 rows": ("fp32", 8, 2, 96, 800),
    "fp32 16 rows, splits": ("fp32", 8, 2, 64, WIDE), "fp32 32 rows": ("fp32", 128, 8, 96, 1000),
    "fp32 32 rows, splits": ("fp32", 8, 2, 96, WIDE)}


@pytest.mark.parametrize("layout", sorted(NO_KEY_LAYOUTS))
def test_tiles_without_a_key(eng, layout):
    # new tokens of sequences without a key (length zero and below), a sequence
    # with keys and idle ones beside them, rows behind the last sequence
    dt, hq, hkv, d, keys = NO_KEY_LAYOUTS[layout]
    seqs, pad = [(20, 20), (0, 50), (33, 33), (40, 300), (0, 0), (9, 9)], 3
    p = ch.Paged(seqs, hq, hkv, d, 16, DTYPES[dt], 33, pad, columns=WIDE // 16)
    p.kv_lens.copy_(torch.tensor([0, 50, -7, 300, 0, -2 ** 31 + 9], dtype=torch.int32))
    live = torch.zeros(p.tokens, dtype=torch.bool)
    live[53:93] = True
    none = ~live
    none[-pad:] = False
    out = torch.full((p.tokens, hq, d), 7.0, device="cuda", dtype=DTYPES[dt])
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = ch.attend_ref(p)
    eng.cache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, out=out, lse=lse)
    ch.check("out", out[live.cuda()], ref[0][live], ref[1][live])
    ch.check("lse", lse[:, live.cuda()], ref[2][:, live], ref[3][:, live])
    assert not out[none.cuda()].any() and (lse[:, none.cuda()] == -math.inf).all()
    assert (out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all()
    before = p.both.clone()
    k = torch.ones(p.tokens, hkv, d, device="cuda", dtype=DTYPES[dt])
    eng.cache_append(k, 2 * k, *p.arrays())
    changed = (~(torch.eq(before, p.both) | (before.isnan() & p.both.isnan()))).any(-1).nonzero()
    want = {(int(p.table[3, pos // 16]), pos % 16) for pos in range(260, 300)}
    assert {(int(r[0]), int(r[3])) for r in changed} == want


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_a_page_table_without_columns(eng, dt):
    p = ch.Paged([(40, 300), (1, 5)], 16, 2, 96, 16, DTYPES[dt], 34, pad=1)
    table = p.table[:, :0].contiguous()
    args = (p.k_pages, p.v_pages, p.cu, p.kv_lens, table)
    out = torch.full((p.tokens, 16, 96), 7.0, device="cuda", dtype=DTYPES[dt])
    lse = torch.full((16, p.tokens), 7.0, device="cuda")
    for hints in ({}, dict(max_new=40, max_kv=300)):
        eng.cache_forward(p.q.cuda(), *args, out=out, lse=lse, **hints)
        assert not out[:-1].any() and (lse[:, :-1] == -math.inf).all()
        assert (out[-1] == 7.0).all() and (lse[:, -1] == 7.0).all()
    before = p.both.clone()
    k = torch.ones(p.tokens, 2, 96, device="cuda", dtype=DTYPES[dt])
    eng.cache_append(k, k, *args)
    assert torch.equal(before.nan_to_num(9.0), p.both.nan_to_num(9.0))


@pytest.mark.parametrize("keys", LAYOUTS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_large_values_under_growing_scores(eng, dt, d, keys):
    # V between 2^121 and 2^122; of every 64 keys one counts, whose weight grows
    # from 1 to 2^7.5: against the first one as reference the sum would leave
    # fp32, against the largest it is below 2^126.  (The others' scores fall, so
    # that no part of the keys has many weights near its own largest.)
    n, kv, hq, hkv = 40, 700, 8, 2
    p = ch.Paged([(n, kv)], hq, hkv, d, 16, DTYPES[dt], 35, columns=WIDE // 16)
    score = -100.0 - 2.0 * torch.arange(kv)
    score[5::64] = torch.arange(len(score[5::64])).mul(1.5).clamp(max=7.5)
    k = torch.zeros(kv, hkv, d)
    k[..., 0] = (score * math.log(2) * math.sqrt(d))[:, None]
    g = torch.Generator().manual_seed(36)
    v = (1 + torch.rand(kv, hkv, d, generator=g)) * 2.0 ** 121
    p.k[0], p.v[0] = k.to(DTYPES[dt]), v.to(DTYPES[dt])
    p.q = torch.zeros(n, hq, d, dtype=DTYPES[dt])
    p.q[..., 0] = 1.0
    pages = p.table[0, :-(-kv // 16)].long().cpu()
    for to, x in ((p.k_pages, p.k[0]), (p.v_pages, p.v[0])):
        rows = torch.zeros(len(pages) * 16, hkv, d, dtype=DTYPES[dt])
        rows[:kv] = x
        to[pages.cuda()] = rows.view(-1, 16, hkv, d).transpose(1, 2).contiguous().cuda()
    out, lse = eng.cache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, save=True)
    ref = ch.attend_ref(p)
    assert torch.isfinite(out).all()
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("n,hq,hkv,d,pad", [(32, 28, 4, 128, 0), (8, 32, 8, 128, 3), (64, 14, 2, 64, 0),
                                            (12, 40, 1, 64, 5), (5, 8, 2, 256, 0)])
def test_single_tokens_without_hints(eng, n, hq, hkv, d, pad, dt):
    # a call that does not know its longest chunk takes a batch of single tokens for
    # what it is: the layout, and so every bit, of a call that says so
    p = ch.Paged([(1, 1 + 37 * i % 900) for i in range(n)], hq, hkv, d, 16, DTYPES[dt], 37, pad, columns=2 ** 14 // 16)
    q = p.q.cuda()
    hints = dict(max_kv=8192)
    want = eng.cache_forward(q, *p.arrays(), max_new=1, save=True, **hints)
    got = eng.cache_forward(q, *p.arrays(), save=True, **hints)
    live = slice(0, p.tokens - pad)
    assert torch.equal(got[0][live], want[0][live]) and torch.equal(got[1][:, live], want[1][:, live])
    size = []
    for max_new in (0, 1):
        cache, batch = ga.cache_args(*p.arrays(), p.tokens, max_new, 8192, 0)
        size.append(ga.load().glacier_attn_cache_workspace(eng._h, cache, batch, hq))
    assert size[0] == size[1]
    ref = ch.attend_ref(p)
    ch.check("out", got[0], ref[0], ref[1])
    ch.check("lse", got[1], ref[2], ref[3])


@pytest.mark.parametrize("seqs,hq,hkv,d,keys", [
    ([(200, 900)], 14, 2, 64, 3000), ([(130, 700), (60, 60)], 32, 8, 128, 2500), ([(150, 1500)], 8, 2, 256, 6000),
    ([(30, 700)], 8, 2, 128, WIDE), ([(1, 1500)], 28, 4, 128, 3000)])
def test_an_infinite_value_in_the_last_split(eng, seqs, hq, hkv, d, keys):
    # an infinity in V makes its columns infinite in every row that sees it (not NaN),
    # whichever split of the keys it lies in and however many there are
    p = ch.Paged(seqs, hq, hkv, d, 16, BF16, 38, columns=WIDE // 16)
    ref = ch.attend_ref(p)
    n, kv = seqs[0]
    sees = torch.zeros(p.tokens, dtype=torch.bool)
    for pos in (kv - 1, kv - n, kv // 2, 0):
        for what in (math.inf, -math.inf):
            both = p.both.clone()
            both[p.table[0, pos // 16], 1, :, pos % 16, 3::7] = what
            out, lse = eng.cache_forward(p.q.cuda(), both[:, 0], both[:, 1], p.cu, p.kv_lens, p.table, max_kv=keys,
                                         save=True)
            sees[:n] = torch.arange(kv - n, kv) >= pos
            assert (out[sees.cuda()][..., 3::7] == what).all()
            rest = ref[0].clone()
            rest[sees, :, 3::7] = math.nan
            ch.check("out", torch.where(rest.isnan().cuda(), 0.0, out.double()), rest, ref[1])
            ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("count", [65, 4096, 4097, 20000])
def test_many_sequences_most_of_them_idle(eng, dt, count):
    # chunks and single tokens at both ends of a long batch and within it
    busy = {0: (40, 90), 1: (1, 7), count // 3: (1, 200), count // 2: (70, 70), count - 2: (3, 30), count - 1: (1, 65)}
    seqs = [busy.get(b, (0, 0)) for b in range(count)]
    p = ch.Paged(seqs, 8, 2, 64, 16, DTYPES[dt], 40, pad=2)
    out = torch.full((p.tokens, 8, 64), 7.0, device="cuda", dtype=DTYPES[dt])
    lse = torch.full((8, p.tokens), 7.0, device="cuda")
    ref = ch.attend_ref(p)
    for hints in ({}, dict(max_new=70, max_kv=200), dict(max_new=70, max_kv=90000)):
        eng.cache_forward(p.q.cuda(), *p.arrays(), out=out, lse=lse, **hints)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
        assert (out[-2:] == 7.0).all() and (lse[:, -2:] == 7.0).all()
    k = torch.randn(p.tokens, 2, 64, device="cuda").to(DTYPES[dt])
    eng.cache_append(k, 2 * k, *p.arrays())
    t = 0
    for b, (n, kv) in sorted(busy.items()):
        for pos in range(kv - n, kv):
            page = int(p.table[b, pos // 16])
            assert torch.equal(p.k_pages[page, :, pos % 16], k[t]) and torch.equal(p.v_pages[page, :, pos % 16], 2 * k[t])
            t += 1


def test_the_search_for_a_sequence_does_not_grow_with_the_batch(eng):
    # 2^19 sequences, all but two idle: a search that looks at all of them in turn in
    # each of as many workgroups takes half a second here, a narrowing one some ms
    n, page = 2 ** 19, 16
    p = ch.Paged([(1, 40), (5, 33)], 8, 1, 64, page, BF16, 41)
    cu = torch.full((n + 1,), 6, device="cuda", dtype=torch.int32)
    cu[:n // 2 + 1] = 0
    cu[n // 2 + 1:n] = 1
    lens = torch.zeros(n, device="cuda", dtype=torch.int32)
    lens[n // 2], lens[n - 1] = 40, 33
    table = torch.full((n, p.table.shape[1]), -1, device="cuda", dtype=torch.int32)
    table[n // 2], table[n - 1] = p.table[0], p.table[1]
    args = (p.q.cuda(), p.k_pages, p.v_pages, cu, lens, table)
    ref = ch.attend_ref(p)
    out, lse = eng.cache_forward(*args, save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    eng.cache_forward(*args, save=True)
    stop.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(stop) < 100.0, f"{start.elapsed_time(stop)} ms"
