"""The paged cache in 4 bits (glacier_attn_qcache_*), through the Python front end,
against its definition in 64 bits."""
import math

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402
import quant_harness as qh  # noqa: E402
from test_cache_gpu import BATCHES, CHUNKS, WIDE  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


def _appended(eng, name, dt, theta):
    """A batch's new tokens appended to pages of ones; (batch, k, v, q, q_rot)."""
    seqs, hq, hkv, d, page, pad = BATCHES[name]
    p = ch.Paged(seqs, hq, hkv, d, page, dt, 21, pad, device="cpu")
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(p.tokens, hkv, d, generator=g).to(dt) for _ in range(2))
    pages = torch.full((p.n_pages, 2, hkv, ga.quant_page_bytes(page, d)), 255, dtype=torch.uint8, device="cuda")
    index = (pages[:, 0], pages[:, 1], p.cu.cuda(), p.kv_lens.cuda(), p.table.cuda())
    q = None if theta is None else p.q.cuda()
    q_rot = eng.qcache_append(k.cuda(), v.cuda(), *index, rope_freq_base=theta, q=q)
    return p, k, v, q_rot, index


@pytest.mark.parametrize("theta", [None, 1e6])
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_append_and_read(eng, name, dt, theta):
    dt = DTYPES[dt]
    p, k, v, q_rot, index = _appended(eng, name, dt, theta)
    pos, live = p.positions(), sum(n for n, _ in p.seqs)
    turned = ch.rotate(k.double(), pos, theta).float()
    want_k, want_v = qh.held(turned), qh.held(v)
    got_k, got_v = (torch.full(k.shape, 7.0, dtype=dt, device="cuda") for _ in range(2))
    eng.qcache_read(*index, p.tokens, p.d, dt, k=got_k, v=got_v)
    assert torch.equal(got_k[:live].cpu().double(), want_k[:live])
    assert torch.equal(got_v[:live].cpu().double(), want_v[:live])
    assert (got_k[live:] == 7.0).all() and (got_v[live:] == 7.0).all()
    # the pages themselves: every token at its place, every other byte as it was
    bytes_ = torch.full((p.n_pages, 2, p.hkv, ga.quant_page_bytes(p.page, p.d)), 255, dtype=torch.uint8)
    (kn, ks), (vn, vs) = qh.parts(turned), qh.parts(v)
    seq = [b for b, (n, _) in enumerate(p.seqs) for _ in range(n)]
    for t in range(live):
        at = int(pos[t])
        to = bytes_[int(p.table[seq[t], at // p.page])]
        qh.put(to[0], p.page, p.d, "k", at % p.page, kn[t], ks[t])
        qh.put(to[1], p.page, p.d, "v", at % p.page, vn[t], vs[t])
    assert torch.equal(index[0].cpu(), bytes_[:, 0]) and torch.equal(index[1].cpu(), bytes_[:, 1])
    if theta is not None:
        want = ch.rotate(p.q.double(), pos, theta)
        ch.check("q_rot", q_rot[:live], want[:live],
                 ((ch.half_step(dt) + ch.F) * want.abs() + 4 * ch.F * ch.F * ch.pair_size(p.q.double()))[:live])


def test_values_at_the_borders(eng):
    # ties between two numbers, magnitudes past the largest scale's, subnormal and zero
    # scales, two elements of one magnitude, NaN and infinities
    g = torch.Generator().manual_seed(9)
    rows = [torch.linspace(-8, 8, 64) / 2, torch.arange(64).float() % 17 - 8, torch.zeros(64),
            torch.randn(64, generator=g) * 1e6, torch.randn(64, generator=g) * 2.0 ** -22,
            torch.randn(64, generator=g) * 2.0 ** -18, torch.randn(64, generator=g) * 1e-30,
            torch.full((64,), -3.0), torch.full((64,), 3.4e38), 21504.0 * (torch.rand(64, generator=g) * 2 - 1),
            -torch.arange(64).float() * 0.5, 2.0 ** torch.arange(-32, 32).float()]
    for x in (math.nan, math.inf, -math.inf):
        rows.append(torch.randn(64, generator=g))
        rows[-1][40] = x
    x = torch.stack(rows)[:, None]  # [T, 1, 64]
    T = len(rows)
    pages = torch.zeros(2, 2, 1, ga.quant_page_bytes(16, 64), dtype=torch.uint8, device="cuda")
    index = (pages[0], pages[1], torch.tensor([0, T], dtype=torch.int32, device="cuda"),
             torch.tensor([T], dtype=torch.int32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    index = (pages[:1].reshape(2, 1, -1)[:1], pages[1:].reshape(2, 1, -1)[:1], *index[2:])
    eng.qcache_append(x.cuda(), x.flip(0).contiguous().cuda(), *index)
    k, v = eng.qcache_read(*index, T, 64, torch.float32)
    want = qh.held(x)
    assert torch.equal(k.cpu().double().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))
    assert torch.equal(v.cpu().double().nan_to_num(nan=1e300), want.flip(0).nan_to_num(nan=1e300))
    assert want[12:].isnan().sum() == 3 * 32  # a group each
    # bf16 reads the same values
    kb, _ = eng.qcache_read(*index, T, 64, torch.bfloat16)
    assert torch.equal(kb.double().nan_to_num(nan=1e300), k.double().nan_to_num(nan=1e300))


@pytest.mark.parametrize("columns", [0, WIDE])
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_attention(eng, name, dt, columns):
    seqs, hq, hkv, d, page, pad = BATCHES[name]
    p = qh.QPaged(seqs, hq, hkv, d, page, DTYPES[dt], 5, pad, columns=columns // page)
    q = p.q.cuda()
    out = torch.full_like(q, 7.0)
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = qh.attend_ref(p)
    hints = dict(max_new=max(n for n, _ in seqs), max_kv=max(kv for _, kv in seqs))
    for kw in (hints, dict(max_kv=20000), {}):
        eng.qcache_forward(q, *p.arrays(), out=out, lse=lse, **kw)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
    if pad:  # rows behind the last sequence stay as they were
        assert (out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all()
    again, none = eng.qcache_forward(q, *p.arrays())
    live = slice(0, p.tokens - pad)
    assert none is None and torch.equal(again[live], out[live])
    eng.qcache_forward(q, *p.arrays(), out=q)  # over its own queries
    assert torch.equal(q[live], out[live])


@pytest.mark.parametrize("keys", [512, 3000, WIDE])
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(CHUNKS))
def test_chunks_in_every_layout(eng, name, dt, keys):
    # (WIDE: the table is too wide for the pages to be written out where there are many
    # sequences; elsewhere max_kv steers)
    seqs, hq, hkv, d, page, pad = CHUNKS[name]
    p = qh.QPaged(seqs, hq, hkv, d, page, DTYPES[dt], 15, pad, columns=keys // page)
    out = torch.full((p.tokens, hq, d), 7.0, device="cuda", dtype=DTYPES[dt])
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = qh.attend_ref(p)
    eng.qcache_forward(p.q.cuda(), *p.arrays(), max_kv=keys, out=out, lse=lse)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])
    assert not pad or ((out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all())


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_wrong_hints_change_nothing_but_the_layout(eng, dt):
    p = qh.QPaged([(70, 400), (1, 2500)], 8, 2, 128, 16, DTYPES[dt], 6)
    ref = qh.attend_ref(p)
    for kw in (dict(max_new=1, max_kv=1), dict(max_new=70, max_kv=300), dict(max_new=10 ** 6, max_kv=10 ** 9)):
        out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True, **kw)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_rows_without_a_key(eng, dt, columns):
    # a length below the number of new tokens leaves the first rows at negative
    # positions: they see nothing, get 0 and -inf; appending drops them, reading gives 0
    p = qh.QPaged([(6, 9), (3, 3)], 16, 2, 64, 16, DTYPES[dt], 7, columns=columns)
    p.kv_lens[1] = 1
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    assert not out[6:8].any() and (lse[:, 6:8] == -math.inf).all()
    assert out[8].any() and not out.isnan().any()
    k, v = eng.qcache_read(*p.arrays(), p.tokens, p.d, DTYPES[dt])
    assert not k[6:8].any() and not v[6:8].any() and torch.equal(k[8].cpu().double(), p.k[1][0])
    before = p.both.clone()
    eng.qcache_append(*(torch.randn(p.tokens, 2, 64, device="cuda").to(DTYPES[dt]) for _ in range(2)),
                      p.k_pages, p.v_pages, p.cu, p.kv_lens - torch.tensor([9, 1], device="cuda").int(), p.table)
    assert torch.equal(before, p.both)


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_bad_pages_hold_no_keys(eng, dt, columns):
    seqs = [(4, 100), (1, 70), (20, 64)]
    p = qh.QPaged(seqs, 8, 2, 64, 16, DTYPES[dt], 8, columns=columns)
    p.table[0, 2], p.table[1, 0], p.table[2, 1] = -1, p.n_pages, 2 ** 31 - 1
    gone = [(0, j) for j in range(32, 48)] + [(1, j) for j in range(16)] + [(2, j) for j in range(16, 32)]
    for kw in ({}, dict(max_new=20, max_kv=100)):
        out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True, **kw)
        # the same without those keys, as one key fewer each: compared with the plain form
        ref = ch.attend_ref(p, hidden=gone)
        far = qh.attend_ref(p)
        ch.check("out", out, ref[0], ref[1] + far[1])
        ch.check("lse", lse, ref[2], ref[3] + far[3])
    k, _ = eng.qcache_read(p.k_pages, p.v_pages, torch.tensor([0, 100, 170, 234], device="cuda").int(), p.kv_lens,
                           p.table, 234, 64, DTYPES[dt])
    assert not k[32:48].any() and not k[100:116].any() and k[:32].any()


@pytest.mark.parametrize("columns", [0, WIDE // 16])
@pytest.mark.parametrize("hq,d", [(4, 64), (16, 128), (6, 96), (8, 256), (4, 32)])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_not_finite_keys_reach_only_rows_that_see_them(eng, dt, hq, d, columns):
    # a group with a NaN or an infinity is NaN: as a key it makes every row that sees it
    # NaN, as a value its 32 columns
    def change(p):
        p.v[0][33, 0, 5] = math.nan
        p.v[0][38, 1, d - 1] = -math.inf
        p.k[1][50, 0, 3] = math.inf

    p = qh.QPaged([(8, 40), (3, 52)], hq, 2, d, 16, DTYPES[dt], 12, columns=columns, change=change)
    clean = qh.QPaged([(8, 40), (3, 52)], hq, 2, d, 16, DTYPES[dt], 12, columns=columns)
    for kw in ({}, dict(max_new=8, max_kv=52)):
        out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True, **kw)
        # (a wave that meets one sums its keys again, 128-row tiles in another order)
        want, bound, *_ = qh.attend_ref(clean)
        odd = torch.zeros_like(out, dtype=torch.bool)
        half = hq // 2
        odd[1:8, :half, :32] = True  # positions 33 .. 39 of 32 .. 39
        odd[6:8, half:, (d - 1) // 32 * 32:] = True
        odd[9:, :half] = True  # positions 50, 51 of 49 .. 51
        assert torch.equal(out.isnan(), odd)
        ch.check("out", torch.where(odd, 0.0, out), torch.where(odd.cpu(), 0.0, want), bound)
        assert lse[:half, 9:].isnan().all() and not lse[half:].isnan().any() and not lse[:, :9].isnan().any()


@pytest.mark.parametrize("power", [-20, 0, 6])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_scores_far_from_zero(eng, dt, power):
    # scores of size 2^power, all of one sign in the second sequence
    def change(p):
        p.q *= 2.0 ** power
        p.k[1] = p.k[1].abs()
        p.q[3:] = -p.q[3:].abs()

    p = qh.QPaged([(3, 90), (2, 700)], 8, 2, 64, 16, DTYPES[dt], 13, change=change)
    ref = qh.attend_ref(p)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])


@pytest.mark.parametrize("size", [2.0 ** -16, 2.0 ** -10, 2.0 ** 14])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_values_of_every_size(eng, dt, size):
    # scales down to fp16's subnormals and up to the largest one
    def change(p):
        for b in range(len(p.v)):
            p.v[b] *= size / p.v[b].abs().max()

    p = qh.QPaged([(2, 200), (1, 1500)], 8, 1, 128, 32, DTYPES[dt], 14, change=change)
    ref = qh.attend_ref(p)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    ch.check("out", out, ref[0], ref[1])
    ch.check("lse", lse, ref[2], ref[3])


def test_empty_calls(eng):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = torch.zeros(0, 2, ga.quant_page_bytes(16, 64), dtype=torch.uint8, device="cuda")
    q, k = torch.zeros(0, 4, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda")
    for n in (0, 2):
        index = (pages, pages, z(n + 1), z(n), z(n, 3))
        out, lse = eng.qcache_forward(q, *index, save=True)
        assert out.shape == q.shape and lse.shape == (4, 0)
        assert eng.qcache_append(k, k, *index) is None
        assert eng.qcache_read(*index, 0, 64, torch.float32)[0].shape == k.shape
    # rows, but no page at all: they see nothing
    q = torch.ones(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    out, lse = eng.qcache_forward(q, pages, pages, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), z(1) + 2,
                                  z(1, 3), save=True)
    assert not out.any() and (lse == -math.inf).all()
    out, lse = eng.qcache_forward(q, pages, pages, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), z(1) + 2,
                                  z(1, 0), save=True)
    assert not out.any() and (lse == -math.inf).all()


def test_offsets_past_32_bits(eng):
    # pages 2^30 bytes apart, four and more of them
    p = qh.QPaged([(2, 70)], 8, 2, 128, 16, torch.bfloat16, 17, spare=1)
    size = p.both[0, 0].numel()
    whole = torch.empty((p.n_pages - 1) * 2 ** 30 + 2 * size, dtype=torch.uint8, device="cuda")
    k, v = (torch.as_strided(whole, (p.n_pages, 2, size // 2), (2 ** 30, size // 2, 1), side * size) for side in (0, 1))
    k.copy_(p.k_pages), v.copy_(p.v_pages)
    index = (k, v, *p.arrays()[2:])
    ref = qh.attend_ref(p)
    for kw in ({}, dict(max_new=2, max_kv=10 ** 9)):
        out, _ = eng.qcache_forward(p.q.cuda(), *index, **kw)
        ch.check("out", out, ref[0], ref[1])
    got, _ = eng.qcache_read(*index, 2, 128, torch.float32)
    assert torch.equal(got.cpu().double(), p.k[0][68:])
    new = torch.randn(2, 2, 128, device="cuda")
    eng.qcache_append(new, new, *index)
    got, back = eng.qcache_read(*index, 2, 128, torch.float32)
    assert torch.equal(got.cpu().double(), qh.held(new.cpu())) and torch.equal(got, back)


def _step(eng, p, k, v, index, work):
    q = eng.qcache_append(k, v, *index, rope_freq_base=1e4, q=p.q.cuda() if work is None else work)
    return eng.qcache_forward(q, *index, max_new=1, max_kv=400, save=True)


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_captured_steps_follow_their_arrays(eng, dt):
    # two graphs of one engine, replayed side by side on two streams with lengths that
    # change between the replays; eager steps in between, each against its eager twin
    dt = DTYPES[dt]
    sets = []
    for seed in (31, 32):
        p = qh.QPaged([(1, 100), (1, 250), (1, 17)], 8, 2, 64, 16, dt, seed, columns=25)
        g = torch.Generator().manual_seed(seed)
        k, v = (torch.randn(3, 2, 64, generator=g).to(dt).cuda() for _ in range(2))
        sets.append((p, k, v, p.arrays(), p.q.cuda()))
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for (p, k, v, index, q), stream in zip(sets, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _step(eng, p, k, v, index, q)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(_step(eng, p, k, v, index, q))
        graphs.append(graph)
    for turn in range(4):
        for p, *_ in sets:
            p.kv_lens -= torch.tensor([turn, 40, 1], dtype=torch.int32, device="cuda")
            p.kv_lens.clamp_(min=1)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        got = [(o.clone(), x.clone()) for o, x in outs]
        for (p, k, v, index, q), (o, x) in zip(sets, got):
            want = _step(eng, p, k, v, index, q)
            assert torch.equal(o, want[0]) and torch.equal(x, want[1])


def test_another_stream(eng):
    p = qh.QPaged([(1, 300), (60, 200)], 8, 2, 128, 16, torch.bfloat16, 33)
    want, _ = eng.qcache_forward(p.q.cuda(), *p.arrays(), max_new=60, max_kv=300)
    q = p.q.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, _ = eng.qcache_forward(q, *p.arrays(), max_new=60, max_kv=300)
    stream.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("cu", [[0, 5, 3, 4], [-7, 2, 900, 3], [4, 4, 1, 0], [0, 2 ** 31 - 1, -2 ** 31, 8]])
def test_wrong_offsets_stay_in_their_rows(eng, cu):
    # offsets that no batch has: nothing past the tensors is touched, and the calls end
    p = qh.QPaged([(2, 30), (2, 40), (4, 50)], 8, 2, 64, 16, torch.bfloat16, 34)
    wrong = torch.tensor(cu, dtype=torch.int32, device="cuda")
    index = (p.k_pages, p.v_pages, wrong, p.kv_lens, p.table)
    rows = torch.full((10, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    for kw in ({}, dict(max_new=10 ** 6)):
        eng.qcache_forward(p.q.cuda(), *index, out=rows[1:9], **kw)
    k, v = (torch.full((10, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    eng.qcache_read(*index, 8, 64, torch.bfloat16, k=k[1:9], v=v[1:9])
    eng.qcache_append(p.q[:, :2].contiguous().cuda(), p.q[:, 2:4].contiguous().cuda(), *index)
    torch.cuda.synchronize()
    for t in (rows, k, v):
        assert (t[0] == 7.0).all() and (t[9] == 7.0).all()


def test_lengths_past_the_table(eng):
    # keys past the table's columns are not there; neither are tokens appended there
    p = qh.QPaged([(1, 64), (40, 64)], 4, 2, 64, 16, torch.bfloat16, 35)
    table = p.table[:, :2].contiguous()
    short = qh.QPaged([(1, 64), (40, 64)], 4, 2, 64, 16, torch.bfloat16, 35)
    for columns in (2, 3):
        table = p.table[:, :columns].contiguous()
        index = (p.k_pages, p.v_pages, p.cu, p.kv_lens, table)
        gone = [(b, j) for b in (0, 1) for j in range(16 * columns, 64)]
        ref, far = ch.attend_ref(short, hidden=gone), qh.attend_ref(short)
        out, lse = eng.qcache_forward(p.q.cuda(), *index, save=True)
        ch.check("out", out, ref[0], ref[1] + far[1])
        ch.check("lse", lse, ref[2], ref[3] + far[3])
        before = p.both.clone()
        eng.qcache_append(*(torch.randn(41, 2, 64, device="cuda").bfloat16() for _ in range(2)),
                          p.k_pages, p.v_pages, torch.tensor([0, 1, 1], device="cuda").int(), p.kv_lens, table)
        assert torch.equal(before, p.both)


def _written_out(eng, p):
    """Whether a call without hints writes the pages out first: from a mean of 256 rows
    (token, head of the group) a sequence on, where tiles of more than 16 rows are taken."""
    cache, batch = ga.qcache_args(*p.arrays(), p.tokens, 0, 0, 0, p.d, p.dtype)
    size = ga._lib.glacier_attn_qcache_workspace(eng._h, ga.ctypes.byref(cache), ga.ctypes.byref(batch), p.hq)
    assert p.tokens * (p.hq // p.hkv) > 256 * len(p.seqs)
    return size >= 2 * p.table.numel() * p.page * p.hkv * p.d * p.q.element_size()


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("seqs,hq,hkv,d,page,pad", [
    ([(90, 400), (75, 1500)], 28, 4, 128, 16, 3), ([(300, 300)], 14, 2, 64, 32, 0), ([(60, 61), (40, 700)], 8, 1, 96, 16, 2),
    ([(200, 900), (1, 800), (0, 40)], 16, 4, 256, 16, 1)])
def test_chunks_of_many_rows(eng, seqs, hq, hkv, d, page, pad, dt):
    # with hints in tiles of 16 rows, without them written out
    p = qh.QPaged(seqs, hq, hkv, d, page, DTYPES[dt], 23, pad, columns=16384 // page)
    assert _written_out(eng, p) == (dt == "bf16" or 64 < d <= 128)
    out = torch.full((p.tokens, hq, d), 7.0, device="cuda", dtype=DTYPES[dt])
    lse = torch.full((hq, p.tokens), 7.0, device="cuda")
    ref = qh.attend_ref(p)
    for hints in (dict(max_new=max(n for n, _ in seqs), max_kv=max(n for _, n in seqs)), {}):
        eng.qcache_forward(p.q.cuda(), *p.arrays(), out=out, lse=lse, **hints)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
    assert not pad or ((out[-pad:] == 7.0).all() and (lse[:, -pad:] == 7.0).all())


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_many_rows_without_a_key(eng, dt):
    p = qh.QPaged([(25, 30), (20, 20)], 28, 2, 96, 16, DTYPES[dt], 24, columns=1024)
    assert _written_out(eng, p)
    p.kv_lens[1] = 5
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    assert not out[25:40].any() and (lse[:, 25:40] == -math.inf).all()
    assert out[40].any() and not out.isnan().any()
    ref = qh.attend_ref(p)
    ch.check("out", out[:25], ref[0][:25], ref[1][:25])
    p.kv_lens[0] = -3
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    assert not out[:40].any() and (lse[:, :40] == -math.inf).all()


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_many_rows_and_bad_pages(eng, dt):
    p = qh.QPaged([(24, 100), (19, 70), (20, 64)], 28, 2, 128, 16, DTYPES[dt], 25, columns=1024)
    assert _written_out(eng, p)
    p.table[0, 2], p.table[1, 0], p.table[2, 1] = -1, p.n_pages, 2 ** 31 - 1
    gone = [(0, j) for j in range(32, 48)] + [(1, j) for j in range(16)] + [(2, j) for j in range(16, 32)]
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    ref, far = ch.attend_ref(p, hidden=gone), qh.attend_ref(p)
    ch.check("out", out, ref[0], ref[1] + far[1])
    ch.check("lse", lse, ref[2], ref[3] + far[3])


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_many_rows_and_keys_that_are_not_finite(eng, dt, d):
    def change(p):
        p.v[0][33, 0, 5] = math.nan
        p.k[1][50, 0, 3] = math.inf

    args = ([(28, 40), (23, 52)], 28, 2, d, 16, DTYPES[dt], 26)
    p, clean = qh.QPaged(*args, change=change, columns=1024), qh.QPaged(*args)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    want, bound, *_ = qh.attend_ref(clean)
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[21:28, :14, :32] = True  # positions 33 .. 39 of 12 .. 39
    odd[49:, :14] = True  # positions 50, 51 of 29 .. 51
    assert torch.equal(out.isnan(), odd)
    ch.check("out", torch.where(odd, 0.0, out), torch.where(odd.cpu(), 0.0, want), bound)
    assert lse[:14, 49:].isnan().all() and not lse[14:].isnan().any() and not lse[:, :49].isnan().any()


@pytest.mark.parametrize("cu", [[0, 25, 3, 40], [-7, 2, 900, 3], [44, 4, 1, 0], [0, 2 ** 31 - 1, -2 ** 31, 60]])
def test_many_rows_and_wrong_offsets(eng, cu):
    p = qh.QPaged([(20, 30), (20, 40), (20, 50)], 28, 2, 64, 16, torch.bfloat16, 27, columns=1024)
    assert _written_out(eng, p)
    wrong = torch.tensor(cu, dtype=torch.int32, device="cuda")
    rows = torch.full((62, 28, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    eng.qcache_forward(p.q.cuda(), p.k_pages, p.v_pages, wrong, p.kv_lens, p.table, out=rows[1:61])
    torch.cuda.synchronize()
    assert (rows[0] == 7.0).all() and (rows[61] == 7.0).all()


def test_two_engines_and_threads(eng):
    # an engine and a stream each, called from two threads at once
    import threading

    sets = [qh.QPaged([(1, 300), (2, 90)], 8, 2, 128, 16, torch.bfloat16, 40 + i) for i in range(2)]
    want = [eng.qcache_forward(p.q.cuda(), *p.arrays())[0] for p in sets]
    own = [ga.GpuAttentionEngine(0, ga.PREC_BF16) for _ in sets]
    got, failed = [None, None], []

    def run(i):
        try:
            p, q, stream = sets[i], sets[i].q.cuda(), torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                outs = [own[i].qcache_forward(q, *p.arrays())[0] for _ in range(20)]
            stream.synchronize()
            got[i] = outs
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)
    for e in own:
        e.close()


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_captured_chunks_that_are_written_out(eng, dt):
    # two graphs, whose workspaces hold the pages written out, side by side, with lengths
    # that change between the replays
    sets, graphs, outs, streams = [], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (51, 52):
        p = qh.QPaged([(24, 90), (20, 300)], 28, 2, 128, 16, DTYPES[dt], seed, columns=1024)
        assert _written_out(eng, p)
        sets.append((p, p.q.cuda()))
    for (p, q), stream in zip(sets, streams):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(eng.qcache_forward(q, *p.arrays(), save=True))
        graphs.append(graph)
    for turn in range(4):
        for p, _ in sets:
            p.kv_lens -= torch.tensor([9 * turn, 40], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        got = [(o.clone(), x.clone()) for o, x in outs]
        for (p, q), (o, x) in zip(sets, got):
            want = eng.qcache_forward(q, *p.arrays(), save=True)
            assert torch.equal(o, want[0]) and torch.equal(x, want[1])
