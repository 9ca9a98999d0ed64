"""Calls of the 4-bit cache at the ends of what its header allows."""
import math

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402
import quant_harness as qh  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


@pytest.mark.parametrize("n_pages", [0, 3])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (8, 1, 96), (14, 2, 64), (16, 4, 256)])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_tables_without_a_column(eng, dt, hq, hkv, d, n_pages):
    # chunks of any length over a table of no pages see no key, append nowhere, read zeros
    dt, T = DTYPES[dt], 1000
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = torch.full((2, n_pages, hkv, ga.quant_page_bytes(16, d)), 255, dtype=torch.uint8, device="cuda")
    index = (pages[0], pages[1], ints(0, 600, 990), ints(700, 500), torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    q = torch.randn(T, hq, d, device="cuda").to(dt)
    k, v = (torch.randn(T, hkv, d, device="cuda").to(dt) for _ in range(2))
    for kw in ({}, dict(max_new=600, max_kv=700)):
        out, lse = torch.full_like(q, 7.0), torch.full((hq, T), 7.0, device="cuda")
        eng.qcache_forward(q, *index, out=out, lse=lse, **kw)
        assert not out[:990].any() and (lse[:, :990] == -math.inf).all()
        assert (out[990:] == 7.0).all() and (lse[:, 990:] == 7.0).all()
    eng.qcache_append(k, v, *index)
    assert (pages == 255).all()
    eng.qcache_read(*index, T, d, dt, k=k, v=v)
    assert not k[:990].any() and not v[:990].any() and k[990:].all()


@pytest.mark.parametrize("chunk", [1, 3, 40])
@pytest.mark.parametrize("power", [100, 118, 127])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_queries_of_every_size(eng, dt, d, power, chunk):
    # Queries up to the type's largest: in columns whose keys are zero they change nothing
    # (even heads; the others' columns hold ordinary values); as they are over small keys
    # (odd heads), one key has all the weight.
    def change(p):
        for k in p.k:
            k[:, :, :32 if d > 32 else 16] = 0.0
            k[:, 1] *= 2.0 ** -18
        big = 2.0 ** power * (1.0 + torch.rand(p.q.shape, generator=torch.Generator().manual_seed(3)) * 0.99)
        p.q[:, :2, :16] = big[:, :2, :16] * torch.where(p.q[:, :2, :16] < 0, -1.0, 1.0)
        if d > 32:
            p.q[:, :1, 16:32] = big[:, :1, 16:32]  # of one sign: the sum of them is past the type's range
        p.q[:, 2:] = big[:, 2:] * torch.where(p.q[:, 2:] < 0, -1.0, 1.0)

    p = qh.QPaged([(chunk, 300), (1, 1100)], 4, 2, d, 16, DTYPES[dt], 71, change=change)
    assert torch.isfinite(p.q).all()
    ref = qh.attend_ref(p)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), max_kv=1100, save=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    # a score is off by a few 2^-24 of its largest terms, which are zero in the even heads
    for h in range(4):
        live = slice(0, p.tokens)
        ch.check(f"lse{h}", lse[h:h + 1], ref[2][h:h + 1], ref[3][h:h + 1])
        if h < 2:
            ch.check(f"out{h}", out[:, h], ref[0][live, h], ref[1][live, h])
