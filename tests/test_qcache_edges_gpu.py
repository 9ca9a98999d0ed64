"""Calls of the 4-bit cache at the ends of what its header allows."""
import math

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")

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
