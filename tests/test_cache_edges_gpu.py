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
LAYOUTS = [512, 3000, WIDE]  # max_kv: 16-row tiles, 128-row tiles whole, in splits


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
