"""Products with 4-bit weights and adapters of every rank: partly filled tiles of 16 ranks, and
every kernel that forms x A_p."""
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


@pytest.mark.parametrize("cols,group", [(896, 32), (320, 64)])
@pytest.mark.parametrize("T", [1, 8, 15, 16, 17, 130])
@pytest.mark.parametrize("rank", [2, 15, 17, 31, 32, 33, 47, 48, 49, 63, 64])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_ranks(eng, dt, rank, T, cols, group):
    # two projections with an adapter, the second without one; the low rank's share is of the
    # base's size, so that a rank that is lost or taken twice is far out of the bounds
    dt, g = DTYPES[dt], torch.Generator().manual_seed(100 * rank + T)
    x = torch.randn(T, cols, generator=g).to(dt)
    projs, refs = [], []
    for i, out in enumerate((132, 20, 64)):
        w, kw = qh.Weights(out, cols, group, False, 50 + i), {}
        if i != 1:
            kw = {"a": torch.randn(cols, rank, generator=g), "b": torch.randn(rank, out, generator=g), "scaling": 0.75 - i}
        packed = eng.quant_pack(w.numbers.cuda(), w.s.cuda())
        projs.append({"w": packed, "out": out, **{k: v.cuda() if k in "ab" else v for k, v in kw.items()}})
        refs.append(qh.project_ref(x, w, dt, **kw))
    for i, (y, ref) in enumerate(zip(eng.proj_quant_forward(x.cuda(), projs, rank=rank, group=group), refs)):
        ch.check(f"y{i}", y, *ref)
