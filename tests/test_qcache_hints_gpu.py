"""Attention over a 4-bit cache where sequences are longer than the call's max_kv said."""
import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402
import quant_harness as qh  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}

# Several tokens of one sequence among single ones, most keys just past the hint: a sequence's
# earlier tile has more splits than its last one (1024 keys: 4 of 256, 1025: 3 of 384; 2048: 8,
# 2049: 6).
BATCHES = {
    "three": ([(3, 1025), (1, 1000)], 8, 1, 64, 1024),
    "four": ([(4, 2049)] + [(1, 1900)] * 7, 28, 4, 128, 2048),
    "last": ([(1, 700), (1, 3), (0, 90), (1, 1100), (1, 64), (5, 1026)], 6, 1, 96, 1024),
    "two_long": ([(1, 500), (6, 1283), (1, 2600), (5, 1026)] + [(1, 300 + i) for i in range(9)], 7, 1, 64, 1024),
}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_sequences_longer_than_the_hint(eng, name, dt):
    seqs, hq, hkv, d, hint = BATCHES[name]
    p = qh.QPaged(seqs, hq, hkv, d, 16, DTYPES[dt], 61)
    ref = qh.attend_ref(p)
    for kw in (dict(max_new=1, max_kv=hint), dict(max_kv=hint), dict(max_kv=hint - 300)):
        out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True, **kw)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])


def test_a_captured_step_whose_sequence_grows(eng):
    # captured with the lengths of its time, replayed while the first sequence drafts its way past them
    p = qh.QPaged([(3, 1040), (1, 1000)], 8, 1, 64, 16, torch.bfloat16, 62)
    q, (k, v, cu, lens, table) = p.q.cuda(), p.arrays()
    lens -= torch.tensor([16, 0], dtype=torch.int32, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out, lse = eng.qcache_forward(q, k, v, cu, lens, table, max_kv=1024, save=True)
    for grown in (1024, 1025, 1026, 1040):
        lens[0] = grown
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        now = qh.QPaged([(3, 1040), (1, 1000)], 8, 1, 64, 16, torch.bfloat16, 62, device="cpu")
        now.seqs = [(3, grown), (1, 1000)]
        now.k[0], now.v[0], now.steps[0] = now.k[0][:grown], now.v[0][:grown], now.steps[0][:grown]
        ref = qh.attend_ref(now)
        ch.check("out", out, ref[0], ref[1])
        ch.check("lse", lse, ref[2], ref[3])
