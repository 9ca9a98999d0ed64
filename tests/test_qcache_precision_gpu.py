"""How near the attention over a 4-bit cache comes to 64 bits, where the worst case's bounds say
little: values whose low bits the result has to show, and root mean squares of random ones.

F is half a step of fp32.  A matrix instruction's sum is counted as off by up to 2 F of it.
Of three bf16 terms of x the third holds its last eight bits: without it a value is off by up to
500 F (terms cut) or 128 F (rounded), and a sum of random terms by 165 F or 37 F of their length."""
import math

import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402
import quant_harness as qh  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
F = ch.F
HEADS = [32, 64, 96, 128, 192, 256]


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


def _rms(x):
    return float(x.double().square().mean().sqrt())


def _first_tokens(d, hq, dt, seed, q_of):
    """32 sequences of one token each: a row's log-sum-exp is its one key's score."""
    def change(p):
        p.q = q_of(p.q.shape, torch.Generator().manual_seed(seed))

    return qh.QPaged([(1, 1)] * 32, hq, 2, d, 16, dt, seed, change=change)


@pytest.mark.parametrize("hq", [8, 32])
@pytest.mark.parametrize("d", HEADS)
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_scores_of_one_column(eng, dt, d, hq):
    # A query of one value, every column in turn: lse = q (n - 8) s / sqrt(D).  The product is
    # exact but for 2 F, s d F, the scale's constant, root and division F each and its product F,
    # the change of base F and its constant F: 9 F of the score, and 12 with what they add up to.
    def q_of(shape, g):
        q = torch.zeros(shape)
        value = (1.0 + torch.rand(shape[:2], generator=g)) * torch.exp2(torch.randint(-8, 8, shape[:2], generator=g).float())
        at = torch.arange(shape[0] * shape[1]).view(shape[:2]) % d
        return q.scatter(2, at[..., None], value[..., None])

    p = _first_tokens(d, hq, DTYPES[dt], 27, q_of)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    want = torch.stack([torch.stack([(p.q[b, h].double() * p.k[b][0, h // (hq // 2)]).sum() / math.sqrt(d)
                                     for b in range(32)]) for h in range(hq)])
    assert (want != 0).double().mean() > 0.8
    ch.check("lse", lse, want, 12 * F * want.abs())
    held = torch.stack([p.v[b][0].repeat_interleave(hq // 2, 0) for b in range(32)])
    assert torch.equal(out.double().cpu(), held)


@pytest.mark.parametrize("d", HEADS)
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_scores_as_a_whole(eng, dt, d):
    # Random queries.  fp32: D terms of length L, each addition off by F / sqrt(3) of a partial sum,
    # a few F L, 10 were matrix instructions to cut; without the third term of q 37 F L.  bf16: of
    # each group the sums pass through 136 times a partial sum of q, 770 rms(q), in at most 5
    # roundings, once scaled: 1.3 U with U = F 136 sqrt(32) rms(q) |s|, |s| the root of the groups'
    # squares; 4 U.
    def q_of(shape, g):
        return torch.randn(shape, generator=g)

    p = _first_tokens(d, 32, DTYPES[dt], 28, q_of)
    _, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    off, unit = [], []
    for b in range(32):
        for h in range(32):
            k, q = p.k[b][0, h // 16], p.q[b, h].double()
            off.append(float(lse[h, b]) - float((q * k).sum()) / math.sqrt(d))
            if dt == "bf16":
                s = p.steps[b][0, h // 16, ::32]
                unit.append(4 * 136 * math.sqrt(32) * float(s.square().sum().sqrt()) / math.sqrt(d))
            else:
                unit.append(16 * float((q * k).square().sum().sqrt()) / math.sqrt(d))
    assert _rms(torch.tensor(off).double() / torch.tensor(unit).double()) <= F


@pytest.mark.parametrize("d", HEADS)
def test_fp32_weights_keep_their_24_bits(eng, d):
    # Two keys: the first zero in all columns, with a V of zeros, the second with a score
    # z = -1 .. 0, so its weight w = exp(z) beside the first one's 1: out = w / (1 + w) v.
    # z: 9 F (above) of at most 1; the exponential 2 F, the sum F, its reciprocal 2 F, products
    # 3 F: within 24 F of out.  Weights in two bf16 terms would be off by up to 120 F.
    def change(p):
        g = torch.Generator().manual_seed(29)
        p.q = torch.randn(p.q.shape, generator=g)
        for b in range(32):
            p.k[b][0], p.v[b][0] = 0.0, 0.0
        for b in range(32):
            for h in range(p.hq):
                at = h // (p.hq // p.hkv)
                k = qh.held(p.k[b][1, at])
                z = float((p.q[b, h].double() * k).sum()) / math.sqrt(d)
                want = -0.05 - 0.9 * float(torch.rand(1, generator=g))
                # (one column only, so that the score is its product alone)
                col = int(torch.argmax(k.abs()))
                p.q[b, h] = 0.0
                p.q[b, h, col] = want * math.sqrt(d) / float(k[col])
                assert math.isfinite(z)

    p = qh.QPaged([(1, 2)] * 32, 16, 2, d, 16, torch.float32, 30, change=change)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    want, total = torch.zeros(32, 16, d, dtype=torch.float64), torch.zeros(16, 32, dtype=torch.float64)
    for b in range(32):
        for h in range(16):
            z = float((p.q[b, h].double() * p.k[b][1, h // 8]).sum()) / math.sqrt(d)
            want[b, h] = math.exp(z) / (1.0 + math.exp(z)) * p.v[b][1, h // 8]
            total[h, b] = math.log1p(math.exp(z))
    ch.check("out", out, want, 24 * F * want.abs())
    # (the sum of the weights F, its logarithm 2 F, the changes of base 3 F, z's share 9 F)
    ch.check("lse", lse, total, 24 * F * total.abs())


@pytest.mark.parametrize("d", HEADS)
def test_fp32_rows_as_a_whole(eng, d):
    # 200 random keys: weights off by the scores' error (a few F, as above, and F |z - max|, six
    # or seven), the exponential's 2 F; sums of w v of length L rounded 20 times: about 10 F L, 30
    # were matrix instructions to cut, all to one side.
    p = qh.QPaged([(4, 200), (1, 190), (30, 150)], 8, 2, d, 16, torch.float32, 31)
    out, lse = eng.qcache_forward(p.q.cuda(), *p.arrays(), save=True)
    got, off, t = out.cpu().double(), [], 0
    for b, (n, kv) in enumerate(p.seqs):
        see = torch.arange(kv)[None] <= torch.arange(kv - n, kv)[:, None]
        for h in range(8):
            k, v = p.k[b][:, h // 4], p.v[b][:, h // 4]
            z = (p.q[t:t + n, h].double() @ k.t() / math.sqrt(d)).masked_fill(~see, -math.inf)
            w = torch.softmax(z, -1)
            off.append(((got[t:t + n, h] - w @ v) / (w.square() @ v.square()).sqrt()).flatten())
        t += n
    assert _rms(torch.cat(off)) <= 32 * F
