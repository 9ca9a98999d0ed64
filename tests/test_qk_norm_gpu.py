"""Per-head norms of queries and keys with the rotation (glacier_rmsnorm_qk_*),
through the Python front end, against their definition in 64 bits."""
import pytest

import glacier_attn as ga

torch = pytest.importorskip("torch")
import cache_harness as ch  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


def _inputs(T, hq, hkv, d, dtype, seed, far):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = (3.0 * n(T, h, d) for h in (hq, hkv))
    dq, dk = (0.1 * n(T, h, d) for h in (hq, hkv))
    wq, wk = (1.0 + 0.3 * n(d) for _ in range(2))
    pos = torch.randint(0, far, (T,), generator=g, dtype=torch.int32)
    dev = lambda x: x.to("cuda", dtype)  # noqa: E731
    return dev(q), dev(k), dev(dq), dev(dk), wq.cuda(), wk.cuda(), pos


SHAPES = [  # T, hq, hkv, D, theta, positions below
    (1, 1, 1, 8, 1e4, 3),
    (1, 28, 4, 128, 1e6, 131072),
    (3, 14, 2, 64, 1e6, 100),
    (5, 5, 1, 80, 5e5, 70000),
    (7, 8, 2, 256, 1e6, 4096),
    (33, 16, 16, 40, 1e4, 512),
    (65, 3, 3, 72, 1e4, 2 ** 30),
    (130, 32, 8, 128, 5e5, 4096),
    (257, 7, 1, 96, None, 9),
    (1, 130, 1, 32, 1e4, 77),
    (9000, 2, 1, 16, 1e4, 9000),
    (6, 2, 5, 48, 1e4, 300),
]


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("T,hq,hkv,d,theta,far", SHAPES)
def test_forward(eng, T, hq, hkv, d, theta, far, dt):
    q, k, _, _, wq, wk, pos = _inputs(T, hq, hkv, d, DTYPES[dt], 1, far)
    yq, yk = eng.qk_norm_forward(q, k, wq, wk, EPS, rope_freq_base=theta, positions=pos.cuda())
    for name, x, w, y in (("q", q, wq, yq), ("k", k, wk, yk)):
        ch.check(name, y, *ch.norm_ref(x, w, pos, theta, EPS, DTYPES[dt]))
    # in place, and positions 0 .. T - 1 without an array
    a, b = q.clone(), k.clone()
    eng.qk_norm_forward(a, b, wq, wk, EPS, rope_freq_base=theta, q_out=a, k_out=b)
    count = torch.arange(T)
    ch.check("q in place", a, *ch.norm_ref(q, wq, count, theta, EPS, DTYPES[dt]))
    ch.check("k in place", b, *ch.norm_ref(k, wk, count, theta, EPS, DTYPES[dt]))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("T,hq,hkv,d,theta,far", SHAPES)
def test_backward(eng, T, hq, hkv, d, theta, far, dt):
    q, k, gq, gk, wq, wk, pos = _inputs(T, hq, hkv, d, DTYPES[dt], 2, far)
    start = torch.linspace(-1, 1, d, device="cuda")
    dwq, dwk = start.clone(), start.clone()
    dq, dk = eng.qk_norm_backward(gq, gk, q, k, wq, wk, EPS, rope_freq_base=theta,
                                  positions=pos.cuda(), dq_weight=dwq, dk_weight=dwk)
    refs = {}
    for name, dy, x, w, dx, dw in (("q", gq, q, wq, dq, dwq), ("k", gk, k, wk, dk, dwk)):
        rx, bx, rw, bw = refs[name] = ch.norm_grad_ref(dy, x, w, pos, theta, EPS, DTYPES[dt])
        ch.check(f"d{name}", dx, rx, bx)
        full = rw + start.double().cpu()  # accumulated: one more addition
        ch.check(f"d{name}_weight", dw, full, bw + ch.F * (full.abs() + rw.abs()))
    # one weight gradient only, none, and in place: the same input gradients
    only = start.clone()
    a, b = gq.clone(), gk.clone()
    eng.qk_norm_backward(a, b, q, k, wq, wk, EPS, rope_freq_base=theta, positions=pos.cuda(), dq=a,
                         dk=b, dk_weight=only)
    assert torch.equal(a, dq) and torch.equal(b, dk) and torch.equal(only, dwk)
    c, e = eng.qk_norm_backward(gq, gk, q, k, wq, wk, EPS, rope_freq_base=theta, positions=pos.cuda())
    assert torch.equal(c, dq) and torch.equal(e, dk)


def test_gradient_against_differences(eng):
    # L = sum dy . y in fp32 rows, central differences of the 64-bit definition
    q, k, gq, gk, wq, wk, pos = _inputs(2, 2, 1, 16, torch.float32, 3, 50)
    dwq = torch.zeros(16, device="cuda")
    dq, _ = eng.qk_norm_backward(gq, gk, q, k, wq, wk, EPS, rope_freq_base=1e4, positions=pos.cuda(),
                                 dq_weight=dwq)

    def loss(x, w):
        return float((ch.norm_ref(x, w, pos, 1e4, EPS, torch.float32)[0] * gq.double().cpu()).sum())

    step = 1e-6  # 64-bit differences: truncation ~step^2, cancellation ~1e-16 / step
    for at in ((0, 0, 0), (0, 1, 7), (1, 0, 15), (1, 1, 8)):
        up, down = q.double().cpu().clone(), q.double().cpu().clone()
        up[at] += step
        down[at] -= step
        slope = (loss(up, wq) - loss(down, wq)) / (2 * step)
        assert abs(float(dq[at]) - slope) <= 1e-5 * (abs(slope) + float(dq.abs().max()))
    for i in (0, 9):
        up, down = wq.double().cpu().clone(), wq.double().cpu().clone()
        up[i] += step
        down[i] -= step
        slope = (loss(q, up) - loss(q, down)) / (2 * step)
        assert abs(float(dwq[i]) - slope) <= 1e-5 * (abs(slope) + float(dwq.abs().max()))


def test_zero_rows_and_zero_tokens(eng):
    # an all-zero head: r = eps^-1/2 is finite, the row stays zero
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(2, 1, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda")
    yq, yk = eng.qk_norm_forward(q, k, w, w, EPS, rope_freq_base=1e4)
    assert not yq.any() and not yk.any()
    e = torch.empty(0, 4, 64, device="cuda")
    yq, yk = eng.qk_norm_forward(e, torch.empty(0, 1, 64, device="cuda"), w, w, EPS)
    assert yq.shape == (0, 4, 64) and yk.shape == (0, 1, 64)


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_tiny_rows_without_eps(eng, dt):
    # 1 / sqrt(mean x^2) is 1e14: its cube leaves fp32, the gradients do not
    q, k, gq, gk, wq, wk, pos = _inputs(5, 6, 2, 64, DTYPES[dt], 8, 100)
    q, k = q * 1e-14, k * 1e-14
    yq, yk = eng.qk_norm_forward(q, k, wq, wk, 0.0, rope_freq_base=1e4, positions=pos.cuda())
    dwq, dwk = torch.zeros_like(wq), torch.zeros_like(wk)
    dq, dk = eng.qk_norm_backward(gq, gk, q, k, wq, wk, 0.0, rope_freq_base=1e4, positions=pos.cuda(),
                                  dq_weight=dwq, dk_weight=dwk)
    for name, x, w, y, g, dx, dw in (("q", q, wq, yq, gq, dq, dwq), ("k", k, wk, yk, gk, dk, dwk)):
        ch.check(name, y, *ch.norm_ref(x, w, pos, 1e4, 0.0, DTYPES[dt]))
        rx, bx, rw, bw = ch.norm_grad_ref(g, x, w, pos, 1e4, 0.0, DTYPES[dt])
        ch.check(f"d{name}", dx, rx, bx)
        ch.check(f"d{name}_weight", dw, rw, bw)


def test_repeatable_and_captured(eng):
    q, k, gq, gk, wq, wk, pos = _inputs(700, 28, 4, 128, torch.bfloat16, 4, 4096)
    pos = pos.cuda()
    yq, yk = torch.empty_like(q), torch.empty_like(k)
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dwq, dwk = torch.zeros_like(wq), torch.zeros_like(wk)

    def step():
        dwq.zero_()
        dwk.zero_()
        eng.qk_norm_forward(q, k, wq, wk, EPS, rope_freq_base=1e6, positions=pos, q_out=yq, k_out=yk)
        eng.qk_norm_backward(gq, gk, q, k, wq, wk, EPS, rope_freq_base=1e6, positions=pos, dq=dq, dk=dk,
                             dq_weight=dwq, dk_weight=dwk)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        new = _inputs(700, 28, 4, 128, torch.bfloat16, 10 + seed, 4096)
        for to, x in zip((q, k, gq, gk, wq, wk, pos), new):
            to.copy_(x)
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (yq, yk, dq, dk, dwq, dwk)]
        for t in (yq, yk, dq, dk):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, (yq, yk, dq, dk, dwq, dwk)))


def test_offsets_past_32_bits(eng):
    # rows past 2^31 elements: the first and last tokens of one call
    T, hq, hkv, d = 2 ** 31 // (30 * 128) + 100, 30, 2, 128
    q = torch.zeros(T, hq, d, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(T, hkv, d, device="cuda", dtype=torch.bfloat16)
    ends = torch.tensor([0, 1, T - 2, T - 1])
    sq, sk, gq, gk, wq, wk, _ = _inputs(4, hq, hkv, d, torch.bfloat16, 6, 9)
    q[ends.cuda()], k[ends.cuda()] = sq, sk
    eng.qk_norm_forward(q, k, wq, wk, EPS, rope_freq_base=1e6, q_out=q, k_out=k)
    for name, x, w, y in (("q", sq, wq, q), ("k", sk, wk, k)):
        ch.check(name, y[ends.cuda()], *ch.norm_ref(x, w, ends, 1e6, EPS, torch.bfloat16))
    dy, dyk = torch.zeros_like(q), torch.zeros_like(k)
    q.zero_()
    k.zero_()
    q[ends.cuda()], k[ends.cuda()], dy[ends.cuda()], dyk[ends.cuda()] = sq, sk, gq, gk
    dwq, dwk = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
    eng.qk_norm_backward(dy, dyk, q, k, wq, wk, EPS, rope_freq_base=1e6, dq=dy, dk=dyk, dq_weight=dwq,
                         dk_weight=dwk)
    for name, g, x, w, dx, dw in (("q", gq, sq, wq, dy, dwq), ("k", gk, sk, wk, dyk, dwk)):
        rx, bx, rw, bw = ch.norm_grad_ref(g, x, w, ends, 1e6, EPS, torch.bfloat16)
        ch.check(f"d{name}", dx[ends.cuda()], rx, bx)
        ch.check(f"d{name}_weight", dw, rw, bw)
