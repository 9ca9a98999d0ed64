"""Products with 4-bit weights (glacier_proj_quant_*), through the Python front end,
against their definition in 64 bits; and a step of an answer in 4 bits as a whole."""
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


def _pack(eng, w):
    return eng.quant_pack(w.numbers.cuda(), w.s.cuda(), None if w.o is None else w.o.cuda())


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("out,cols,group", [(16, 128, 32), (4, 32, 32), (100, 320, 64), (36, 1120, 32), (256, 896, 128)])
def test_pack(eng, out, cols, group, offsets):
    w = qh.Weights(out, cols, group, offsets, 3)
    packed = _pack(eng, w)
    assert packed.numel() == eng.quant_bytes(out, cols, group, offsets)
    assert torch.equal(packed.cpu(), w.packed())


CASES = {  # tokens, in, outs, group, offsets, rank, bias
    "one": (1, 32, (4,), 32, False, 0, False),
    "token": (1, 896, (896, 128, 128), 32, False, 16, True),
    "token_wide": (1, 3584, (512,), 128, True, 0, False),
    "token_deep": (1, 4864, (20,), 64, True, 64, True),
    "three": (3, 320, (100, 36), 32, True, 8, False),
    "sixteen": (16, 1536, (1000,), 64, False, 0, True),
    "seventeen": (17, 1120, (64, 16, 52, 4), 32, False, 5, False),
    "thirty_two": (32, 256, (2000,), 128, False, 1, True),
    "forty": (40, 2048, (528,), 128, True, 16, True),
    "prompt": (150, 896, (896, 128, 128), 32, True, 16, True),
    "many": (515, 160, (272,), 32, False, 0, False),
}


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("name", sorted(CASES))
def test_products(eng, name, dt):
    T, cols, outs, group, offsets, rank, bias = CASES[name]
    dt, g = DTYPES[dt], torch.Generator().manual_seed(8)
    x = torch.randn(T, cols, generator=g).to(dt)
    projs, refs = [], []
    for i, out in enumerate(outs):
        w = qh.Weights(out, cols, group, offsets, 40 + i)
        pr = {"w": _pack(eng, w), "out": out}
        kw = {}
        if bias and i != 1:
            kw["bias"] = torch.randn(out, generator=g)
        if rank and i != 2:  # (a projection without an adapter among others)
            kw["a"], kw["b"], kw["scaling"] = torch.randn(cols, rank, generator=g), torch.randn(rank, out, generator=g), -1.5
        for k, v in kw.items():
            pr[k] = v.cuda() if isinstance(v, torch.Tensor) else v
        projs.append(pr)
        refs.append(qh.project_ref(x, w, dt, **kw))
    ys = eng.proj_quant_forward(x.cuda(), projs, rank=rank, group=group, mins=offsets)
    for i, (y, ref) in enumerate(zip(ys, refs)):
        ch.check(f"y{i}", y, *ref)
    again = eng.proj_quant_forward(x.cuda(), projs, rank=rank, group=group, mins=offsets)
    assert all(torch.equal(a, b) for a, b in zip(ys, again))


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_outputs_and_their_neighbours(eng, dt):
    # given outputs are written, and nothing beside them
    dt, w = DTYPES[dt], qh.Weights(36, 128, 32, False, 5)
    x = torch.randn(19, 128).to(dt).cuda()
    whole = torch.full((840,), 7.0, dtype=dt, device="cuda")
    y = whole[80:80 + 19 * 36].view(19, 36)
    pr = {"w": _pack(eng, w), "out": 36, "y": y}
    assert eng.proj_quant_forward(x, [pr])[0] is y
    ch.check("y", y, *qh.project_ref(x.cpu(), w, dt))
    assert (whole[:80] == 7.0).all() and (whole[80 + 19 * 36:] == 7.0).all()


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_a_token_that_is_not_finite_stays_alone(eng, dt):
    dt, w = DTYPES[dt], qh.Weights(48, 160, 32, False, 6)
    x = torch.randn(20, 160).to(dt).cuda()
    want, = eng.proj_quant_forward(x, [{"w": _pack(eng, w), "out": 48}])
    x[3, 159], x[17, 0] = math.nan, math.inf
    got, = eng.proj_quant_forward(x, [{"w": _pack(eng, w), "out": 48}])
    fine = torch.ones(20, dtype=torch.bool, device="cuda")
    fine[[3, 17]] = False
    assert torch.equal(got[fine], want[fine]) and got[3].isnan().all() and not torch.isfinite(got[17]).any()


def test_no_tokens(eng):
    w = qh.Weights(16, 64, 32, False, 7)
    y, = eng.proj_quant_forward(torch.zeros(0, 64, device="cuda"), [{"w": _pack(eng, w), "out": 16}])
    assert y.shape == (0, 16)


def test_quantise_rows(eng):
    w = torch.randn(40, 256)
    w[3, 32:64] = 0.0
    numbers, scales = ga.quantise_rows(w, 32)
    n = torch.stack([numbers & 15, numbers >> 4], -1).flatten(1).double() - 8
    back = (n.unflatten(1, (-1, 32)) * scales.double()[..., None]).flatten(1)
    step = scales.double().abs().repeat_interleave(32, 1)
    # half a step and, next to the element that n = 0 stands for, one (7 against 8)
    assert ((back - w).abs() <= 1.01 * step).all() and ((back - w).abs() <= 0.51 * step).double().mean() > 0.98
    x = torch.randn(2, 256, device="cuda", dtype=torch.bfloat16)
    y, = eng.proj_quant_forward(x, [{"w": eng.quant_pack(numbers.cuda(), scales.cuda()), "out": 40}])
    want = x.cpu().double() @ back.t()
    assert float((y.cpu().double() - want).norm() / want.norm()) < 2.0 ** -8


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_captured_products(eng, dt):
    # two graphs of one engine, with adapters (a workspace each), side by side
    dt, sets, streams = DTYPES[dt], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed, T in ((1, 1), (2, 20)):
        g = torch.Generator().manual_seed(seed)
        w = qh.Weights(512, 896, 32, False, seed)
        pr = {"w": _pack(eng, w), "out": 512, "a": torch.randn(896, 16, generator=g).cuda(),
              "b": torch.randn(16, 512, generator=g).cuda(), "scaling": 2.0}
        sets.append((torch.randn(T, 896, generator=g).to(dt).cuda(), pr))
    graphs, outs = [], []
    for (x, pr), stream in zip(sets, streams):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(eng.proj_quant_forward(x, [dict(pr)], rank=16)[0])
        graphs.append(graph)
    for turn in range(4):
        for x, _ in sets:
            x.mul_(-1.25)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (x, pr), y in zip(sets, outs):
            assert torch.equal(y, eng.proj_quant_forward(x, [dict(pr)], rank=16)[0])


def _step(eng, x, layer, index, d, lens):
    """One layer's attention part of a step: q, k, v, the cache, O."""
    T, hq, hkv = x.shape[0], layer["hq"], layer["hkv"]
    q, k, v = eng.proj_quant_forward(x, [dict(p) for p in layer["qkv"]], rank=8)
    q = eng.qcache_append(k.view(T, hkv, d), v.view(T, hkv, d), *index[:3], lens, index[4], rope_freq_base=1e4,
                          q=q.view(T, hq, d))
    out, _ = eng.qcache_forward(q, *index[:3], lens, index[4], max_new=1, max_kv=64)
    return eng.proj_quant_forward(out.view(T, hq * d), [dict(layer["o"])], rank=8)[0]


def test_an_answer_in_4_bits(eng):
    # a prompt in one chunk, then tokens: the projections, the cache and the attention
    # together, eager and as a replayed graph, against the same step in 64 bits
    hq, hkv, d, width, seqs = 4, 2, 64, 256, 3
    g = torch.Generator().manual_seed(77)

    def adapter(rows, cols):
        return {"a": torch.randn(cols, 8, generator=g) / 16, "b": torch.randn(8, rows, generator=g) / 4, "scaling": 2.0}

    ws, layer = {}, {"hq": hq, "hkv": hkv, "qkv": []}
    for name, rows, cols in (("q", hq * d, width), ("k", hkv * d, width), ("v", hkv * d, width), ("o", width, hq * d)):
        w, ad = qh.Weights(rows, cols, 32, False, ord(name)), adapter(rows, cols)
        ws[name] = (w, ad)
        pr = {"w": _pack(eng, w), "out": rows, "a": ad["a"].cuda(), "b": ad["b"].cuda(), "scaling": ad["scaling"]}
        if name == "o":
            layer["o"] = pr
        else:
            layer["qkv"].append(pr)
    pages = torch.full((2, 12, hkv, ga.quant_page_bytes(16, d)), 255, dtype=torch.uint8, device="cuda")
    table = torch.randperm(12, generator=g).view(3, 4).int().cuda()
    chunk = [20, 1, 33]
    cu = torch.tensor([0, 20, 21, 54], dtype=torch.int32, device="cuda")
    one = torch.arange(4, dtype=torch.int32, device="cuda")
    lens = torch.tensor(chunk, dtype=torch.int32, device="cuda")
    x0 = torch.randn(54, width, generator=g).bfloat16()
    steps = [torch.randn(seqs, width, generator=g).bfloat16() for _ in range(5)]

    got = [_step(eng, x0.cuda(), layer, (pages[0], pages[1], cu, lens, table), d, lens)]
    x = steps[0].cuda()
    index = (pages[0], pages[1], one, lens, table)
    lens += 1
    got.append(_step(eng, x, layer, index, d, lens))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        y = _step(eng, x, layer, index, d, lens)
    for s in steps[1:]:
        x.copy_(s.cuda())
        lens += 1
        graph.replay()
        got.append(y.clone())

    # the same in 64 bits, with the roundings to bf16 that the calls' types ask for
    def product(x, name):
        w, ad = ws[name]
        return (x.double() @ w.w.t() + 2.0 * (x.double() @ ad["a"].double()) @ ad["b"].double()).bfloat16()

    cached = [([], []) for _ in chunk]
    total = [0] * seqs
    for turn, x in enumerate([x0] + steps):
        new = chunk if turn == 0 else [1] * seqs
        pos = torch.cat([torch.arange(total[b], total[b] + new[b]) for b in range(seqs)])
        q, k, v = (product(x, n).view(len(x), -1, d) for n in "qkv")
        q = ch.rotate(q.double(), pos, 1e4).bfloat16().double()
        k, v = qh.held(ch.rotate(k.double(), pos, 1e4).float()), qh.held(v)
        out, t = torch.zeros(len(x), hq, d, dtype=torch.float64), 0
        for b in range(seqs):
            cached[b][0].append(k[t:t + new[b]]), cached[b][1].append(v[t:t + new[b]])
            ks, vs = torch.cat(cached[b][0]), torch.cat(cached[b][1])
            see = torch.arange(len(ks))[None] <= torch.arange(total[b], total[b] + new[b])[:, None]
            for h in range(hq):
                z = (q[t:t + new[b], h] @ ks[:, h // 2].t() / 8.0).masked_fill(~see, -math.inf)
                out[t:t + new[b], h] = torch.softmax(z, -1) @ vs[:, h // 2]
            t += new[b]
            total[b] += new[b]
        want = product(out.bfloat16().view(len(x), -1), "o").double()
        # (a rounding of q, k or v to bf16 that falls the other way may move a number of
        # the cache by a step: the norm is looked at, and few of them move)
        assert float((got[turn].cpu().double() - want).norm() / want.norm()) < 2.0 ** -6


# tokens, outputs: by their number of tiles of 16 by 16 each takes another kernel
SHAPES = {"deep": (5, 36), "few": (33, 132), "hundreds": (130, 1000), "thousand": (300, 1300), "thousands": (300, 4100),
          "most": (1300, 8200)}


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("group,offsets", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_shapes_and_groups(eng, shape, group, offsets, dt):
    (T, out), dt, g = SHAPES[shape], DTYPES[dt], torch.Generator().manual_seed(12)
    cols = 8192 + group if shape == "deep" else {32: 352, 64: 320, 128: 384}[group]
    w = qh.Weights(out, cols, group, offsets, 13)
    x = torch.randn(T, cols, generator=g).to(dt)
    kw = {"a": torch.randn(cols, 7, generator=g), "b": torch.randn(7, out, generator=g), "scaling": 0.5,
          "bias": torch.randn(out, generator=g)}
    pr = {"w": _pack(eng, w), "out": out, **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}}
    y, = eng.proj_quant_forward(x.cuda(), [pr], rank=7, group=group, mins=offsets)
    ch.check("y", y, *qh.project_ref(x, w, dt, **kw))


def test_fp32_of_every_size(eng):
    # x down to 2^-100 and up to where eight times it is still finite: three bf16 terms
    # hold all of it
    w, g = qh.Weights(64, 256, 64, False, 14), torch.Generator().manual_seed(15)
    x = torch.randn(9, 256, generator=g)
    x *= torch.tensor([2.0 ** e for e in (-100, -60, -20, 0, 20, 60, 100, 1, 2)])[:, None]
    x[7:] = 0.0
    x[7, 5], x[8, 200] = torch.finfo(torch.float32).max / 16, -torch.finfo(torch.float32).max / 16
    y, = eng.proj_quant_forward(x.cuda(), [{"w": _pack(eng, w), "out": 64}], group=64)
    ch.check("y", y, *qh.project_ref(x, w, torch.float32))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("T", [3001, 50001])
def test_many_tokens_of_few_outputs(eng, dt, T):
    dt, w = DTYPES[dt], qh.Weights(20, 96, 32, True, 16)
    x = torch.randn(T, 96, generator=torch.Generator().manual_seed(17)).to(dt)
    kw = {"a": torch.randn(96, 3), "b": torch.randn(3, 20), "scaling": 1.0}
    pr = {"w": _pack(eng, w), "out": 20, "a": kw["a"].cuda(), "b": kw["b"].cuda(), "scaling": 1.0}
    y, = eng.proj_quant_forward(x.cuda(), [pr], rank=3, mins=True)
    ch.check("y", y, *qh.project_ref(x, w, dt, **kw))


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_one_weight_in_two_projections(eng, dt):
    # one W, A and B twice, and tensors that begin inside others
    dt, w = DTYPES[dt], qh.Weights(64, 128, 64, False, 18)
    packed, rows = _pack(eng, w), torch.randn(7, 128).to(dt).cuda()
    a, b = torch.randn(128, 9).cuda(), torch.randn(9, 64).cuda()
    pr = {"w": packed, "out": 64, "a": a, "b": b, "scaling": 0.25}
    one, two = eng.proj_quant_forward(rows[2:], [dict(pr), dict(pr, scaling=-0.25)], rank=9, group=64)
    for y, s in ((one, 0.25), (two, -0.25)):
        ch.check("y", y, *qh.project_ref(rows[2:].cpu(), w, dt, a=a.cpu(), b=b.cpu(), scaling=s))
