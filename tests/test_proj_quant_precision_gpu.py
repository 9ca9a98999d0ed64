"""How near the products with 4-bit weights come to 64 bits, where the worst case's bounds say
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
F = ch.F
GROUPS = [(g, o) for g in (32, 64, 128) for o in (False, True)]
# tokens, outputs: by their number of tiles of 16 by 16 each takes another kernel
SHAPES = {"few": (33, 132), "hundreds": (130, 1000), "thousand": (300, 1300), "thousands": (300, 4100),
          "most": (1300, 8200)}


@pytest.fixture(scope="module")
def eng():
    assert torch.cuda.is_available(), "GPU tests need a ROCm GPU"
    e = ga.GpuAttentionEngine(0, ga.PREC_BF16)
    yield e
    e.close()


def _rms(x):
    return float(x.double().square().mean().sqrt())


def _products(eng, x, w, group, offsets):
    packed = eng.quant_pack(w.numbers.cuda(), w.s.cuda(), None if w.o is None else w.o.cuda())
    return eng.proj_quant_forward(x.cuda(), [{"w": packed, "out": w.out}], group=group, mins=offsets)[0].cpu().double()


@pytest.mark.parametrize("group,offsets", GROUPS)
@pytest.mark.parametrize("shape", ["token", "deep"] + sorted(SHAPES))
def test_one_value_a_token_keeps_its_24_bits(eng, shape, group, offsets):
    # Token t has one value, in column t (and then in column t + T, ..): y = (n - 8) s x + o x.
    # The products of three terms are exact and are added smallest first, 2 F at most; s d, o d0
    # and their sum F each, the offsets' product 2 F more: within 6 F of both terms' sizes.
    g = torch.Generator().manual_seed(21)
    T, out = {"token": (1, 20), "deep": (5, 36), **SHAPES}[shape]
    cols = 8192 + group if shape == "deep" else {32: 352, 64: 320, 128: 384}[group]
    w = qh.Weights(out, cols, group, offsets, 22)
    packed = eng.quant_pack(w.numbers.cuda(), w.s.cuda(), None if w.o is None else w.o.cuda())
    whole = (w.n - 8).double() * w.s.double().repeat_interleave(group, 1)
    passes = -(-cols // T)
    for i in range(passes) if passes <= 400 else torch.randperm(passes, generator=g)[:60].tolist():
        at = (torch.arange(T) + i * T) % cols
        value = (1.0 + torch.rand(T, generator=g)) * torch.exp2(torch.randint(-40, 40, (T,), generator=g).float())
        x = torch.zeros(T, cols)
        x[torch.arange(T), at] = value
        y, = eng.proj_quant_forward(x.cuda(), [{"w": packed, "out": out}], group=group, mins=offsets)
        a, b = whole[:, at].t() * value.double()[:, None], w.off[:, at].t() * value.double()[:, None]
        ch.check("y", y, a + b, 6 * F * (a.abs() + b.abs()))


@pytest.mark.parametrize("group,offsets", GROUPS)
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_fp32_products_as_a_whole(eng, shape, group, offsets):
    # Sums of `cols` random terms of length L (their root of squares).  Of the groups' sums each
    # addition is off by F / sqrt(3) of a partial sum of at most about L, the parts of a group by
    # as much of its own: a few F L; were matrix instructions to cut, three of a group's length
    # each, all to one side, 10 F L.  Without the third term: 165 F L.
    T, out = SHAPES[shape]
    cols = {32: 352, 64: 320, 128: 384}[group]
    w = qh.Weights(out, cols, group, offsets, 23)
    x = torch.randn(T, cols, generator=torch.Generator().manual_seed(24))
    y = _products(eng, x, w, group, offsets)
    length = (x.double().square() @ (w.w.square() + w.off.square()).t()).sqrt()
    assert _rms((y - x.double() @ w.w.t()) / length) <= 16 * F


@pytest.mark.parametrize("group,offsets", GROUPS)
@pytest.mark.parametrize("shape", ["deep"] + sorted(SHAPES))
def test_bf16_products_that_cancel(eng, shape, group, offsets):
    # The second half's columns are the first half's negated, in another order in each group:
    # every product is zero, and what comes out is the sums' own error, hardly rounded.  Of a
    # group the sums pass through 136 times a partial sum of x, about 136 sqrt(group) rms(x), at
    # most 16 roundings of F / sqrt(3) of that, once scaled: 2.4 U with U = F 136 sqrt(group)
    # rms(x) |s|, |s| the root of the groups' squares; of the offsets a few F of their own terms
    # and of the sums.  8 U: two bits fewer anywhere would show.
    T, out = {"deep": (5, 36), **SHAPES}[shape]
    half = 4096 + group if shape == "deep" else {32: 192, 64: 192, 128: 256}[group]
    g = torch.Generator().manual_seed(25)
    w = qh.Weights(out, 2 * half, group, offsets, 26)
    order = torch.cat([torch.randperm(group, generator=g) + i for i in range(0, half, group)])
    w.n[:, half:] = w.n[:, :half][:, order]
    w.numbers = (w.n[:, 0::2] | w.n[:, 1::2] << 4).to(torch.uint8)
    w.s[:, half // group:] = w.s[:, :half // group]
    if offsets:
        w.o[:, half // group:] = w.o[:, :half // group]
    x = torch.randn(T, 2 * half, generator=g).bfloat16()
    x[:, half:] = -x[:, :half][:, order]
    y = _products(eng, x, w, group, offsets)
    unit = 136 * math.sqrt(group) * w.s.double().square().sum(1).sqrt()
    if offsets:
        unit = unit + 4 * math.sqrt(2 * half) * w.o.double().abs().amax(1)
    # (the sums of the groups: rounded F / sqrt(3) of a partial sum each)
    chain = math.sqrt(2 * half / group) * (x.double().square() @ ((w.n - 8).double()
                                           * w.s.double().repeat_interleave(group, 1)).square().t()).sqrt()
    assert _rms(y / (unit * _rms(x) + chain)) <= 8 * F
