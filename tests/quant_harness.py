"""Plain 64-bit forms of the 4-bit cache and the 4-bit weights, with the bounds
that the kernels' results have to keep.  F: half a step of fp32, relative."""
import functools
import math

import torch

import cache_harness as ch

F = ch.F
LARGEST = 2688.0  # of a cache's scales


def groups(d):
    g = -(-d // 32)
    return g + (g in (5, 7))


def quantise(x):
    """x [..., 32] (64 bits): (n - 8, s), both 64 bits, s nan where x is not finite."""
    top, low = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    m = torch.where(top >= -low, top, low) / -8.0
    _, e = torch.frexp(m)
    unit = torch.exp2((e - 5).double())  # five significant bits
    s = (torch.round(m / unit) * unit).clamp(-LARGEST, LARGEST).to(torch.float16).double()
    n = torch.floor(x / s + 0.5).clamp(-8.0, 7.0)
    odd = ~torch.isfinite(x).all(-1, keepdim=True)
    s = torch.where(odd, math.nan, s)
    return torch.where((s == 0) | odd, 0.0, n), s


def parts(x):
    """quantise of x [..., D] by groups of its columns: (n - 8) [..., 32 G], s [..., G]."""
    d = x.shape[-1]
    wide = torch.nn.functional.pad(x.double(), (0, 32 * groups(d) - d))
    n, s = quantise(wide.unflatten(-1, (-1, 32)))
    return n.flatten(-2), s[..., 0]


def held(x):
    """What the cache holds of x [..., D]."""
    n, s = parts(x)
    return (n.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :x.shape[-1]]


@functools.lru_cache(maxsize=None)
def word_places(d, side, row):
    """Of every column of a token at `row` of its page: byte of its number, whether it
    is the byte's upper half; of every group: byte of its scale behind the words."""
    g = groups(d)
    byte, upper, scale = [], [], []
    for col in range(32 * g):
        r, j = divmod(col, 8)
        word = (row * 4 + r % 4) * g + r // 4 if side == "k" else (row // 4 * 4 * g + r) * 4 + row % 4
        bit = 4 * (j // 2) + 16 * (j % 2)
        byte.append(4 * word + bit // 8)
        upper.append(bit % 8 == 4)
    for i in range(g):
        scale.append(2 * (row * g + i) if side == "k" else 2 * ((row // 4 * g + i) * 4 + row % 4))
    return torch.tensor(byte), torch.tensor(upper), torch.tensor(scale)


def put(part, page, d, side, row, n, s):
    """One token's numbers n - 8 [Hkv, 32 G] and scales [Hkv, G] into a page's bytes
    [Hkv, 18 G page] (uint8, CPU)."""
    byte, upper, scale = word_places(d, side, row)
    n = (n + 8).to(torch.uint8)
    part[:, byte.unique()] = 0
    for up in (False, True):
        part[:, byte[upper == up]] |= n[:, upper == up] << (4 if up else 0)
    bits = s.to(torch.float16).view(torch.int16).int() & 0xffff
    behind = 16 * groups(d) * page
    part[:, behind + scale], part[:, behind + scale + 1] = (bits & 255).to(torch.uint8), (bits >> 8).to(torch.uint8)


def take(part, page, d, side, row):
    """put back: (n - 8, s) in 64 bits."""
    byte, upper, scale = word_places(d, side, row)
    n = torch.where(upper, part[:, byte] >> 4, part[:, byte] & 15).double() - 8
    behind = 16 * groups(d) * page
    bits = part[:, behind + scale].int() | part[:, behind + scale + 1].int() << 8
    return n, torch.where(bits > 32767, bits - 65536, bits).to(torch.int16).view(torch.float16).double()


class QPaged(ch.Paged):
    """ch.Paged held in 4 bits: k, v are what the pages hold; rows without a token are
    bytes of ones (scales that are NaN)."""

    def __init__(self, seqs, hq, hkv, d, page, dtype, seed, pad=0, spare=3, device="cuda", columns=0, change=None):
        super().__init__(seqs, hq, hkv, d, page, torch.float32, seed, pad, spare, "cpu", columns)
        if change is not None:
            change(self)
        self.dtype, self.q = dtype, self.q.to(dtype)
        size = 18 * groups(d) * page
        both = torch.full((self.n_pages, 2, hkv, size), 255, dtype=torch.uint8)
        self.steps = []  # |s| of every key's column
        for b, (_, kv) in enumerate(seqs):
            (kn, ks), (vn, vs) = parts(self.k[b]), parts(self.v[b])
            for p in range(kv):
                to = both[self.table[b, p // page]]
                put(to[0], page, d, "k", p % page, kn[p], ks[p])
                put(to[1], page, d, "v", p % page, vn[p], vs[p])
            self.k[b], self.v[b] = held(self.k[b]), held(self.v[b])
            self.steps.append(ks.abs().repeat_interleave(32, -1)[..., :d])
        self.both = both.to(device)
        self.k_pages, self.v_pages = self.both[:, 0], self.both[:, 1]
        self.table, self.cu, self.kv_lens = self.table.to(device), self.cu.to(device), self.kv_lens.to(device)


def attend_ref(p):
    """(out, bound, lse, bound) [T, Hq, D] and [Hq, T] of p's rows over what its pages
    hold, NaN behind the last sequence.

    A score.  fp32: 3 D products of exact terms are added, (3 D + 16) F of the sum of
    their sizes.  bf16: of each group 33 terms are added whose sums stay below 136 + 143
    times sum |q| |s|, in fp32; then up to 8 groups.  Or, where the pages are written
    out first, D products as they are; the larger one counts.
    A weight: twice the score's error, the exponential's few half steps, and in bf16
    the 2^-16 that two bf16 terms leave; one below 2^-126 of the largest is zero (the
    exponential's result is no subnormal), which counts where the largest one's V is
    zero.  V is exact; n weights are added in turn."""
    u, bf = ch.half_step(p.dtype), p.dtype == torch.bfloat16
    q = p.q.double()
    out = torch.full((p.tokens, p.hq, p.d), math.nan, dtype=torch.float64)
    out_b, lse = out.clone(), torch.full((p.hq, p.tokens), math.nan, dtype=torch.float64)
    lse_b = lse.clone()
    t = 0
    for b, (n, kv) in enumerate(p.seqs):
        if n == 0:
            continue
        see = torch.arange(kv)[None, :] <= torch.arange(kv - n, kv)[:, None]
        for h in range(p.hq):
            at = h // (p.hq // p.hkv)
            k, v = p.k[b][:, at], p.v[b][:, at]
            rows = slice(t, t + n)
            z = (q[rows, h] @ k.t() / math.sqrt(p.d)).masked_fill(~see, -math.inf)
            terms = 34 * 279 * p.steps[b][:, at] + 8 * k.abs() if bf else (3 * p.d + 16) * k.abs()
            size = (q[rows, h].abs() @ (terms + (p.d + 8) * k.abs()).t() / math.sqrt(p.d)).masked_fill(~see, 0.0)
            top = z.amax(-1, keepdim=True)
            w = torch.where(see, torch.exp(z - torch.where(top.isinf(), 0.0, top)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            seen_v = torch.where(see.any(0)[:, None], v, 0.0)
            o, a = w @ seen_v, w @ seen_v.abs()
            off = (F * size.amax(-1) + (kv + 64) * F)[:, None]
            out[rows, h] = o
            out_b[rows, h] = u * o.abs() + ((2.0 ** -16 if bf else 0.0) + 4 * off) * a + 2.0 ** -126 * seen_v.abs().sum(0)
            lse[h, rows] = torch.where(total == 0, -math.inf, top + torch.log(torch.where(total == 0, 1.0, total)))[:, 0]
            lse_b[h, rows] = 2 * off[:, 0] + 4 * F * torch.where(lse[h, rows].isinf(), 0.0, lse[h, rows].abs())
        t += n
    return out, out_b, lse, lse_b


class Weights:
    """Random weights [out, in] in 4 bits: numbers and scales as quant_pack takes them."""

    def __init__(self, out, cols, group, offsets, seed):
        g = torch.Generator().manual_seed(seed)
        self.out, self.group = out, group
        self.n = torch.randint(0, 16, (out, cols), generator=g)
        self.s = ((torch.rand(out, cols // group, generator=g) + 0.1) * 0.05
                  * torch.where(torch.rand(out, cols // group, generator=g) < 0.5, -1.0, 1.0)).half()
        self.o = (torch.randn(out, cols // group, generator=g) * 0.05).half() if offsets else None
        self.numbers = (self.n[:, 0::2] | self.n[:, 1::2] << 4).to(torch.uint8)
        self.step = self.s.double().abs().repeat_interleave(group, 1)
        self.off = self.o.double().repeat_interleave(group, 1) if offsets else torch.zeros(out, cols).double()
        self.w = (self.n - 8).double() * self.s.double().repeat_interleave(group, 1) + self.off

    def packed(self):
        """The documented layout, on the CPU."""
        out, cols = self.n.shape
        rows, wide = -(-out // 16) * 16, -(-cols // 128) * 128
        n = torch.full((rows, wide), 8)
        n[:out, :cols] = self.n
        tiles, blocks, per = rows // 16, wide // 128, 128 // self.group
        words = torch.zeros(tiles, blocks, 64, 4, dtype=torch.int64)
        for entry in range(64):
            c, r = divmod(entry, 16)
            for i in range(4):
                for e in range(8):
                    at = n[r::16, 32 * i + 8 * c + e::128]
                    words[:, :, entry, i] |= at << (4 * (e // 2) + 16 * (e % 2))
        found = [words.view(-1).to(torch.int32).view(torch.uint8)]
        for t in (self.s, self.o):
            if t is not None:
                full = torch.zeros(rows, blocks * per, dtype=torch.float16)
                full[:out, :cols // self.group] = t
                found.append(full.view(tiles, 16, blocks, per).transpose(1, 2).reshape(-1).view(torch.uint8))
        return torch.cat(found)


def project_ref(x, w, dtype, bias=None, a=None, b=None, scaling=0.0):
    """(y, bound): x [T, in] times w.w, with the adapter and the bias.

    fp32: 3 in products of exact terms (and as many of the offsets) are added.  bf16: of
    each group 2 group terms are added whose sums stay below 136 + 143 times sum |x| |s|
    (offsets: 136 sum |x| / 136), then the groups.  The adapter: in + 64 and rank
    additions."""
    u, x, cols = ch.half_step(dtype), x.double(), x.shape[1]
    y, bf = x @ w.w.t(), dtype == torch.bfloat16
    many = cols // w.group + 64
    if bf:
        size = x.abs() @ ((2 * w.group + 4) * 279 * w.step + many * 8 * w.step
                          + (2 * w.group + many) * w.off.abs()).t()
    else:
        size = (3 * cols + 64) * (x.abs() @ (8 * w.step + w.off.abs()).t())
    if a is not None:
        a, b = a.double(), b.double()
        y = y + scaling * ((x @ a) @ b)
        size = size + (cols + 128 + a.shape[1]) * abs(scaling) * ((x.abs() @ a.abs()) @ b.abs())
    if bias is not None:
        y = y + bias.double()
        size = size + 4 * bias.double().abs()
    return y, u * y.abs() + F * (size + 4 * y.abs())
