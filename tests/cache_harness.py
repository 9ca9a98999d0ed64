"""Plain 64-bit forms of the per-head q/k norms and of the paged cache, with
the bounds that their fp32 and bf16 results have to keep.

u(t) is half a step of the type, relative to the value (bf16 2^-8, fp32 2^-24);
every bound below is that of the roundings the kernels make, each counted at
its largest.
"""
import math

import torch

F = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotation(positions, theta, d):
    """cos, sin [T, D/2] in 64 bits."""
    i = torch.arange(d // 2, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.exp(-2.0 * i / d * math.log(theta))[None, :]
    return torch.cos(angle), torch.sin(angle)


def rotate(x, positions, theta, sign=1.0):
    """x [T, H, D] (64 bits) turned by sign * position; theta None: as it is."""
    if theta is None:
        return x
    c, s = (t[:, None, :] for t in rotation(positions, theta, x.shape[-1]))
    a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat([a * c - sign * b * s, b * c + sign * a * s], -1)


def pair_size(x):
    """The length of each element's rotation pair, for bounds."""
    a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    r = torch.sqrt(a * a + b * b)
    return torch.cat([r, r], -1)


def norm_ref(x, w, positions, theta, eps, dtype):
    """(y, bound).  The sum of D squares, the root, the division, two products
    and the rotation (its cos and sin off by 2^-22: the reduced angle is rounded
    to fp32) stay within 32 half steps of the pair's length for D <= 256 (lanes
    add at most 16 squares each, then 5 steps of a tree)."""
    x, w = x.double().cpu(), w.double().cpu()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    y = rotate(n, positions, theta)
    return y, half_step(dtype) * y.abs() + 32 * F * pair_size(n)


def norm_grad_ref(dy, x, w, positions, theta, eps, dtype):
    """(dx, bound, dw, bound).  dx is a difference of two terms, each good to 64
    half steps of its absolute terms; dw a sum of N terms in some fixed order,
    off by at most N half steps of the sum of their sizes."""
    dy, x, w = dy.double().cpu(), x.double().cpu(), w.double().cpu()
    d = x.shape[-1]
    g = rotate(dy, positions, theta, -1.0)
    gs = pair_size(dy)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    wg = w * g
    dx = r * wg - r ** 3 * x * (wg * x).sum(-1, keepdim=True) / d
    size = r * w.abs() * gs + r ** 3 * x.abs() * (w.abs() * gs * x.abs()).sum(-1, keepdim=True) / d
    terms = g * x * r
    n = terms.shape[0] * terms.shape[1]
    return (dx, half_step(dtype) * dx.abs() + 64 * F * size, terms.sum((0, 1)),
            (n + 64) * F * (gs * x.abs() * r).sum((0, 1)))


class Paged:
    """A batch of sequences in a paged cache.  seqs: (new tokens, tokens with
    them) each; every page that a sequence needs is a random one of `spare`
    more than are needed; unused table entries are -1; K and V share one
    allocation, so that pages are more than a page apart.  Rows of a page that
    hold no token are NaN.  columns: of the page table, at least what is needed."""

    def __init__(self, seqs, hq, hkv, d, page, dtype, seed, pad=0, spare=3, device="cuda", columns=0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.hq, self.hkv, self.d, self.page, self.dtype = seqs, hq, hkv, d, page, dtype
        self.tokens = sum(n for n, _ in seqs) + pad
        need = [-(-kv // page) for _, kv in seqs]
        order = torch.randperm(sum(need) + spare, generator=g)
        self.n_pages = len(order)
        table = torch.full((len(seqs), max(need + [columns - 1, 1]) + 1), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k].to(torch.int32)
            at += k
        normal = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
        self.k = [normal(kv, hkv, d) for _, kv in seqs]
        self.v = [normal(kv, hkv, d) for _, kv in seqs]
        self.q = normal(self.tokens, hq, d)
        both = torch.full((self.n_pages, 2, hkv, page, d), math.nan, dtype=dtype)
        for b, (_, kv) in enumerate(seqs):
            for p in range(kv):
                both[table[b, p // page], 0, :, p % page] = self.k[b][p]
                both[table[b, p // page], 1, :, p % page] = self.v[b][p]
        self.both = both.to(device)
        self.k_pages, self.v_pages = self.both[:, 0], self.both[:, 1]
        self.table = table.to(device)
        self.cu = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32).to(device)
        self.kv_lens = torch.tensor([kv for _, kv in seqs], dtype=torch.int32, device=device)

    def arrays(self):
        return self.k_pages, self.v_pages, self.cu, self.kv_lens, self.table

    def positions(self):
        """Of every row (0 behind the last sequence)."""
        at = [torch.arange(kv - n, kv) for n, kv in self.seqs]
        at.append(torch.zeros(self.tokens - sum(n for n, _ in self.seqs), dtype=torch.int64))
        return torch.cat(at)


def attend_ref(p, hidden=()):
    """(out, bound, lse, bound) [T, Hq, D] and [Hq, T] of p's rows over its keys,
    NaN behind the last sequence.  hidden: (sequence, position) keys that no row
    sees.

    Scores: D products are added in fp32, so a score is off by at most
    (D + 8) F of the sum of its terms' sizes, and a weight by twice that and
    by the exponential's few half steps; n weights are added in turn.  In bf16
    each weight is rounded before it multiplies V."""
    u = half_step(p.dtype)
    q = p.q.double()
    out = torch.full((p.tokens, p.hq, p.d), math.nan, dtype=torch.float64)
    out_b, lse = out.clone(), torch.full((p.hq, p.tokens), math.nan, dtype=torch.float64)
    lse_b = lse.clone()
    t = 0
    for b, (n, kv) in enumerate(p.seqs):
        if n == 0:
            continue
        see = torch.arange(kv)[None, :] <= torch.arange(kv - n, kv)[:, None]
        for s, j in hidden:
            if s == b:
                see[:, j] = False
        for h in range(p.hq):
            k, v = (x[b][:, h // (p.hq // p.hkv)].double() for x in (p.k, p.v))
            rows = slice(t, t + n)
            z = (q[rows, h] @ k.t() / math.sqrt(p.d)).masked_fill(~see, -math.inf)
            size = (q[rows, h].abs() @ k.abs().t() / math.sqrt(p.d)).masked_fill(~see, 0.0)
            top = z.amax(-1, keepdim=True)
            w = torch.where(see, torch.exp(z - torch.where(top.isinf(), 0.0, top)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            o, a = w @ v, w @ v.abs()
            off = ((p.d + 8) * F * size.amax(-1) + (kv + 64) * F)[:, None]
            out[rows, h], out_b[rows, h] = o, u * o.abs() + ((u if u > F else 0.0) + 4 * off) * a
            lse[h, rows] = torch.where(total == 0, -math.inf, top + torch.log(torch.where(total == 0, 1.0, total)))[:, 0]
            lse_b[h, rows] = 2 * off[:, 0] + 4 * F * torch.where(lse[h, rows].isinf(), 0.0, lse[h, rows].abs())
        t += n
    return out, out_b, lse, lse_b


def check(name, got, ref, bound):
    """got within bound of ref, infinities equal; rows that are NaN in ref are not looked at."""
    got = got.double().cpu()
    live = ~ref.isnan()
    assert not got[live].isnan().any(), f"{name}: NaN"
    inf = live & ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{name}: infinities differ"
    live &= ~ref.isinf()
    over = ((got - ref).abs() - bound)[live]
    worst = ((got - ref).abs() / bound.clamp(min=1e-300))[live]
    assert (over <= 0).all(), f"{name}: {int((over > 0).sum())} of {over.numel()} outside, worst {float(worst.max()):.3g} of the bound"
