"""Plain attention in 64 bits for the tests of the attention kernels, and how far a kernel may be from it."""
import math

import torch


def reference(q, k, v, scale, causal=True):
    """One sequence: q [n, H, D], k and v [m, Hkv, D] -> (o [n, H, D], bound of the kernels' error [n, H, D]), 64 bits.

    With u = eps / 2 of the tensors' type a kernel may differ by
      u |o|                 the rounding of the result,
      u A                   that of the weights, relative to each: A = sum p |v|,
      2 (ds + 2^-16) A      scores in 32 bits, ds = (D + 4) 2^-23 scale |q|.|k| + |s| 2^-22 (products and sums, then the
                            scale and the argument's reduction), and exp2 itself, in numerator and denominator,
      m 2^-23 A             32-bit sums over m keys,
      2^-25 sum |v|         fp16 only: weights below the smallest normal, next to a denominator of 1 at least,
    and by the last place of the smallest values of the type."""
    n, H, D = q.shape
    m, Hkv, _ = k.shape
    u = torch.finfo(q.dtype).eps / 2
    half = q.dtype == torch.float16
    q, k, v = (t.double() for t in (q, k, v))
    G = H // Hkv
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    if m == 0 or n == 0:
        return o, tol
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(m - n)
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        s = scale * (q[:, h] @ kh.T)
        ds = (D + 4) * 2.0 ** -23 * abs(scale) * (q[:, h].abs() @ kh.abs().T) + s.abs() * 2.0 ** -22
        s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.where(seen, torch.exp(s - torch.where(top > -math.inf, top, 0.0)), 0.0)
        p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
        ds = torch.where(seen, ds, 0.0).amax(-1, keepdim=True)
        a = p @ vh.abs()
        o[:, h] = p @ vh
        tol[:, h] = u * o[:, h].abs() + (u + 2 * (ds + 2.0 ** -16) + m * 2.0 ** -23) * a * 1.01 + 2.0 ** -26
        if half:
            tol[:, h] += 2.0 ** -25 * (seen.double() @ vh.abs()) + 2.0 ** -25
    return o, tol


def packed_reference(q, k, v, queries, keys, scale, causal=True):
    """The same for packed sequences."""
    o, tol, a, b = [], [], 0, 0
    for n, m in zip(queries, keys):
        x, y = reference(q[a:a + n], k[b:b + m], v[b:b + m], scale, causal)
        o.append(x), tol.append(y)
        a, b = a + n, b + m
    return torch.cat(o), torch.cat(tol)


def check(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, the first at {bad.nonzero()[0].tolist()}: "
                           f"{float(got[bad][0])} for {float(want[bad][0])}, allowed {float(tol[bad][0]):.3g}")


def cumulated(lengths, device="cuda"):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)


def rows(gen, n, heads, dim, dtype, gain=1.0, wide=0):
    """[n, heads, dim]; `wide`: a part of rows that are that many elements longer."""
    x = (torch.randn(n, heads * dim + wide, generator=gen, device="cuda") * gain).to(dtype)
    return x[:, wide:].unflatten(1, (heads, dim))


class Paged:
    """Packed keys and values laid into pages in random order.  Everything else of the cache, and the ends of last pages,
    hold `garbage`; table entries behind a sequence's pages are `behind`."""

    def __init__(self, gen, k, v, keys, page, garbage=float("nan"), behind=-1, spare=3, layout="thd"):
        _, heads, dim = k.shape
        need = [-(-m // page) for m in keys]
        pages = sum(need) + spare
        if layout == "htd":     # heads outside of positions
            self.k, self.v = (torch.full((pages, heads, page, dim), garbage, dtype=k.dtype, device="cuda").transpose(1, 2)
                              for _ in range(2))
        else:
            cache = torch.full((2, pages, page, heads, dim), garbage, dtype=k.dtype, device="cuda")
            self.k, self.v = cache[0], cache[1]
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(page + pages)).tolist()
        self.tables = torch.full((len(keys), max(need + [1])), behind, dtype=torch.int32)
        slots, at = [], 0
        for b, m in enumerate(keys):
            mine = order[at:at + need[b]]
            at += need[b]
            self.tables[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
            slots += [mine[j // page] * page + j % page for j in range(m)]
        self.free = order[at:]
        self.tables = self.tables.cuda()
        self.slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
        s = self.slots.long()
        self.k[s // page, s % page] = k
        self.v[s // page, s % page] = v
