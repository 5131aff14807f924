"""Plain 64-bit references of shared prefixes, attention weights and eviction in a paged cache."""
import math

import torch

import paged_ref as ref
from paged_ref import Cache


class Joined:
    """Sequences as the attention behind their prefixes sees them: each one's prefix rows, then
    its own.  `shared`: a Cache of the prefixes; `group[b]`: sequence b's, or None.

    Where a sequence has more new tokens than own keys, positions that hold nothing stand between
    its prefix and them, so that token i of n still sees own key j iff j <= len - n + i."""

    def __init__(self, own, shared, group):
        self.own, self.shared, self.group = own, shared, group
        self.hkv, self.news, self.cu = own.hkv, own.news, own.cu
        self.lens, self.rows = [], []
        for b, g in enumerate(group):
            p = shared.lens[g] if g is not None else 0
            pad = max(0, self.news[b] - own.lens[b])
            self.lens.append(p + pad + own.lens[b])
            self.rows.append([])
            for x in range(2):
                first = shared.rows[g][x] if g is not None else own.rows[b][x][:, :0]
                self.rows[b].append(torch.cat([first, first.new_zeros(own.hkv, pad, own.d), own.rows[b][x]], 1))

    def held(self, b):
        g = self.group[b]
        first = self.shared.held(g) if g is not None else torch.zeros(0, dtype=torch.bool)
        pad = torch.zeros(max(0, self.news[b] - self.own.lens[b]), dtype=torch.bool)
        return torch.cat([first, pad, self.own.held(b)])


def one_pool(own, shared):
    """Both caches' pages as one pool: the CPU tensors k, v, (ks, vs) and the prefixes' table."""
    table = torch.where((shared.table >= 0) & (shared.table < shared.pages), shared.table + own.pages, shared.table)
    pool = {x: torch.cat([getattr(own, x), getattr(shared, x)]) for x in "kv"}
    if own.q8:
        pool.update({x: torch.cat([getattr(own, x).view(torch.uint8), getattr(shared, x).view(torch.uint8)])
                     .view(torch.float8_e8m0fnu) for x in ("ks", "vs")})
    return pool, table


def weights(c, q, lse, causal=True, scale=None, max_len=None):
    """[B, Hkv, max_len] in 64 bits, and the bounds of their errors.

    A weight is a sum of terms p = e^(x - lse).  In 32 bits the score x = scale q k is off by at most
    2 s, s = D 2^-24 scale sum |q k| (its D products and sums); x log2 e, lse log2 e and their difference
    round once each, the first two factors too: 2^-23 (|x| + |lse|) + 2^-24 |x - lse| at most, in natural units
    (2^-22 (|x| + |lse|) in all); exp2 is good to 2^-22.  n terms' sum is off by n 2^-24 of it, and the
    result's smallest step is 2^-126 (terms below it may be flushed)."""
    t, hq, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    room = c.width * c.page if max_len is None else max_len
    w = torch.zeros(len(c.news), c.hkv, room, dtype=torch.float64)
    tol = torch.zeros_like(w)
    for b, n in enumerate(c.news):
        keys, t0 = min(c.lens[b], room), int(c.cu[b])
        held = c.held(b)[:keys]
        pos = torch.arange(keys)
        row = torch.arange(n)[:, None] + c.lens[b] - n
        seen = held[None] & ((pos[None] <= row) if causal else torch.ones_like(row, dtype=torch.bool))
        for h in range(hq):
            k = c.rows[b][0][h // (hq // c.hkv)][:keys]
            qb, z = q[t0:t0 + n, h].double(), lse[h, t0:t0 + n, None].double()
            x = qb @ k.T * scale
            p = torch.where(seen & (z > -math.inf), torch.exp(x - z), 0.0)
            s = d * 2.0 ** -24 * abs(scale) * (qb.abs() @ k.abs().T)
            off = 2 * s + 2.0 ** -22 * (x.abs() + z.abs()) + 2.0 ** -22 + n * hq * 2.0 ** -24
            w[b, h // (hq // c.hkv), :keys] += p.sum(0)
            tol[b, h // (hq // c.hkv), :keys] += torch.where(p > 0, p * off * 1.01, 0.0).sum(0) + n * 2.0 ** -126
    return w, tol


def stays(w, held, length, keep, recent):
    """The positions of one head's rows that stay, in order: Python's sort of plain numbers."""
    at = [j for j in range(len(held)) if held[j]]
    last = [j for j in at if j >= length - recent]
    rest = [j for j in at if j < length - recent]
    rest.sort(key=lambda j: (math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0.0, j))
    return sorted(rest[:max(0, min(keep, len(at)) - len(last))] + last)


def evicted(c, pools, w, to_table, keep, recent):
    """What an eviction leaves: (pools, lens, weights) as CPU tensors."""
    pools = [x.clone() for x in pools]
    old = [x.clone() for x in pools]
    out = torch.zeros(len(c.lens), c.hkv, to_table.shape[1] * c.page)
    lens = []
    for b, n in enumerate(c.lens):
        held = c.held(b)
        for h in range(c.hkv):
            left = stays(w[b, h].tolist(), held.tolist(), n, keep, recent)
            for r, j in enumerate(left):
                out[b, h, r] = w[b, h, j]
                p, t = int(c.table[b, j // c.page]), int(to_table[b, r // c.page])
                if not 0 <= t < pools[0].shape[0]:
                    continue
                for x, y in zip(pools, old):
                    u, v = (z.view(torch.uint8) if z.element_size() == 1 else z for z in (x, y))
                    u[t, h, r % c.page] = v[p, h, j % c.page]
        lens.append(min(keep, int(held.sum())))
    return pools, torch.tensor(lens, dtype=torch.int32), out


__all__ = ["Cache", "Joined", "evicted", "one_pool", "ref", "stays", "weights"]
